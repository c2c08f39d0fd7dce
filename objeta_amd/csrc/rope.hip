// rope.hip — rotary positions, alone or fused with the write of new keys and values into
// the paged cache.
//
// A pair (x, y) at position p turns by the angle a = p f: (x cos a - y sin a, x sin a +
// y cos a). f / 2 pi is held as a 64-bit fraction of a turn, so p times it modulo 2^64 is
// the place on the circle with no reduction to make: the top two bits (after rounding to
// the nearest quarter) give the quadrant, the next 32 the angle within it, |a| <= pi / 4,
// where the Taylor series to a^9 and a^10 leave less than 2e-9 in float.
//
// Bound: HBM (8191 tokens of 72 heads of 128, float to bf16: 453 MB in 83 us, 5.4 TB/s), or the
// latency of dependent reads when tokens are few. One workgroup takes a token; a thread takes
// four pairs (or eight elements of the part that is copied) of every head in turn, so sines and
// cosines are computed once a token and thread, for all its heads, and the next head's elements
// are read ahead.
#include "kernels.hpp"
#include "kv_common.hpp"

#include <cmath>

namespace objeta {
namespace dev {

struct RopeArgs {
    uint64_t turn[128];
    const int32_t* pos;
    const void *q, *k, *v;
    void *q_out, *k_out;  // k_out: rows; NULL when keys and values go to the cache
    uint64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;  // elements
    uint32_t nq, nk, nv, dim, half, layout;  // half: pairs of a rotated head
    float amp;
    int32_t q_out_type, k_out_type;
    // cache
    void *ck, *cv;
    uint64_t layer_off;  // elements
    KvView kv;
    const int32_t *seqs, *cu;
    uint32_t n_batch, first;  // first: the launch's first token
    uint32_t* err;
};

typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));

template <int T> struct Elem;
template <> struct Elem<kDtF32> { typedef float type; typedef f4 vec; };
template <> struct Elem<kDtF16> { typedef _Float16 type; typedef half4 vec; };
template <> struct Elem<kDtBF16> { typedef __bf16 type; typedef bf4 vec; };

// Four elements at p[0], p[step], ...; the first n of them where VEC is false.
template <int T, bool VEC>
__device__ __forceinline__ f4 load4(const void* base, uint64_t at, uint32_t step, uint32_t n) {
    const typename Elem<T>::type* p = static_cast<const typename Elem<T>::type*>(base) + at;
    if constexpr (VEC) {
        return __builtin_convertvector(*reinterpret_cast<const typename Elem<T>::vec*>(p), f4);
    } else {
        f4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (i < n) v[i] = static_cast<float>(p[i * step]);
        return v;
    }
}

template <int T, bool VEC>
__device__ __forceinline__ void store4_as(void* base, uint64_t at, uint32_t step, uint32_t n, f4 v) {
    typename Elem<T>::type* p = static_cast<typename Elem<T>::type*>(base) + at;
    if constexpr (VEC) {
        *reinterpret_cast<typename Elem<T>::vec*>(p) = __builtin_convertvector(v, typename Elem<T>::vec);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i)
            if (i < n) p[i * step] = static_cast<typename Elem<T>::type>(v[i]);
    }
}

template <bool VEC>
__device__ __forceinline__ void store4(int32_t type, void* base, uint64_t at, uint32_t step, uint32_t n, f4 v) {
    if (type == kDtF32) store4_as<kDtF32, VEC>(base, at, step, n, v);
    else if (type == kDtF16) store4_as<kDtF16, VEC>(base, at, step, n, v);
    else store4_as<kDtBF16, VEC>(base, at, step, n, v);
}

// Cosine and sine of `place` / 2^64 turns.
__device__ __forceinline__ void cos_sin(uint64_t place, float& c, float& s) {
    const uint32_t quarter = static_cast<uint32_t>((place + (uint64_t(1) << 61)) >> 62);
    const int32_t in = static_cast<int32_t>((place - (static_cast<uint64_t>(quarter) << 62)) >> 32);
    const float a = static_cast<float>(in) * 1.46291807926715968e-9f;  // 2 pi / 2^32
    const float z = a * a;
    float sp = 2.75573192239859e-6f;  // a^9 / 9! and on
    sp = __builtin_fmaf(sp, z, -1.98412698412698e-4f);
    sp = __builtin_fmaf(sp, z, 8.33333333333333e-3f);
    sp = __builtin_fmaf(sp, z, -1.66666666666667e-1f);
    const float sn = __builtin_fmaf(a * z, sp, a);
    float cp = -2.75573192239859e-7f;  // a^10 / 10! and on
    cp = __builtin_fmaf(cp, z, 2.48015873015873e-5f);
    cp = __builtin_fmaf(cp, z, -1.38888888888889e-3f);
    cp = __builtin_fmaf(cp, z, 4.16666666666667e-2f);
    cp = __builtin_fmaf(cp, z, -0.5f);
    const float cs = __builtin_fmaf(cp, z, 1.0f);
    const float u = (quarter & 1) ? sn : cs, w = (quarter & 1) ? cs : sn;
    c = ((quarter + 1) & 2) ? -u : u;
    s = (quarter & 2) ? -w : w;
}

template <int IN, bool VEC>
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    const uint64_t t = static_cast<uint64_t>(a.first) + blockIdx.x;
    const uint32_t rotated = (a.half + 3) >> 2;                      // units of four pairs
    const uint32_t tail = a.dim - 2 * a.half, copied = (tail + 7) >> 3;  // units of eight elements
    uint32_t units = rotated + copied;
    if (a.nv && units < (a.dim >> 3)) units = a.dim >> 3;
    const uint32_t per = 256 / units;  // heads at a time
    const uint32_t unit = threadIdx.x % units, first = threadIdx.x / units;
    const uint32_t heads = a.nq + a.nk + a.nv, step_h = per * gridDim.y;
    const bool half = a.layout == OBJETA_HIP_ROPE_HALF;

    // Two groups of four elements of head h: the pairs' halves, or eight of the part that is
    // copied. `at`: the first group's place in the head, the second's.
    auto places = [&](bool turn, uint32_t& n, uint32_t& ox, uint32_t& oy, uint32_t& nx, uint32_t& ny, uint32_t& step) {
        if (turn && unit < rotated) {
            const uint32_t i = 4 * unit;
            n = a.half - i < 4 ? a.half - i : 4;
            nx = ny = n;
            step = half || VEC ? 1 : 2;
            ox = half ? i : 2 * i;
            oy = half ? a.half + i : (VEC ? 2 * i + 4 : 2 * i + 1);
        } else {
            ox = turn ? 2 * a.half + 8 * (unit - rotated) : 8 * unit;
            oy = ox + 4, step = 1;
            n = ox < a.dim ? a.dim - ox : 0;
            nx = n < 4 ? n : 4, ny = n < 4 ? 0 : (n < 8 ? n - 4 : 4);
        }
    };
    auto load = [&](uint32_t h, f4& x, f4& y) {
        if (h >= heads) return;
        const bool is_q = h < a.nq, is_k = !is_q && h < a.nq + a.nk;
        const void* in = is_q ? a.q : (is_k ? a.k : a.v);
        const uint64_t stride = is_q ? a.q_stride : (is_k ? a.k_stride : a.v_stride);
        const uint64_t from = t * stride + static_cast<uint64_t>(h - (is_q ? 0 : (is_k ? a.nq : a.nq + a.nk))) * a.dim;
        uint32_t n, ox, oy, nx, ny, step;
        places(is_q || is_k, n, ox, oy, nx, ny, step);
        if (!n) return;
        x = load4<IN, VEC>(in, from + ox, step, nx);
        y = load4<IN, VEC>(in, from + oy, step, ny);
    };

    // The first head's elements, the position and the turns are on their way while the slot is
    // looked up.
    uint32_t h = blockIdx.y * per + first;
    const bool idle = first >= per;
    f4 x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x;
    uint64_t turns[4] = {0, 0, 0, 0};
    int64_t p = 0;
    if (!idle) {
        load(h, x, y);
        if (unit < rotated) {
            p = a.pos[t];
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (VEC || 4 * unit + i < a.half) turns[i] = a.turn[4 * unit + i];
        }
    }

    // where this token's keys and values go: base offset of head 0's row in the pool
    bool keep = a.k_out != nullptr;
    uint64_t slot_off = 0, head_step = a.dim;
    if (a.ck) {
        const int64_t r = static_cast<int64_t>(t);
        const RowEntry<true> entry(a.cu, a.seqs, a.n_batch, r);
        keep = entry.any && !entry.again;  // a later entry's rows of the same sequence take these slots
        if (keep) {
            bool ok = seq_ok(a.kv, entry.seq);
            const int32_t len = ok ? a.kv.lens[entry.seq] : 0;
            const int64_t slot = static_cast<int64_t>(len) - (entry.hi - r);
            ok = ok && len_ok(a.kv, len) && slot >= 0;
            const int32_t page =
                ok ? a.kv.table[static_cast<uint64_t>(entry.seq) * a.kv.max_pages + (slot >> a.kv.shift)] : -1;
            ok = ok && page_ok(a.kv, page);
            if (!ok && threadIdx.x == 0) atomicOr(a.err, kErrIndex);
            keep = ok;
            head_step = static_cast<uint64_t>(a.dim) << a.kv.shift;
            slot_off = a.layer_off + static_cast<uint64_t>(ok ? page : 0) * a.nk * head_step +
                       (static_cast<uint64_t>(slot) & ((1u << a.kv.shift) - 1)) * a.dim;
        }
    }
    if (idle) return;

    f4 cs = {1.0f, 1.0f, 1.0f, 1.0f}, sn = {0.0f, 0.0f, 0.0f, 0.0f};
    if (unit < rotated) {
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) {
            if (VEC || 4 * unit + i < a.half) {
                float c, s;
                cos_sin(static_cast<uint64_t>(p) * turns[i], c, s);
                cs[i] = c * a.amp;
                sn[i] = s * a.amp;
            }
        }
    }
    for (; h < heads; h += step_h) {
        f4 u = x, w = y;
        load(h + step_h, x, y);
        const bool is_q = h < a.nq, is_k = !is_q && h < a.nq + a.nk;
        if (!is_q && !keep) break;
        void* out;
        uint64_t to;
        if (is_q) {
            out = a.q_out;
            to = t * a.q_out_stride + static_cast<uint64_t>(h) * a.dim;
        } else {
            const uint32_t g = is_k ? h - a.nq : h - a.nq - a.nk;
            out = a.ck ? (is_k ? a.ck : a.cv) : a.k_out;
            to = a.ck ? slot_off + g * head_step : t * a.k_out_stride + static_cast<uint64_t>(g) * a.dim;
        }
        const int32_t type = is_q ? a.q_out_type : a.k_out_type;
        const bool turn = is_q || is_k;
        uint32_t n, ox, oy, nx, ny, step;
        places(turn, n, ox, oy, nx, ny, step);
        if (!n) continue;
        if (turn && unit < rotated) {
            const bool pairs = VEC && !half;  // x and y as they lie: two pairs each
            const f4 ex = pairs ? f4{u.x, u.z, w.x, w.z} : u, ey = pairs ? f4{u.y, u.w, w.y, w.w} : w;
            const f4 c = ex * cs - ey * sn, s = ex * sn + ey * cs;
            u = pairs ? f4{c.x, s.x, c.y, s.y} : c;
            w = pairs ? f4{c.z, s.z, c.w, s.w} : s;
        }
        store4<VEC>(type, out, to + ox, step, nx, u);
        store4<VEC>(type, out, to + oy, step, ny, w);
    }
}

}  // namespace dev

using namespace dev;

int32_t check_rope(const objeta_hip_rope* r, uint64_t head_dim, const char* action) {
    if (!r) OBJ_FAIL(kInvalidInput, action, "rope is NULL");
    if (r->rotary_dim < 2 || r->rotary_dim > kMaxHeadDim || r->rotary_dim % 2)
        OBJ_FAIL(kInvalidInput, action, strf("rotary_dim %u must be even, 2 to 256", r->rotary_dim));
    if (r->rotary_dim > head_dim)
        OBJ_FAIL(kInvalidInput, action,
                 strf("rotary_dim %u exceeds head_dim %llu", r->rotary_dim, (unsigned long long)head_dim));
    if (r->layout != OBJETA_HIP_ROPE_INTERLEAVED && r->layout != OBJETA_HIP_ROPE_HALF)
        OBJ_FAIL(kInvalidInput, action, strf("unknown rotary layout %d", r->layout));
    return 0;
}

int32_t check_kv(const objeta_hip_kv_cache* c, const char* action) {
    if (!c) OBJ_FAIL(kInvalidInput, action, "cache is NULL");
    if (!c->k || !c->v || !c->page_table || !c->seq_lens || !c->ref_counts)
        OBJ_FAIL(kInvalidInput, action, "NULL pointer in the cache");
    if (!dtype_ok(c->dtype)) OBJ_FAIL(kInvalidInput, action, strf("cache dtype %d must be F32, F16 or BF16", c->dtype));
    if (!c->n_layers || !c->n_pages || !c->n_kv_heads || !c->n_seqs || !c->max_pages)
        OBJ_FAIL(kInvalidInput, action, "cache of no layers, pages, heads or sequences");
    if (!head_dim_ok(c->head_dim))
        OBJ_FAIL(kInvalidInput, action, strf("head_dim %u must be a multiple of 8 up to 256", c->head_dim));
    if (c->page_size < 8 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
        OBJ_FAIL(kInvalidInput, action, strf("page_size %u must be a power of two, 8 to 256", c->page_size));
    if (reinterpret_cast<uintptr_t>(c->k) % 16 || reinterpret_cast<uintptr_t>(c->v) % 16)
        OBJ_FAIL(kInvalidInput, action, "cache k and v must be 16-byte aligned");
    if (c->n_pages > 0x7FFFFFFFu || c->n_seqs > 0x7FFFFFFFu || c->n_kv_heads > 65535u || c->n_layers > 65535u ||
        static_cast<uint64_t>(c->max_pages) * c->page_size > kMaxTokens ||
        static_cast<double>(c->n_layers) * c->n_pages * c->n_kv_heads * c->page_size * c->head_dim > 1e14)
        OBJ_FAIL(kInvalidInput, action, "cache too large");
    return 0;
}

namespace {

void set_rope(RopeArgs& a, const objeta_hip_rope* r) {
    if (!r) return;
    for (uint32_t i = 0; i < r->rotary_dim / 2; ++i) a.turn[i] = r->turn[i];
    a.half = r->rotary_dim / 2;
    a.layout = static_cast<uint32_t>(r->layout);
    a.amp = r->amplitude;
}

bool aligned(const void* p, uint64_t stride, uint64_t size) {
    return reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && stride % 4 == 0;
}

// One output against the inputs and the other outputs: it may be its own input.
int32_t check_rows(const char* action, const RowSet& out, const RowSet& own, bool same_type, const RowSet* others, int n) {
    if (rows_overlap(out, own) && !(out.p == own.p && out.stride == own.stride && same_type))
        OBJ_FAIL(kInvalidInput, action, "an output overlaps its input without being it (address, stride, type)");
    for (int i = 0; i < n; ++i)
        if (rows_overlap(out, others[i])) OBJ_FAIL(kInvalidInput, action, "an output overlaps another tensor");
    return 0;
}

int32_t check_tensor(const char* action, const char* what, const void* p, uint64_t n, uint64_t stride, uint64_t heads,
                     uint64_t dim, uint64_t size) {
    if (!p) OBJ_FAIL(kInvalidInput, action, strf("%s is NULL", what));
    if (reinterpret_cast<uintptr_t>(p) % size)
        OBJ_FAIL(kInvalidInput, action, strf("%s is not aligned to its element type", what));
    if (!extent_ok(n, stride, heads * dim, size)) OBJ_FAIL(kInvalidInput, action, strf("%s is too large", what));
    if (n > 1 && stride < heads * dim)
        OBJ_FAIL(kInvalidInput, action,
                 strf("%s stride %llu is less than its %llu elements", what, (unsigned long long)stride,
                      (unsigned long long)(heads * dim)));
    return 0;
}

template <bool VEC>
void launch_typed(hipStream_t s, int32_t dtype, dim3 grid, const RopeArgs& a) {
    if (dtype == kDtF32) hipLaunchKernelGGL((rope_kernel<kDtF32, VEC>), grid, dim3(256), 0, s, a);
    else if (dtype == kDtF16) hipLaunchKernelGGL((rope_kernel<kDtF16, VEC>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((rope_kernel<kDtBF16, VEC>), grid, dim3(256), 0, s, a);
}

int32_t launch_rope(hipStream_t s, int32_t dtype, uint64_t n_tokens, RopeArgs& a, const char* action) {
    const uint64_t in = dtype_size(dtype), qo = dtype_size(a.q_out_type), ko = dtype_size(a.k_out_type);
    // four elements at once where every row starts on their boundary and the parts are whole
    bool vec = a.half % 4 == 0;
    if (a.nq) vec = vec && aligned(a.q, a.q_stride, in) && aligned(a.q_out, a.q_out_stride, qo);
    if (a.nk) vec = vec && aligned(a.k, a.k_stride, in) && (a.ck || aligned(a.k_out, a.k_out_stride, ko));
    if (a.nv) vec = vec && aligned(a.v, a.v_stride, in);
    // A workgroup a token computes its sines once; few tokens take more, each with a part of the
    // heads, so that no thread has several heads to wait for (32 tokens appended, 40 heads:
    // 4.4 us, by a workgroup a token 6.0; one token of 36 heads 3.6 and 5.0).
    const uint32_t rotated = (a.half + 3) / 4, tail = (a.dim - 2 * a.half + 7) / 8;
    const uint32_t units = a.nv && rotated + tail < a.dim / 8 ? a.dim / 8 : rotated + tail;
    const uint64_t turns = (a.nq + a.nk + a.nv + 256 / units - 1) / (256 / units), room = 1024 / n_tokens;
    const uint64_t y = room < 1 ? 1 : (room < turns ? room : turns);
    for (uint64_t first = 0; first < n_tokens; first += kMostGroups) {
        const uint64_t n = n_tokens - first < kMostGroups ? n_tokens - first : kMostGroups;
        const dim3 grid(static_cast<uint32_t>(n), static_cast<uint32_t>(y));
        a.first = static_cast<uint32_t>(first);
        if (vec) launch_typed<true>(s, dtype, grid, a);
        else launch_typed<false>(s, dtype, grid, a);
        OBJ_HIP(hipGetLastError(), action);
    }
    return 0;
}

}  // namespace

}  // namespace objeta

using namespace objeta;

extern "C" {

int32_t objeta_hip_rope_init(const objeta_hip_rope_params* params, objeta_hip_rope* out) {
    OBJ_GUARD_BEGIN
    const char* action = "rope_init";
    if (!params || !out) OBJ_FAIL(kInvalidInput, action, "NULL argument");
    const objeta_hip_rope_params p = *params;
    if (p.rotary_dim < 2 || p.rotary_dim > kMaxHeadDim || p.rotary_dim % 2)
        OBJ_FAIL(kInvalidInput, action, strf("rotary_dim %u must be even, 2 to 256", p.rotary_dim));
    if (p.layout != OBJETA_HIP_ROPE_INTERLEAVED && p.layout != OBJETA_HIP_ROPE_HALF)
        OBJ_FAIL(kInvalidInput, action, strf("unknown rotary layout %d", p.layout));
    if (p.scaling < OBJETA_HIP_ROPE_NONE || p.scaling > OBJETA_HIP_ROPE_YARN)
        OBJ_FAIL(kInvalidInput, action, strf("unknown rotary scaling %d", p.scaling));
    if (!(std::isfinite(p.theta) && p.theta > 0.0)) OBJ_FAIL(kInvalidInput, action, "theta must be positive and finite");
    if (p.scaling != OBJETA_HIP_ROPE_NONE && !(std::isfinite(p.factor) && p.factor > 0.0))
        OBJ_FAIL(kInvalidInput, action, "factor must be positive and finite");
    if (!(std::isfinite(p.amplitude) && p.amplitude >= 0.0 && p.amplitude < 1e30))
        OBJ_FAIL(kInvalidInput, action, "amplitude must be finite and not negative");
    const bool yarn = p.scaling == OBJETA_HIP_ROPE_YARN;
    if (yarn && !(p.factor >= 1.0 && p.theta > 1.0 && std::isfinite(p.original_context) && p.original_context > 0.0 &&
                  std::isfinite(p.beta_fast) && p.beta_slow > 0.0 && p.beta_fast > p.beta_slow))
        OBJ_FAIL(kInvalidInput, action,
                 "YARN needs factor >= 1, theta > 1, original_context > 0 and beta_fast > beta_slow > 0");
    const long double pi2 = 6.283185307179586476925286766559005768L;
    const long double r = p.rotary_dim;
    long double theta = p.theta;
    if (p.scaling == OBJETA_HIP_ROPE_NTK && p.rotary_dim > 2) theta *= powl(p.factor, r / (r - 2));
    long double low = 0, high = 0;
    if (yarn) {
        const long double per = r / (2 * logl(theta));
        low = floorl(per * logl(p.original_context / (p.beta_fast * pi2)));
        high = ceill(per * logl(p.original_context / (p.beta_slow * pi2)));
        low = low < 0 ? 0 : low;
        high = high > r - 1 ? r - 1 : high;
    }
    objeta_hip_rope o{};
    for (uint32_t i = 0; i < p.rotary_dim / 2; ++i) {
        long double f = powl(theta, -2.0L * i / r);
        if (p.scaling == OBJETA_HIP_ROPE_LINEAR) f /= p.factor;
        if (yarn) {
            const long double span = high - low < 0.001L ? 0.001L : high - low;
            long double ramp = (i - low) / span;
            ramp = ramp < 0 ? 0 : (ramp > 1 ? 1 : ramp);
            f = f / p.factor * ramp + f * (1 - ramp);
        }
        if (!std::isfinite(static_cast<double>(f))) OBJ_FAIL(kInvalidInput, action, "frequencies are not finite");
        long double turns = f / pi2;
        turns -= floorl(turns);
        const long double scaled = floorl(ldexpl(turns, 64) + 0.5L);
        o.turn[i] = scaled >= 18446744073709551616.0L ? 0 : static_cast<uint64_t>(scaled);
    }
    o.rotary_dim = p.rotary_dim;
    o.layout = p.layout;
    o.amplitude = static_cast<float>(p.amplitude > 0.0 ? p.amplitude : (yarn ? 0.1 * std::log(p.factor) + 1.0 : 1.0));
    *out = o;
    return 0;
    OBJ_GUARD_END
}

int32_t objeta_hip_rope_device(objeta_hip_context* ctx, objeta_hip_stream stream, const objeta_hip_rope* rope,
                               const int32_t* d_positions, uint64_t n_tokens, uint64_t head_dim, int32_t dtype,
                               int32_t out_dtype, const void* d_q, uint64_t q_stride, void* d_q_out,
                               uint64_t q_out_stride, uint64_t n_q_heads, const void* d_k, uint64_t k_stride,
                               void* d_k_out, uint64_t k_out_stride, uint64_t n_k_heads) {
    OBJ_GUARD_BEGIN
    const char* action = "rope_device";
    OBJ_TRY(check_ctx(ctx, action));
    if (!head_dim_ok(head_dim))
        OBJ_FAIL(kInvalidInput, action, strf("head_dim %llu must be a multiple of 8 up to 256", (unsigned long long)head_dim));
    OBJ_TRY(check_rope(rope, head_dim, action));
    if (!dtype_ok(dtype) || !dtype_ok(out_dtype)) OBJ_FAIL(kInvalidInput, action, "dtype must be F32, F16 or BF16");
    if (n_q_heads == 0 || n_q_heads > 65535 || n_k_heads > 65535)
        OBJ_FAIL(kInvalidInput, action, "n_q_heads must be 1 to 65535, n_k_heads 0 to 65535");
    if (n_tokens >= (uint64_t(1) << 31)) OBJ_FAIL(kInvalidInput, action, "too many tokens");
    if (n_tokens == 0) return 0;
    if (!d_positions) OBJ_FAIL(kInvalidInput, action, "positions are NULL");
    const uint64_t in = dtype_size(dtype), os = dtype_size(out_dtype);
    OBJ_TRY(check_tensor(action, "q", d_q, n_tokens, q_stride, n_q_heads, head_dim, in));
    OBJ_TRY(check_tensor(action, "q_out", d_q_out, n_tokens, q_out_stride, n_q_heads, head_dim, os));
    RowSet q{d_q, q_stride * in, n_q_heads * head_dim * in, n_tokens};
    RowSet qo{d_q_out, q_out_stride * os, n_q_heads * head_dim * os, n_tokens}, k{}, ko{};
    if (n_k_heads) {
        OBJ_TRY(check_tensor(action, "k", d_k, n_tokens, k_stride, n_k_heads, head_dim, in));
        OBJ_TRY(check_tensor(action, "k_out", d_k_out, n_tokens, k_out_stride, n_k_heads, head_dim, os));
        k = RowSet{d_k, k_stride * in, n_k_heads * head_dim * in, n_tokens};
        ko = RowSet{d_k_out, k_out_stride * os, n_k_heads * head_dim * os, n_tokens};
    }
    const RowSet other_q[] = {k, ko}, other_k[] = {q};
    OBJ_TRY(check_rows(action, qo, q, dtype == out_dtype, other_q, 2));
    OBJ_TRY(check_rows(action, ko, k, dtype == out_dtype, other_k, 1));
    OBJ_HIP(hipSetDevice(ctx->device), "hipSetDevice");
    RopeArgs a{};
    set_rope(a, rope);
    a.pos = d_positions;
    a.q = d_q, a.q_out = d_q_out, a.q_stride = q_stride, a.q_out_stride = q_out_stride;
    a.nq = static_cast<uint32_t>(n_q_heads), a.nk = static_cast<uint32_t>(n_k_heads);
    a.dim = static_cast<uint32_t>(head_dim);
    if (n_k_heads) a.k = d_k, a.k_out = d_k_out, a.k_stride = k_stride, a.k_out_stride = k_out_stride;
    a.q_out_type = a.k_out_type = out_dtype;
    a.err = ctx->err_word;
    return launch_rope(resolve_stream(ctx, stream), dtype, n_tokens, a, action);
    OBJ_GUARD_END
}

int32_t objeta_hip_kv_append_device(objeta_hip_context* ctx, objeta_hip_stream stream, const objeta_hip_kv_cache* cache,
                                    uint64_t layer, const int32_t* d_seqs, const int32_t* d_cu_rows, uint64_t n_batch,
                                    uint64_t n_rows, int32_t dtype, const void* d_k, uint64_t k_stride, const void* d_v,
                                    uint64_t v_stride, const objeta_hip_rope* rope, const int32_t* d_positions,
                                    const void* d_q, uint64_t q_stride, uint64_t n_q_heads, int32_t q_out_dtype,
                                    void* d_q_out, uint64_t q_out_stride) {
    OBJ_GUARD_BEGIN
    const char* action = "kv_append_device";
    OBJ_TRY(check_ctx(ctx, action));
    OBJ_TRY(check_kv(cache, action));
    const uint64_t dim = cache->head_dim, nk = cache->n_kv_heads;
    if (layer >= cache->n_layers)
        OBJ_FAIL(kInvalidInput, action, strf("layer %llu out of bounds (len=%u)", (unsigned long long)layer, cache->n_layers));
    if (rope) OBJ_TRY(check_rope(rope, dim, action));
    if (!dtype_ok(dtype) || (n_q_heads && !dtype_ok(q_out_dtype)))
        OBJ_FAIL(kInvalidInput, action, "dtype must be F32, F16 or BF16");
    if (n_q_heads > 65535) OBJ_FAIL(kInvalidInput, action, "n_q_heads must be 0 to 65535");
    if (n_q_heads == 0 && (d_q || d_q_out)) OBJ_FAIL(kInvalidInput, action, "q or q_out without n_q_heads");
    if (n_rows >= (uint64_t(1) << 31) || n_batch >= (uint64_t(1) << 31)) OBJ_FAIL(kInvalidInput, action, "too many rows");
    if (n_rows == 0 || (n_batch == 0 && n_q_heads == 0)) return 0;
    if (n_batch && (!d_seqs || !d_cu_rows)) OBJ_FAIL(kInvalidInput, action, "sequences or cu_rows are NULL");
    if (rope && !d_positions) OBJ_FAIL(kInvalidInput, action, "positions are NULL");
    const uint64_t in = dtype_size(dtype);
    OBJ_TRY(check_tensor(action, "k", d_k, n_rows, k_stride, nk, dim, in));
    OBJ_TRY(check_tensor(action, "v", d_v, n_rows, v_stride, nk, dim, in));
    const RowSet k{d_k, k_stride * in, nk * dim * in, n_rows}, v{d_v, v_stride * in, nk * dim * in, n_rows};
    const uint64_t pool = static_cast<uint64_t>(cache->n_layers) * cache->n_pages * nk * cache->page_size * dim *
                          dtype_size(cache->dtype);
    const RowSet ck{cache->k, pool, pool, 1}, cv{cache->v, pool, pool, 1};
    RowSet q{}, qo{};
    if (n_q_heads) {
        const uint64_t os = dtype_size(q_out_dtype);
        OBJ_TRY(check_tensor(action, "q", d_q, n_rows, q_stride, n_q_heads, dim, in));
        OBJ_TRY(check_tensor(action, "q_out", d_q_out, n_rows, q_out_stride, n_q_heads, dim, os));
        q = RowSet{d_q, q_stride * in, n_q_heads * dim * in, n_rows};
        qo = RowSet{d_q_out, q_out_stride * os, n_q_heads * dim * os, n_rows};
        const RowSet others[] = {k, v, ck, cv};
        OBJ_TRY(check_rows(action, qo, q, dtype == q_out_dtype, others, 4));
    }
    const RowSet in_k[] = {k, v, q, cv}, in_v[] = {k, v, q};
    OBJ_TRY(check_rows(action, ck, RowSet{}, true, in_k, 4));
    OBJ_TRY(check_rows(action, cv, RowSet{}, true, in_v, 3));
    OBJ_HIP(hipSetDevice(ctx->device), "hipSetDevice");
    RopeArgs a{};
    set_rope(a, rope);
    a.pos = d_positions;
    a.nq = static_cast<uint32_t>(n_q_heads);
    a.dim = cache->head_dim;
    if (n_q_heads) a.q = d_q, a.q_out = d_q_out, a.q_stride = q_stride, a.q_out_stride = q_out_stride;
    a.q_out_type = n_q_heads ? q_out_dtype : dtype;
    a.k_out_type = cache->dtype;
    if (n_batch) {  // without entries the keys and values are nobody's: queries alone
        a.nk = a.nv = cache->n_kv_heads;
        a.k = d_k, a.k_stride = k_stride, a.v = d_v, a.v_stride = v_stride;
        a.ck = cache->k, a.cv = cache->v;
        a.layer_off = layer * cache->n_pages * nk * cache->page_size * dim;
        a.kv = kv_view(*cache);
        a.seqs = d_seqs, a.cu = d_cu_rows, a.n_batch = static_cast<uint32_t>(n_batch);
    }
    a.err = ctx->err_word;
    return launch_rope(resolve_stream(ctx, stream), dtype, n_rows, a, action);
    OBJ_GUARD_END
}

}  // extern "C"
