// norm.hip — the RMS norm with the residual's addition and 8-bit output, and rows of a matrix
// quantized to 8 bits by the same rule.
//
//   h = x + r                      (float; rounded to the residual's type where it is written back)
//   y_i = h_i (w_i + o) / sqrt(sum h^2 / n + eps)
//   int8: s = max |y| / 127, code = y / s rounded to the nearest, halves to even
//   FP8:  the rule of the official path (quant_rules.hpp) on blocks of 128
//
// Sums of squares, the root and y are held in 64 bits and y is rounded once: codes turn at
// halves of a step, and with sums in 32 bits one in some 40000 would depend on the order they were
// taken in. 64-bit products run at the rate of 32-bit ones here, and the kernel waits for memory.
//
// A row's elements stay in the registers of WAVES waves, eight of each vector in a thread, from
// the one read to the one write. Bound: HBM (8192 rows of 4096 in bf16, the residual in float, to int8
// 69 us, 5.35 TB/s; 14336 rows of 4096 floats quantized 49.9 us, 5.9 TB/s, where a copy reaches 5.1), or the
// latency of one row (one of 2048: 5.6 us a call).
#include "dense_common.hpp"
#include "kernels.hpp"
#include "quant_rules.hpp"

namespace objeta {

int32_t check_dense_rows(const char* action, const char* what, const void* p, uint64_t n, uint64_t stride, uint64_t width,
                         uint64_t size) {
    if (!p) OBJ_FAIL(kInvalidInput, action, strf("%s is NULL", what));
    if (reinterpret_cast<uintptr_t>(p) % size)
        OBJ_FAIL(kInvalidInput, action, strf("%s is not aligned to its element type", what));
    if (n > 1 && stride < width)
        OBJ_FAIL(kInvalidInput, action, strf("%s stride %llu is less than its %llu elements", what, (unsigned long long)stride,
                                             (unsigned long long)width));
    if (n > 1 && stride >= (uint64_t(1) << 31)) OBJ_FAIL(kInvalidInput, action, strf("%s stride is too large", what));
    return 0;
}

int32_t check_dense_apart(const char* action, const char* what, const RowSet& out, const RowSet* others, int n, int own) {
    for (int i = 0; i < n; ++i) {
        if (!rows_overlap(out, others[i])) continue;
        if (i == own && out.p == others[i].p && out.stride == others[i].stride && out.width == others[i].width) continue;
        OBJ_FAIL(kInvalidInput, action, strf("%s overlaps another tensor", what));
    }
    return 0;
}

namespace dev {

struct NormArgs {
    const void *x, *r, *w;
    void *h, *y, *codes, *scales;
    uint64_t x_stride, r_stride, h_stride, y_stride, code_stride;  // elements
    uint64_t first, n_rows;  // the launch's first row; all rows
    uint32_t width;
    int32_t x_type, r_type, w_type, y_type;
    float offset;
    double eps, inv_width;
};
enum : int { kCodesNone = 0, kCodesInt8 = 1, kCodesFp8 = 2 };

// x / s rounded to the nearest whole number, halves to even, |x / s| < 2^22. The candidate from
// the reciprocal is at most one off, and what it leaves, x - n s, is exact in a float (its bits
// lie between those of s and of s / 2), so comparing twice it with s decides.
__device__ __forceinline__ float whole_quotient(float x, float s, float inv) {
    const float n = __builtin_rintf(x * inv);
    const float twice = 2.0f * __builtin_fmaf(-n, s, x);
    const bool odd = (static_cast<int32_t>(n) & 1) != 0;
    if (twice > s || (twice == s && odd)) return n + 1.0f;
    if (twice < -s || (twice == -s && odd)) return n - 1.0f;
    return n;
}

// 1 / sqrt(m), to an error of some 2^-52: the hardware's estimate (to 2^-23 at least) and two steps
// y + y (e / 2 + 3/8 e^2), e = 1 - m y^2, each of which leaves 5/16 e^3.
__device__ __forceinline__ double inverse_root(double m) {
    double y = __builtin_amdgcn_rsq(m);
    if (!(m > 0.0 && m < __builtin_inf())) return y;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const double e = __builtin_fma(-m * y, y, 1.0);
        y = __builtin_fma(y * e, __builtin_fma(e, 0.375, 0.5), y);
    }
    return y;
}

// A row's total, in every lane: within 16 lanes (WAVES 0) by turning them, over a wave, or over the
// waves of a workgroup.
template <int WAVES, class T, class Op, class Wave>
__device__ __forceinline__ T over_row(T v, Op op, Wave wave, T none, T* shared) {
    if constexpr (WAVES == 0) {
        v = op(v, turned<0x128>(v));
        v = op(v, turned<0x124>(v));
        v = op(v, turned<0x122>(v));
        return op(v, turned<0x121>(v));
    } else {
        v = wave(v);
        if constexpr (WAVES > 1) {
            const uint32_t lane = threadIdx.x & 63;
            if (lane == 0) shared[threadIdx.x >> 6] = v;
            __syncthreads();
            v = wave(lane < WAVES ? shared[lane] : none);
        }
        return v;
    }
}

// ONCE: what is read and the codes are not kept in the caches.
template <int WAVES, int VECS, bool NORM, int CODES, bool ONCE>
__global__ __launch_bounds__(WAVES <= 1 ? 256 : 64 * WAVES, VECS >= 3 ? 4 : 1) void rows_kernel(NormArgs a) {
    constexpr uint32_t kLanes = WAVES == 0 ? 16 : 64 * WAVES;
    constexpr uint32_t kRows = WAVES <= 1 ? 256 / kLanes : 1;  // rows of a workgroup
    // All of a row and its weights asked for at once; with more vectors registers do not hold them.
    constexpr bool kEarly = VECS <= (WAVES <= 8 ? 4 : 2);
    __shared__ double sh_sum[WAVES > 1 ? WAVES : 1];
    __shared__ uint32_t sh_max[WAVES > 1 ? WAVES : 1];
    const uint32_t slot = threadIdx.x % kLanes;
    const uint64_t row = a.first + static_cast<uint64_t>(blockIdx.x) * kRows + (kRows > 1 ? threadIdx.x / kLanes : 0);
    if (row >= a.n_rows) return;  // a row's lanes together

    uint32_t left[VECS];  // elements of each vector that are there
    Raw8 rx[VECS], rr[VECS], rw[VECS];
    float y[VECS][8];
    auto place = [&](int v) { return 8 * (slot + v * kLanes); };
    auto load_x = [&](int v) { rx[v] = !left[v] ? Raw8{} : ONCE ? load_raw8_once(a.x_type, a.x, row * a.x_stride + place(v), left[v]) : load_raw8(a.x_type, a.x, row * a.x_stride + place(v), left[v]); };
    auto load_r = [&](int v) { rr[v] = a.r && left[v] ? load_raw8(a.r_type, a.r, row * a.r_stride + place(v), left[v]) : Raw8{}; };
    auto load_w = [&](int v) { rw[v] = left[v] ? load_raw8(a.w_type, a.w, place(v), left[v]) : Raw8{}; };
    auto add = [&](int v) {
        to_floats(a.x_type, rx[v], y[v]);
        if (NORM && a.r) {
            float r[8];
            to_floats(a.r_type, rr[v], r);
#pragma unroll
            for (int i = 0; i < 8; ++i) y[v][i] += r[i];
        }
    };
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
        left[v] = place(v) < a.width ? (a.width - place(v) < 8 ? a.width - place(v) : 8) : 0;
        load_x(v);
        if constexpr (!kEarly) {
            if (NORM) load_r(v);
            add(v);
        }
    }
    if constexpr (kEarly) {
        if constexpr (NORM) {
#pragma unroll
            for (int v = 0; v < VECS; ++v) load_r(v);
#pragma unroll
            for (int v = 0; v < VECS; ++v) load_w(v);
        }
#pragma unroll
        for (int v = 0; v < VECS; ++v) add(v);
    }

    if constexpr (NORM) {
        double sum = 0.0;
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            if (a.h) {
#pragma unroll
                for (int i = 0; i < 8; ++i) y[v][i] = rounded_to(a.r_type, y[v][i]);
                if (left[v]) store_floats(a.r_type, a.h, row * a.h_stride + place(v), left[v], y[v]);
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) sum = __builtin_fma(static_cast<double>(y[v][i]), static_cast<double>(y[v][i]), sum);
        }
        sum = over_row<WAVES>(sum, [](double p, double q) { return p + q; }, [](double p) { return sum_of_wave(p); }, 0.0, sh_sum);
        const double inv = inverse_root(sum * a.inv_width + a.eps);
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            float w[8];
            if (!kEarly) load_w(v);
            to_floats(a.w_type, rw[v], w);
#pragma unroll
            for (int i = 0; i < 8; ++i)
                y[v][i] = static_cast<float>(static_cast<double>(y[v][i]) * inv *
                                             (static_cast<double>(w[i]) + static_cast<double>(a.offset)));
            if (a.y && left[v]) store_floats(a.y_type, a.y, row * a.y_stride + place(v), left[v], y[v]);
        }
    }

    if constexpr (CODES == kCodesInt8) {
        // The largest magnitude; the bits of magnitudes are in their order, with infinities and
        // NaN above all finite ones.
        uint32_t most = 0;
#pragma unroll
        for (int v = 0; v < VECS; ++v)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t m = static_cast<uint32_t>(i) < left[v] ? __float_as_uint(y[v][i]) & 0x7FFFFFFFu : 0u;
                most = m > most ? m : most;
            }
        most = over_row<WAVES>(most, [](uint32_t p, uint32_t q) { return larger(p, q); }, [](uint32_t p) { return max_of_wave(p); }, 0u, sh_max);
        const bool finite = most < 0x7F800000u;
        float s = finite ? __uint_as_float(most) / 127.0f : __builtin_nanf("");
        if (slot == 0) static_cast<float*>(a.scales)[row] = s;
        // Where s or its reciprocal would be no normal number, both sides are taken 2^64 times.
        const bool tiny = s < 1e-30f, zero = !finite || s == 0.0f;
        const float up = tiny ? 18446744073709551616.0f : 1.0f, inv = 1.0f / (s * up);
        s *= up;
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            // x inv + 1.5 2^23 has the nearest whole number in its last byte. The product is off by less than
            // 127 2^-24; where it comes nearer to a half than that, the quotients are taken exactly.
            constexpr float kWhole = 12582912.0f;
            uint32_t t[8];
            float far = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float n = __builtin_fmaf(y[v][i], inv, kWhole);
                t[i] = __float_as_uint(n);
                far = __builtin_fmaxf(far, __builtin_fabsf(__builtin_fmaf(y[v][i], inv, kWhole - n)));
            }
            if (tiny || far > 0.49999f) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float n = __builtin_fminf(__builtin_fmaxf(whole_quotient(y[v][i] * up, s, inv), -127.0f), 127.0f);
                    t[i] = __float_as_uint(n + kWhole);
                }
            }
            uint32_t c[2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                c[i] = zero ? 0 : __builtin_amdgcn_perm(t[4 * i + 1], t[4 * i], 0x0C0C0400u) | __builtin_amdgcn_perm(t[4 * i + 3], t[4 * i + 2], 0x04000C0Cu);
            uint8_t* to = static_cast<uint8_t*>(a.codes) + row * a.code_stride + place(v);
            if (left[v] == 8) {
                if (ONCE) __builtin_nontemporal_store(any_u32x2{c[0], c[1]}, reinterpret_cast<any_u32x2*>(to));
                else *reinterpret_cast<any_u32x2*>(to) = any_u32x2{c[0], c[1]};
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i)
                    if (i < left[v]) to[i] = static_cast<uint8_t>(c[i / 4] >> (8 * (i % 4)));
            }
        }
    }
    if constexpr (CODES == kCodesFp8) {
        // Sixteen lanes hold a block of 128; its largest magnitude as act_quant takes it (NaN
        // passed over).
#pragma unroll
        for (int v = 0; v < VECS; ++v) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float x = __builtin_fabsf(y[v][i]);
                if (left[v] && x > m) m = x;
            }
            m = over_row<0>(m, [](float p, float q) { return larger(p, q); }, 0, 0.0f, static_cast<float*>(nullptr));
            if (!left[v]) continue;
            const rules::Fp8ActScale sc = rules::fp8_act_scale(m);
            uint32_t c[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 8; ++i) c[i / 4] |= static_cast<uint32_t>(rules::fp8_act_code_short(y[v][i], sc.inv)) << (8 * (i % 4));
            const uint32_t at = place(v);
            *reinterpret_cast<any_u32x2*>(static_cast<uint8_t*>(a.codes) + row * a.code_stride + at) = any_u32x2{c[0], c[1]};
            if ((slot & 15) == 0) static_cast<uint8_t*>(a.scales)[row * (a.width / 128) + at / 128] = sc.raw;
        }
    }
}

}  // namespace dev

using namespace dev;

namespace {

constexpr uint64_t kMaxWidth = 65536;             // a row in the registers of 16 waves, eight vectors a thread
constexpr uint64_t kMaxHidden = 32768;            // four, whose sums and weights take registers too
constexpr uint64_t kGroups = kMostGroups / 4;     // of a launch: they have up to 1024 threads

// Matrices of 64 MiB and more quantized past the caches, held / not, us: 14336 rows of 4096 floats 53.8 / 49.9, in
// bf16 37.3 / 35.3; 4096 of 14336 floats 57.9 / 51.6; beyond 16384 elements a row 2000 of 18432 43.7 / 45.8. A
// norm's codes are read by the next product, and its float rows took longer so (16384 of 1536 39.7 / 42.5).
bool quantized_once(const NormArgs& a) {
    return a.width <= 16384 && a.n_rows * a.width * (a.x_type == kDtF32 ? 4 : 2) >= (uint64_t(64) << 20);
}

template <int WAVES, int VECS, bool NORM>
void launch_shape(hipStream_t s, uint32_t groups, int codes, const NormArgs& a) {
    const dim3 block(WAVES <= 1 ? 256 : 64 * WAVES);
    if constexpr (!NORM) {
        if (WAVES * VECS <= 32 && quantized_once(a)) hipLaunchKernelGGL((rows_kernel<WAVES, VECS, NORM, kCodesInt8, WAVES * VECS <= 32>), dim3(groups), block, 0, s, a);
        else hipLaunchKernelGGL((rows_kernel<WAVES, VECS, NORM, kCodesInt8, false>), dim3(groups), block, 0, s, a);
    } else if (codes == kCodesInt8) hipLaunchKernelGGL((rows_kernel<WAVES, VECS, NORM, kCodesInt8, false>), dim3(groups), block, 0, s, a);
    else if (codes == kCodesFp8) hipLaunchKernelGGL((rows_kernel<WAVES, VECS, NORM, kCodesFp8, false>), dim3(groups), block, 0, s, a);
    else hipLaunchKernelGGL((rows_kernel<WAVES, VECS, NORM, kCodesNone, false>), dim3(groups), block, 0, s, a);
}

// Waves of a row and vectors of a thread. A vector that a row does not fill costs what a full one does,
// so that the smallest shape that holds a row is taken; of rows enough to fill the card those with few
// waves, which wait for one another less (8192 rows of 6144: four waves of three vectors 85 us, sixteen of
// one 105), of fewer rows those with most (32 rows of 4096: eight waves of one 6.2 us, four of two 7.1).
template <bool NORM>
int32_t launch_rows(hipStream_t s, int codes, NormArgs a, const char* action) {
    const uint32_t vectors = (a.width + 7) / 8;
    const bool many = a.n_rows >= 1024;
    const uint64_t rows = vectors <= 32 ? 16 : vectors <= (many ? 128u : 64u) ? 4 : 1;  // of a workgroup
    for (a.first = 0; a.first < a.n_rows; a.first += kGroups * rows) {
        const uint64_t n = (a.n_rows - a.first + rows - 1) / rows;
        const uint32_t g = static_cast<uint32_t>(n < kGroups ? n : kGroups);
        if (vectors <= 16) launch_shape<0, 1, NORM>(s, g, codes, a);
        else if (vectors <= 32) launch_shape<0, 2, NORM>(s, g, codes, a);
        else if (vectors <= 64) launch_shape<1, 1, NORM>(s, g, codes, a);
        else if (vectors <= 128) many ? launch_shape<1, 2, NORM>(s, g, codes, a) : launch_shape<2, 1, NORM>(s, g, codes, a);
        else if (vectors <= 256) launch_shape<4, 1, NORM>(s, g, codes, a);
        else if (vectors <= 512) many ? launch_shape<4, 2, NORM>(s, g, codes, a) : launch_shape<8, 1, NORM>(s, g, codes, a);
        else if (vectors <= 768 && many) launch_shape<4, 3, NORM>(s, g, codes, a);
        else if (vectors <= 1024) many ? launch_shape<8, 2, NORM>(s, g, codes, a) : launch_shape<16, 1, NORM>(s, g, codes, a);
        else if (vectors <= 1536 && many) launch_shape<8, 3, NORM>(s, g, codes, a);
        else if (vectors <= 2048) many ? launch_shape<8, 4, NORM>(s, g, codes, a) : launch_shape<16, 2, NORM>(s, g, codes, a);
        else if (vectors <= 4096) launch_shape<16, 4, NORM>(s, g, codes, a);
        else if constexpr (!NORM) launch_shape<16, 8, NORM>(s, g, codes, a);
        OBJ_HIP(hipGetLastError(), action);
    }
    return 0;
}

}  // namespace

}  // namespace objeta

using namespace objeta;

extern "C" {

int32_t objeta_hip_rms_norm_device(objeta_hip_context* ctx, objeta_hip_stream stream, uint64_t n_tokens, uint64_t hidden,
                                   int32_t dtype, const void* d_x, uint64_t x_stride, int32_t weight_dtype,
                                   const void* d_weight, float weight_offset, double eps, int32_t residual_dtype,
                                   const void* d_residual, uint64_t residual_stride, void* d_residual_out,
                                   uint64_t residual_out_stride, int32_t out_dtype, void* d_out, uint64_t out_stride,
                                   int32_t codes, void* d_codes, uint64_t codes_stride, void* d_scales) {
    OBJ_GUARD_BEGIN
    const char* action = "rms_norm_device";
    OBJ_TRY(check_ctx(ctx, action));
    if (hidden == 0 || hidden > kMaxHidden)
        OBJ_FAIL(kInvalidInput, action, strf("hidden %llu must be 1 to 32768", (unsigned long long)hidden));
    if (!dtype_ok(dtype) || !dtype_ok(weight_dtype)) OBJ_FAIL(kInvalidInput, action, "dtype must be F32, F16 or BF16");
    if ((d_residual || d_residual_out) && !dtype_ok(residual_dtype))
        OBJ_FAIL(kInvalidInput, action, "residual dtype must be F32, F16 or BF16");
    if (d_out && !dtype_ok(out_dtype)) OBJ_FAIL(kInvalidInput, action, "out dtype must be F32, F16 or BF16");
    if (codes < OBJETA_HIP_CODES_NONE || codes > OBJETA_HIP_CODES_FP8)
        OBJ_FAIL(kInvalidInput, action, strf("unknown codes %d", codes));
    if (codes == OBJETA_HIP_CODES_FP8 && hidden % 128)
        OBJ_FAIL(kInvalidInput, action, strf("hidden %llu must be a multiple of 128 for FP8 codes", (unsigned long long)hidden));
    if (!(eps >= 0.0 && eps < 1e300)) OBJ_FAIL(kInvalidInput, action, "eps must be finite and not negative");
    if (!(weight_offset > -1e30f && weight_offset < 1e30f)) OBJ_FAIL(kInvalidInput, action, "weight offset must be finite");
    if (n_tokens >= (uint64_t(1) << 31)) OBJ_FAIL(kInvalidInput, action, "too many tokens");
    if (!d_out && !d_residual_out && codes == OBJETA_HIP_CODES_NONE) OBJ_FAIL(kInvalidInput, action, "no output is given");
    if (n_tokens == 0) return 0;
    const uint64_t n = n_tokens, xs = dtype_size(dtype), rs = dtype_size(residual_dtype), os = dtype_size(out_dtype);
    OBJ_TRY(check_dense_rows(action, "x", d_x, n, x_stride, hidden, xs));
    OBJ_TRY(check_dense_rows(action, "weight", d_weight, 1, 0, hidden, dtype_size(weight_dtype)));
    RowSet in[6] = {row_set(d_x, n, x_stride, hidden, xs), row_set(d_residual, n, residual_stride, hidden, rs),
                    row_set(d_weight, 1, 0, hidden, dtype_size(weight_dtype)), {}, {}, {}};
    int sets = 3;
    if (d_residual) OBJ_TRY(check_dense_rows(action, "residual", d_residual, n, residual_stride, hidden, rs));
    if (d_residual_out) {
        OBJ_TRY(check_dense_rows(action, "residual out", d_residual_out, n, residual_out_stride, hidden, rs));
        const RowSet set = row_set(d_residual_out, n, residual_out_stride, hidden, rs);
        OBJ_TRY(check_dense_apart(action, "residual out", set, in, sets, d_residual ? 1 : -1));
        in[sets++] = set;
    }
    if (d_out) {
        OBJ_TRY(check_dense_rows(action, "out", d_out, n, out_stride, hidden, os));
        const RowSet set = row_set(d_out, n, out_stride, hidden, os);
        OBJ_TRY(check_dense_apart(action, "out", set, in, sets, 0));
        in[sets++] = set;
    }
    if (codes != OBJETA_HIP_CODES_NONE) {
        OBJ_TRY(check_dense_rows(action, "codes", d_codes, n, codes_stride, hidden, 1));
        const uint64_t per = codes == OBJETA_HIP_CODES_INT8 ? 1 : hidden / 128, size = codes == OBJETA_HIP_CODES_INT8 ? 4 : 1;
        OBJ_TRY(check_dense_rows(action, "scales", d_scales, n, per, per, size));
        RowSet set = row_set(d_codes, n, codes_stride, hidden, 1);
        OBJ_TRY(check_dense_apart(action, "codes", set, in, sets, -1));
        in[sets++] = set;
        set = row_set(d_scales, n, per, per, size);
        OBJ_TRY(check_dense_apart(action, "scales", set, in, sets, -1));
    }
    NormArgs a{};
    a.x = d_x, a.r = d_residual, a.w = d_weight, a.h = d_residual_out, a.y = d_out, a.codes = d_codes, a.scales = d_scales;
    a.x_stride = x_stride, a.r_stride = residual_stride, a.h_stride = residual_out_stride, a.y_stride = out_stride;
    a.code_stride = codes_stride;
    a.n_rows = n, a.width = static_cast<uint32_t>(hidden);
    a.x_type = dtype, a.r_type = residual_dtype, a.w_type = weight_dtype, a.y_type = out_dtype;
    a.offset = weight_offset, a.eps = eps, a.inv_width = 1.0 / static_cast<double>(hidden);
    const OnDevice on(ctx->device);
    OBJ_HIP(on.status(), action);
    return launch_rows<true>(resolve_stream(ctx, stream), codes, a, action);
    OBJ_GUARD_END
}

int32_t objeta_hip_quantize_rows_i8_device(objeta_hip_context* ctx, objeta_hip_stream stream, uint64_t n_rows, uint64_t cols,
                                           int32_t dtype, const void* d_x, uint64_t x_stride, int8_t* d_codes,
                                           uint64_t codes_stride, float* d_scales) {
    OBJ_GUARD_BEGIN
    const char* action = "quantize_rows_i8_device";
    OBJ_TRY(check_ctx(ctx, action));
    if (cols == 0 || cols > kMaxWidth)
        OBJ_FAIL(kInvalidInput, action, strf("cols %llu must be 1 to 65536", (unsigned long long)cols));
    if (!dtype_ok(dtype)) OBJ_FAIL(kInvalidInput, action, "dtype must be F32, F16 or BF16");
    if (n_rows >= (uint64_t(1) << 31)) OBJ_FAIL(kInvalidInput, action, "too many rows");
    if (n_rows == 0) return 0;
    OBJ_TRY(check_dense_rows(action, "x", d_x, n_rows, x_stride, cols, dtype_size(dtype)));
    OBJ_TRY(check_dense_rows(action, "codes", d_codes, n_rows, codes_stride, cols, 1));
    OBJ_TRY(check_dense_rows(action, "scales", d_scales, n_rows, 1, 1, 4));
    RowSet sets[2] = {row_set(d_x, n_rows, x_stride, cols, dtype_size(dtype)), row_set(d_codes, n_rows, codes_stride, cols, 1)};
    OBJ_TRY(check_dense_apart(action, "codes", sets[1], sets, 1, -1));
    OBJ_TRY(check_dense_apart(action, "scales", row_set(d_scales, n_rows, 1, 1, 4), sets, 2, -1));
    NormArgs a{};
    a.x = d_x, a.codes = d_codes, a.scales = d_scales;
    a.x_stride = x_stride, a.code_stride = codes_stride;
    a.n_rows = n_rows, a.width = static_cast<uint32_t>(cols), a.x_type = dtype;
    const OnDevice on(ctx->device);
    OBJ_HIP(on.status(), action);
    return launch_rows<false>(resolve_stream(ctx, stream), kCodesInt8, a, action);
    OBJ_GUARD_END
}

}  // extern "C"
