// attn_cached.hip — attention over the paged key/value cache (objeta_hip_attn_cached_device):
// which kernel takes a call, how its keys are cut over workgroups, and the join of the parts.
#include "attn_cached.hpp"
#include "kernels.hpp"

namespace objeta {
namespace dev {

// Joins the parts of one (row, head): with M the largest m, l = sum l_s 2^(m_s - M),
// o = sum o_s 2^(m_s - M) / l. LANES lanes read a part's o, four values each, four parts at a
// time; a wave's lanes hold m, l and weight of 64 parts. WAVES waves take the parts of one
// (row, head): one where there are many of these with few parts each (9280 of up to 8 parts of
// 128: 10.0 us, with four waves 19.3), four otherwise (128 of up to 128 parts: 6.0 us, with one
// 9.6).
template <int QT, int LANES, int WAVES, bool PAGED>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a) {
    typedef typename ElemOf<QT>::type elem;
    constexpr uint32_t kAtOnce = WAVES * 64 / LANES;
    __shared__ f32x4 sh_o[256];
    const uint32_t tid = threadIdx.x, lane = tid & 63;
    const uint64_t rh = static_cast<uint64_t>(blockIdx.x) * (4 / WAVES) + tid / (64 * WAVES);
    const uint32_t row = static_cast<uint32_t>(rh / a.n_heads), head = static_cast<uint32_t>(rh % a.n_heads);
    const uint32_t slot = tid % (64 * WAVES), part = slot / LANES, x = slot % LANES * 4;
    bool any = row < a.n_rows;
    uint32_t n = 0, at_row = 0;
    if constexpr (PAGED) {
        if (any) {
            const RowEntry<false> entry(a.cu, a.seqs, a.n_batch, row);
            any = entry.any && entry.lo >= 0 && static_cast<uint32_t>(entry.hi) <= a.n_rows;
            if (any) {
                const int32_t rows = entry.hi - entry.lo;
                int32_t len = seq_ok(a.kv, entry.seq) ? a.kv.lens[entry.seq] : 0;
                if (!len_ok(a.kv, len) || rows > len || (a.tree && rows > 64)) len = 0;
                n = splits_of(len, a.picked ? *a.picked : a.chunk, a.n_splits);
                at_row = row - static_cast<uint32_t>(entry.lo);
            }
        }
    } else {
        any = any && TokenRange(a.cu, a.n_batch, a.n_rows, static_cast<int32_t>(row)).any;
        if (any) n = a.n_splits;
    }
    const uint64_t step = static_cast<uint64_t>(a.n_rows) * a.n_heads;
    f32x4 v[4], o = {0.0f, 0.0f, 0.0f, 0.0f};
    auto load = [&](uint32_t s0) {
#pragma unroll
        for (uint32_t y = 0; y < 4; ++y) {
            const uint32_t s = s0 + part + y * kAtOnce;
            v[y] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (s < n && x < a.dim) v[y] = *reinterpret_cast<const f32x4*>(a.part + (s * step + rh) * a.dim + x);
        }
    };
    load(0);
    float m = -kInf, l = 0.0f;
    if (lane < n) m = a.part_ml[2 * (lane * step + rh)], l = a.part_ml[2 * (lane * step + rh) + 1];
    float top = m;
    for (uint32_t s = 64 + lane; s < n; s += 64) top = __builtin_fmaxf(top, a.part_ml[2 * (s * step + rh)]);
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) top = __builtin_fmaxf(top, __shfl_xor(top, d, 64));
    const float ref = top == -kInf ? 0.0f : top;
    float sum = 0.0f;
    for (uint32_t base = 0; base < n; base += 64) {
        if (base) {
            const uint64_t at = 2 * ((base + lane) * step + rh);
            m = base + lane < n ? a.part_ml[at] : -kInf, l = base + lane < n ? a.part_ml[at + 1] : 0.0f;
        }
        const float w = exp2_hw(m - ref);
        sum = __builtin_fmaf(l, w, sum);
        const uint32_t end = n - base < 64 ? n : base + 64;
        for (uint32_t s0 = base; s0 < end; s0 += 4 * kAtOnce) {
            if (s0) load(s0);
#pragma unroll
            for (uint32_t y = 0; y < 4; ++y) o += v[y] * __shfl(w, static_cast<int>(s0 - base + part + y * kAtOnce), 64);
        }
    }
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
    sh_o[tid] = o;
    __syncthreads();
    if (!any || part != 0 || x >= a.dim) return;
#pragma unroll
    for (uint32_t p = 1; p < kAtOnce; ++p) o += sh_o[p * LANES + tid];
    if constexpr (PAGED) {  // a row past what max_rows allows for has no parts
        const uint32_t group = a.n_heads / a.n_kv;
        if (static_cast<uint64_t>(at_row) * group + head % group >= static_cast<uint64_t>(a.n_tiles) * a.tile_rows)
            sum = o.x = o.y = o.z = o.w = __builtin_nanf("");
    }
    store_out<QT>(static_cast<elem*>(a.out) + row * a.out_stride + static_cast<uint64_t>(head) * a.dim + x,
                  o * (sum == 0.0f ? 0.0f : 1.0f / sum));
    if (a.lse && x == 0) a.lse[rh] = sum == 0.0f ? -kInf : (top + __builtin_amdgcn_logf(sum)) * kLn2;
}

}  // namespace dev

using namespace dev;

namespace {

template <int QT, int LANES, bool PAGED>
int32_t launch_join_lanes(hipStream_t s, const AttnArgs& a, const char* action) {
    const uint32_t rows = a.n_rows * a.n_heads;
    if (a.n_splits <= 16 && rows >= 4096)
        hipLaunchKernelGGL((attn_join_kernel<QT, LANES, 1, PAGED>), dim3((rows + 3) / 4), dim3(256), 0, s, a);
    else
        hipLaunchKernelGGL((attn_join_kernel<QT, LANES, 4, PAGED>), dim3(rows), dim3(256), 0, s, a);
    OBJ_HIP(hipGetLastError(), action);
    return 0;
}

template <int QT, bool PAGED>
int32_t launch_join(hipStream_t s, const AttnArgs& a, const char* action) {
    if (a.dim <= 64) return launch_join_lanes<QT, 16, PAGED>(s, a, action);
    if (a.dim <= 128) return launch_join_lanes<QT, 32, PAGED>(s, a, action);
    return launch_join_lanes<QT, 64, PAGED>(s, a, action);
}

}  // namespace

int32_t attn_parts(objeta_hip_context* ctx, hipStream_t s, AttnArgs& a) {
    const size_t parts = static_cast<size_t>(a.n_splits) * a.n_rows * a.n_heads;
    void* ws = nullptr;
    OBJ_TRY(ensure_workspace(ctx, s, kWsAttn, parts * (a.dim + 2) * sizeof(float) + sizeof(uint32_t), &ws));
    a.part = static_cast<float*>(ws);
    a.part_ml = a.part + parts * a.dim;
    if (a.pick) a.picked = reinterpret_cast<uint32_t*>(a.part_ml + 2 * parts);
    return 0;
}

int32_t launch_attn_join(hipStream_t s, int32_t dtype, bool paged, const AttnArgs& a, const char* action) {
    if (dtype == kDtF32) return paged ? launch_join<kDtF32, true>(s, a, action) : launch_join<kDtF32, false>(s, a, action);
    if (dtype == kDtF16) return paged ? launch_join<kDtF16, true>(s, a, action) : launch_join<kDtF16, false>(s, a, action);
    return paged ? launch_join<kDtBF16, true>(s, a, action) : launch_join<kDtBF16, false>(s, a, action);
}

}  // namespace objeta

using namespace objeta;

extern "C" {

int32_t objeta_hip_attn_cached_device(objeta_hip_context* ctx, objeta_hip_stream stream,
                                      const objeta_hip_kv_cache* cache, uint64_t layer, const int32_t* d_seqs,
                                      const int32_t* d_cu_rows, uint64_t n_batch, uint64_t n_rows, uint64_t max_rows,
                                      uint64_t max_len, int32_t dtype, const void* d_q, uint64_t q_stride,
                                      uint64_t n_q_heads, const uint64_t* d_tree, float scale, void* d_out,
                                      uint64_t out_stride, float* d_lse) {
    OBJ_GUARD_BEGIN
    const char* action = "attn_cached_device";
    OBJ_TRY(check_ctx(ctx, action));
    OBJ_TRY(check_kv(cache, action));
    const objeta_hip_kv_cache& c = *cache;
    if (layer >= c.n_layers)
        OBJ_FAIL(kInvalidInput, action, strf("layer %llu out of bounds (len=%u)", (unsigned long long)layer, c.n_layers));
    if (!dtype_ok(dtype)) OBJ_FAIL(kInvalidInput, action, "dtype must be F32, F16 or BF16");
    if (dtype != c.dtype && dtype != kDtF32)
        OBJ_FAIL(kUnsupported, action, "q must be float or of the cache's type");
    OBJ_TRY(check_heads(action, n_q_heads, c.n_kv_heads, n_rows, scale));
    if (n_batch > 65535) OBJ_FAIL(kInvalidInput, action, "at most 65535 entries a call");
    if (n_batch == 0 || n_rows == 0) return 0;
    if (!d_seqs || !d_cu_rows) OBJ_FAIL(kInvalidInput, action, "sequences or cu_rows are NULL");
    if (max_rows == 0 || max_len == 0) OBJ_FAIL(kInvalidInput, action, "max_rows and max_len must be positive");
    const uint64_t es = dtype_size(dtype), dim = c.head_dim;
    OBJ_TRY(check_attn_rows(action, "q", d_q, n_rows, q_stride, n_q_heads, dim, es));
    OBJ_TRY(check_attn_rows(action, "out", d_out, n_rows, out_stride, n_q_heads, dim, es));
    if (reinterpret_cast<uintptr_t>(d_lse) % 4 || reinterpret_cast<uintptr_t>(d_tree) % 8)
        OBJ_FAIL(kInvalidInput, action, "lse or tree masks are not aligned");
    const uint64_t pool = static_cast<uint64_t>(c.n_layers) * c.n_pages * c.n_kv_heads * c.page_size * dim * dtype_size(c.dtype);
    const RowSet out{d_out, out_stride * es, n_q_heads * dim * es, n_rows};
    const RowSet lse{d_lse, n_q_heads * 4, n_q_heads * 4, n_rows};
    const RowSet in[] = {{d_q, q_stride * es, n_q_heads * dim * es, n_rows}, {c.k, pool, pool, 1}, {c.v, pool, pool, 1}};
    for (const RowSet& r : in)
        if (rows_overlap(out, r) || rows_overlap(lse, r)) OBJ_FAIL(kInvalidInput, action, "an output overlaps q or the cache");
    if (rows_overlap(out, lse)) OBJ_FAIL(kInvalidInput, action, "out overlaps lse");
    OBJ_HIP(hipSetDevice(ctx->device), "hipSetDevice");

    AttnArgs a{};
    a.q = d_q, a.k = c.k, a.v = c.v, a.out = d_out, a.lse = d_lse;
    a.q_stride = q_stride, a.out_stride = out_stride;
    a.cu = d_cu_rows, a.seqs = d_seqs, a.tree = d_tree;
    a.n_batch = static_cast<uint32_t>(n_batch), a.n_rows = static_cast<uint32_t>(n_rows);
    a.n_heads = static_cast<uint32_t>(n_q_heads), a.n_kv = c.n_kv_heads;
    a.group = a.n_heads / a.n_kv;
    a.dim = c.head_dim;
    a.scale_log2 = scale * kLog2e;
    a.kv = kv_view(c);
    a.layer_off = layer * c.n_pages * c.n_kv_heads * c.page_size * dim;
    a.err = ctx->err_word;
    const hipStream_t s = resolve_stream(ctx, stream);

    // rows of an entry and head; the host's bounds, no more than can be
    const uint64_t rows = (max_rows < n_rows ? max_rows : n_rows) * a.group;
    const uint64_t most = static_cast<uint64_t>(c.max_pages) * c.page_size;
    const uint64_t len = max_len < most ? max_len : most;
    // one wave's 32 rows: each wave reads keys of its own; more: 128 rows share the tiles
    const bool stream_form = rows <= 32;
    a.tile_rows = stream_form ? (rows <= 16 ? 16 : 32) : 128;
    a.n_tiles = static_cast<uint32_t>((rows + a.tile_rows - 1) / a.tile_rows);
    // Keys are cut so that there are about 1024 workgroups if every sequence were the
    // longest, in chunks of at least 256 keys; of two tiles a wave where all workgroups then
    // have a CU to themselves (4000 keys of one sequence, float cache: 14.7 us against 22.4;
    // 30000 keys, which then have not, 46.0 against 37.3).
    const uint64_t units = n_batch * a.n_kv * a.n_tiles;
    uint64_t splits = (1024 + units - 1) / units;
    const uint64_t room = most_parts(n_rows, n_q_heads, dim);
    splits = splits < room ? splits : room;
    const bool float_cache = c.dtype == kDtF32, can_wide = stream_form && a.tile_rows == 16;
    const uint64_t waves = stream_waves(static_cast<int>((dim <= 64 ? 64 : (dim <= 128 ? 128 : 256)) * dtype_size(c.dtype)));
    const uint64_t whole = stream_form ? 64 * waves : 256;
    uint64_t chunk = ((len + splits - 1) / splits + whole - 1) / whole * whole;
    if (chunk < 256 && !(can_wide && units * ((len + whole - 1) / whole) <= 256)) chunk = 256;
    // Few keys, some tiles a wave, stay in one piece: the join costs more than the waves' longer
    // way (bf16, one sequence: 700 keys 10.1 us against 11.5, 1000 11.9 and 11.7; float queries 700
    // 11.8 and 12.6, 1000 14.3 and 12.7; 40 sequences of 300 to 900 14.7 and 18.6, 64 of 300 to 2000
    // 32.2 and 38.8; float cache, one of 130 keys 11.9 and 12.9, of 260 15.6 and 12.9). With a
    // workgroup or more a CU anyway, more keys do (float cache, 100 of 200 to 500: 43 and 54).
    if (stream_form) {
        uint64_t few = 576;
        const uint64_t tiles = float_cache ? 2 : (units < 64 ? 3 : (units < 128 ? 4 : units / 32));
        if (units <= 256 && can_wide) few = 64 * waves * tiles;
        else if (units <= 256) few = 32 * waves * (float_cache ? 2 : 4);
        if (len <= few) chunk = few;
    }
    splits = (len + chunk - 1) / chunk;
    a.wide = can_wide && units * splits <= 256;
    a.chunk = static_cast<uint32_t>(chunk);
    a.n_splits = static_cast<uint32_t>(splits);
    a.pick = !stream_form && splits > 1 && n_batch <= 64;
    if (splits > 1) OBJ_TRY(attn_parts(ctx, s, a));
    OBJ_TRY(stream_form ? launch_attn_stream(s, dtype, c.dtype, static_cast<uint32_t>(rows), a, action)
                        : launch_attn_cached_block(s, dtype, c.dtype, a, action));
    return splits == 1 ? 0 : launch_attn_join(s, dtype, true, a, action);
    OBJ_GUARD_END
}

}  // extern "C"
