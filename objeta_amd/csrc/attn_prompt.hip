// attn_prompt.hip — attention over packed prompts (objeta_hip_attn_prompt_device).
#include "attn_block.hpp"
#include "attn_cached.hpp"
#include "kernels.hpp"

#include <cmath>

namespace objeta {

using namespace dev;

namespace {

// Parts of the keys that a tile of rows sees, so that few tiles fill the card too: the n with
// the least time, counted in cycles (and a tenth less than one part's). A key takes a workgroup
// alone on its CU 0.39 DT cycles in 16 bits, 1.4 DT in float parts, 2.9 DT in float products;
// two a CU take 1.37 times as long, each. A workgroup's setup, and the parts' way through memory
// to the join, are as measured. Sequences are taken to be of their mean length, which is what
// the host knows; a tile may see two of them, and the tiles of a causal one see half of it in
// the mean. Measured, one part and the parts chosen: float, 1530 tokens of 8 over 2 heads of
// 192: 187 us and 116 (2); 777 of 8 heads of 64: 40 and 25 (4); bf16 of 128, causal: 1024 tokens
// of 8 heads 30 and 26 (4), 5000 of 8 over 2 115 and 97 (3); 512 of 32 over 8: 20, with two
// parts 25 (1).
template <int T, int DT>
uint32_t prompt_splits(const AttnArgs& a) {
    constexpr bool two = T != kDtF32 && Block<T, DT>::kPerCu == 2;
    constexpr double each = two ? 1.37 : 1.0;
    constexpr double key = DT * (T != kDtF32 ? 0.39 : (block_type<T, DT> == kDtF32x3 ? 1.4 : 2.9));
    constexpr double setup = T != kDtF32 ? 2000.0 + 62.0 * DT : 8000.0 + 120.0 * DT;
    const uint64_t tiles = static_cast<uint64_t>(a.n_tiles) * a.n_kv, slots = two ? 512 : 256;
    const double mean = static_cast<double>(a.n_rows) / a.n_batch, longest = a.n_batch > 1 ? 2.0 * mean : mean;
    uint32_t best = 1;
    double best_cost = 0.0;
    for (uint32_t n = 1; n <= 8; ++n) {
        const uint64_t items = tiles * n, rest = items % slots;
        const double turns = static_cast<double>(items / slots) * each + (rest ? (rest > 256 ? each : 1.0) : 0.0);
        const double keys = __builtin_fmax(longest * (items > 256 ? 0.5 + 0.5 * each : 1.0), turns * mean * (a.causal ? 0.5 : 1.0));
        const double join = n > 1 ? 12000.0 + 0.4 * DT * items : 0.0;
        const double cost = key * keys / n + setup * ((items + slots - 1) / slots) + join;
        if (n == 1 || cost < (best == 1 ? 0.9 : 1.0) * best_cost) best = n, best_cost = cost;
    }
    return best;
}

template <int T, int DT>
int32_t launch_prompt(objeta_hip_context* ctx, hipStream_t s, AttnArgs& a, const char* action) {
    const uint64_t room = most_parts(a.n_rows, a.n_heads, a.dim);
    a.n_splits = prompt_splits<T, DT>(a);
    if (a.n_splits > room) a.n_splits = static_cast<uint32_t>(room);
    if (a.n_splits > 1) OBJ_TRY(attn_parts(ctx, s, a));
    const uint64_t groups = static_cast<uint64_t>(a.n_tiles) * a.n_splits * a.n_kv;
    OBJ_TRY(launch_groups(attn_block_kernel<T, block_type<T, DT>, DT, false>, groups, 256, s, a, action));
    return a.n_splits > 1 ? launch_attn_join(s, T, false, a, action) : 0;
}

template <int T>
int32_t launch_prompt_dim(objeta_hip_context* ctx, hipStream_t s, AttnArgs& a, const char* action) {
    if (a.dim <= 64) return launch_prompt<T, 64>(ctx, s, a, action);
    if (a.dim <= 96) return launch_prompt<T, 96>(ctx, s, a, action);
    if (a.dim <= 128) return launch_prompt<T, 128>(ctx, s, a, action);
    if (a.dim <= 192) return launch_prompt<T, 192>(ctx, s, a, action);
    return launch_prompt<T, 256>(ctx, s, a, action);
}

}  // namespace

int32_t check_attn_rows(const char* action, const char* what, const void* p, uint64_t n, uint64_t stride, uint64_t heads,
                        uint64_t dim, uint64_t size) {
    if (!p) OBJ_FAIL(kInvalidInput, action, strf("%s is NULL", what));
    if (!extent_ok(n, stride, heads * dim, size)) OBJ_FAIL(kInvalidInput, action, strf("%s is too large", what));
    if (n > 1 && stride < heads * dim)
        OBJ_FAIL(kInvalidInput, action,
                 strf("%s stride %llu is less than its %llu elements", what, (unsigned long long)stride,
                      (unsigned long long)(heads * dim)));
    if (reinterpret_cast<uintptr_t>(p) % 16 || (n > 1 && stride * size % 16))
        OBJ_FAIL(kInvalidInput, action, strf("%s rows must be 16-byte aligned", what));
    return 0;
}

int32_t check_heads(const char* action, uint64_t n_q_heads, uint64_t n_kv_heads, uint64_t n_rows, float scale) {
    if (n_q_heads == 0 || n_kv_heads == 0 || n_q_heads > 65535 || n_q_heads % n_kv_heads)
        OBJ_FAIL(kInvalidInput, action,
                 strf("n_q_heads %llu must be a multiple of n_kv_heads %llu, at most 65535",
                      (unsigned long long)n_q_heads, (unsigned long long)n_kv_heads));
    if (n_rows > kMaxTokens || n_rows * n_q_heads > kMaxTokens)
        OBJ_FAIL(kInvalidInput, action, "rows times heads must not exceed 2^31 - 2^16");
    if (!(std::isfinite(scale) && scale > 0.0f)) OBJ_FAIL(kInvalidInput, action, "scale must be positive and finite");
    return 0;
}

}  // namespace objeta

using namespace objeta;

extern "C" {

int32_t objeta_hip_attn_prompt_device(objeta_hip_context* ctx, objeta_hip_stream stream, int32_t dtype,
                                      const void* d_q, uint64_t q_stride, uint64_t n_q_heads, const void* d_k,
                                      uint64_t k_stride, const void* d_v, uint64_t v_stride, uint64_t n_kv_heads,
                                      uint64_t head_dim, uint64_t n_tokens, const int32_t* d_cu_seqlens,
                                      uint64_t n_seqs, int32_t causal, float scale, void* d_out, uint64_t out_stride,
                                      float* d_lse) {
    OBJ_GUARD_BEGIN
    const char* action = "attn_prompt_device";
    OBJ_TRY(check_ctx(ctx, action));
    if (!dtype_ok(dtype)) OBJ_FAIL(kInvalidInput, action, "dtype must be F32, F16 or BF16");
    if (!head_dim_ok(head_dim))
        OBJ_FAIL(kInvalidInput, action, strf("head_dim %llu must be a multiple of 8 up to 256", (unsigned long long)head_dim));
    OBJ_TRY(check_heads(action, n_q_heads, n_kv_heads, n_tokens, scale));
    if (n_seqs >= (uint64_t(1) << 31)) OBJ_FAIL(kInvalidInput, action, "too many sequences");
    if (n_tokens == 0 || n_seqs == 0) return 0;
    if (!d_cu_seqlens) OBJ_FAIL(kInvalidInput, action, "cu_seqlens are NULL");
    const uint64_t es = dtype_size(dtype);
    // one row has no next one: its strides may be anything, and the kernels take a row's stride
    // for the bytes that there are to read
    if (n_tokens == 1) {
        q_stride = out_stride = n_q_heads * head_dim;
        k_stride = v_stride = n_kv_heads * head_dim;
    }
    OBJ_TRY(check_attn_rows(action, "q", d_q, n_tokens, q_stride, n_q_heads, head_dim, es));
    OBJ_TRY(check_attn_rows(action, "k", d_k, n_tokens, k_stride, n_kv_heads, head_dim, es));
    OBJ_TRY(check_attn_rows(action, "v", d_v, n_tokens, v_stride, n_kv_heads, head_dim, es));
    OBJ_TRY(check_attn_rows(action, "out", d_out, n_tokens, out_stride, n_q_heads, head_dim, es));
    if (k_stride > kMaxKvStride || v_stride > kMaxKvStride)
        OBJ_FAIL(kInvalidInput, action, strf("k and v strides must not exceed %llu", (unsigned long long)kMaxKvStride));
    const RowSet out{d_out, out_stride * es, n_q_heads * head_dim * es, n_tokens};
    const RowSet in[] = {{d_q, q_stride * es, n_q_heads * head_dim * es, n_tokens},
                         {d_k, k_stride * es, n_kv_heads * head_dim * es, n_tokens},
                         {d_v, v_stride * es, n_kv_heads * head_dim * es, n_tokens},
                         {d_lse, n_q_heads * 4, n_q_heads * 4, n_tokens}};
    for (const RowSet& r : in)
        if (rows_overlap(out, r)) OBJ_FAIL(kInvalidInput, action, "out overlaps q, k, v or lse");
    for (int i = 0; i < 3; ++i)
        if (rows_overlap(in[3], in[i])) OBJ_FAIL(kInvalidInput, action, "lse overlaps q, k or v");
    if (reinterpret_cast<uintptr_t>(d_lse) % 4) OBJ_FAIL(kInvalidInput, action, "lse is not aligned");
    OBJ_HIP(hipSetDevice(ctx->device), "hipSetDevice");
    AttnArgs a{};
    a.q = d_q, a.k = d_k, a.v = d_v, a.out = d_out, a.lse = d_lse;
    a.q_stride = q_stride, a.k_stride = k_stride, a.v_stride = v_stride, a.out_stride = out_stride;
    a.cu = d_cu_seqlens;
    a.n_batch = static_cast<uint32_t>(n_seqs);
    a.n_rows = static_cast<uint32_t>(n_tokens);
    a.n_heads = static_cast<uint32_t>(n_q_heads), a.n_kv = static_cast<uint32_t>(n_kv_heads);
    a.group = a.n_heads / a.n_kv;
    a.dim = static_cast<uint32_t>(head_dim);
    a.scale_log2 = scale * kLog2e;
    a.causal = causal;
    a.n_tiles = static_cast<uint32_t>((n_tokens * a.group + 127) / 128);
    a.err = ctx->err_word;
    const hipStream_t s = resolve_stream(ctx, stream);
    if (dtype == kDtF32) return launch_prompt_dim<kDtF32>(ctx, s, a, action);
    if (dtype == kDtF16) return launch_prompt_dim<kDtF16>(ctx, s, a, action);
    return launch_prompt_dim<kDtBF16>(ctx, s, a, action);
    OBJ_GUARD_END
}

}  // extern "C"
