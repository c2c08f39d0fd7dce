// attn_cached.hpp — the checks and launchers that both attentions' entry points use.
#pragma once

#include "attn_tile.hpp"

namespace objeta {

// Rows of 16-byte alignment, and heads, rows and scale in range (attn_prompt.hip).
int32_t check_attn_rows(const char* action, const char* what, const void* p, uint64_t n, uint64_t stride, uint64_t heads,
                        uint64_t dim, uint64_t size);
int32_t check_heads(const char* action, uint64_t n_q_heads, uint64_t n_kv_heads, uint64_t n_rows, float scale);
// The most parts that keep their workspace within 1 GiB: rows that belong to no sequence count too,
// and a batch padded far would ask for more than it uses.
inline uint64_t most_parts(uint64_t n_rows, uint64_t n_heads, uint64_t dim) {
    const uint64_t most = (uint64_t(1) << 30) / (n_rows * n_heads * (dim + 2) * sizeof(float));
    return most < 1 ? 1 : most;
}
// `n` workgroups of `kernel` in as many launches as they need.
template <class Kernel>
int32_t launch_groups(Kernel kernel, uint64_t n, uint32_t threads, hipStream_t s, dev::AttnArgs a, const char* action) {
    if (n > 0x7FFFFFFFull) OBJ_FAIL(kInvalidInput, action, "too many workgroups");
    for (uint64_t first = 0; first < n; first += kMostGroups) {
        a.first = static_cast<uint32_t>(first);
        const uint32_t now = static_cast<uint32_t>(n - first < kMostGroups ? n - first : kMostGroups);
        hipLaunchKernelGGL(kernel, dim3(now), dim3(threads), 0, s, a);
        OBJ_HIP(hipGetLastError(), action);
    }
    return 0;
}
// Workspace for the parts of a call of several splits, and their join (attn_cached.hip).
int32_t attn_parts(objeta_hip_context* ctx, hipStream_t s, dev::AttnArgs& a);
int32_t launch_attn_join(hipStream_t s, int32_t dtype, bool paged, const dev::AttnArgs& a, const char* action);
// Tiles of 16 rows (rows <= 16) or 32.
int32_t launch_attn_stream(hipStream_t s, int32_t q_type, int32_t kv_type, uint32_t rows, const dev::AttnArgs& a,
                           const char* action);
int32_t launch_attn_cached_block(hipStream_t s, int32_t q_type, int32_t kv_type, const dev::AttnArgs& a,
                                 const char* action);

}  // namespace objeta
