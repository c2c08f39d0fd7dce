// attn_cached_block.hip — the instances of attn_block.hpp for the paged cache, by types and head size.
#include "attn_cached.hpp"
#include "attn_block.hpp"

namespace objeta {

using namespace dev;

namespace {

template <int Q, int K, int DT>
int32_t launch(hipStream_t s, const AttnArgs& a, const char* action) {
    // tiles that there can be: of every entry as many as the longest one's, and no more than all
    // rows fill and one that is not full for every entry with rows
    const uint64_t most = static_cast<uint64_t>(a.n_batch) * a.n_tiles, with_rows = a.n_batch < a.n_rows ? a.n_batch : a.n_rows;
    const uint64_t full = static_cast<uint64_t>(a.n_rows) * a.group / 128 + with_rows, tiles = full < most ? full : most;
    return launch_groups(attn_block_kernel<Q, block_type<K, DT>, DT, true>, tiles * a.n_splits * a.n_kv, 256, s, a, action);
}

template <int Q, int K>
int32_t launch_dim(hipStream_t s, const AttnArgs& a, const char* action) {
    if (a.dim <= 64) return launch<Q, K, 64>(s, a, action);
    if (a.dim <= 96) return launch<Q, K, 96>(s, a, action);
    if (a.dim <= 128) return launch<Q, K, 128>(s, a, action);
    if (a.dim <= 192) return launch<Q, K, 192>(s, a, action);
    return launch<Q, K, 256>(s, a, action);
}

}  // namespace

int32_t launch_attn_cached_block(hipStream_t s, int32_t q_type, int32_t kv_type, const AttnArgs& a, const char* action) {
    if (q_type == kDtF16) return launch_dim<kDtF16, kDtF16>(s, a, action);
    if (q_type == kDtBF16) return launch_dim<kDtBF16, kDtBF16>(s, a, action);
    if (kv_type == kDtF32) return launch_dim<kDtF32, kDtF32>(s, a, action);
    if (kv_type == kDtF16) return launch_dim<kDtF32, kDtF16>(s, a, action);
    return launch_dim<kDtF32, kDtBF16>(s, a, action);
}

}  // namespace objeta
