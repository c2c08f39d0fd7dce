// attn_cached_stream.hip — the instances of attn_stream.hpp for the paged cache, by types and head size.
#include "attn_cached.hpp"
#include "attn_stream.hpp"

namespace objeta {

using namespace dev;

namespace {

template <int Q, int K, int DT, int ROWS, bool WIDE>
int32_t launch(hipStream_t s, const AttnArgs& a, const char* action) {
    const uint64_t groups = static_cast<uint64_t>(a.n_splits) * a.n_batch * a.n_kv;
    return launch_groups(attn_stream_kernel<Q, K, DT, ROWS, WIDE>, (groups + 7) / 8 * 8, 64 * Stream<K, DT, ROWS, WIDE>::kWaves, s, a,
                         action);
}

template <int Q, int K, int ROWS, bool WIDE>
int32_t launch_rows(hipStream_t s, const AttnArgs& a, const char* action) {
    if (a.dim <= 64) return launch<Q, K, 64, ROWS, WIDE>(s, a, action);
    if (a.dim <= 128) return launch<Q, K, 128, ROWS, WIDE>(s, a, action);
    return launch<Q, K, 256, ROWS, WIDE>(s, a, action);
}

template <int Q, int K>
int32_t launch_dim(hipStream_t s, uint32_t rows, const AttnArgs& a, const char* action) {
    if (rows > 16) return launch_rows<Q, K, 32, false>(s, a, action);
    return a.wide ? launch_rows<Q, K, 16, true>(s, a, action) : launch_rows<Q, K, 16, false>(s, a, action);
}

}  // namespace

int32_t launch_attn_stream(hipStream_t s, int32_t q_type, int32_t kv_type, uint32_t rows, const AttnArgs& a, const char* action) {
    if (q_type == kDtF16) return launch_dim<kDtF16, kDtF16>(s, rows, a, action);
    if (q_type == kDtBF16) return launch_dim<kDtBF16, kDtBF16>(s, rows, a, action);
    if (kv_type == kDtF32) return launch_dim<kDtF32, kDtF32>(s, rows, a, action);
    if (kv_type == kDtF16) return launch_dim<kDtF32, kDtF16>(s, rows, a, action);
    return launch_dim<kDtF32, kDtBF16>(s, rows, a, action);
}

}  // namespace objeta
