// Attention of few query rows over the cache in 8 bits (kv_attn_rows.cuh).
#include "kv_attn_rows.cuh"

namespace kd {

cudaError_t launch_attention_rows8(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream) {
  return by_head_dim(c.D, [&](auto dim) { return launch_rows_dim<8, decltype(dim)::value>(c, s, p, a, ws, stream); });
}

cudaError_t launch_attention_weights8(const kd_cache& c, const kd_cache_seqs& s, const kd_cache_queries& p, const AttnShape& a, const AttnWorkspace& ws, cudaStream_t stream) {
  return by_head_dim(c.D, [&](auto dim) { return launch_weights_dim<8, decltype(dim)::value>(c, s, p, a, ws, stream); });
}

}  // namespace kd
