// Paged attention over a bf16 cache, queries and weights in 3 part(s).
#include "paged_attn_tc.cuh"

namespace nrc {
cudaError_t paged_attn_bf16_3(pattn::Plan& p, int nt, cudaStream_t s) { return pattn::launch_hd<true, 3>(p, nt, s); }
}  // namespace nrc
