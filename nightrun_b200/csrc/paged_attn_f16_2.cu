// Paged attention over a f16 cache, queries and weights in 2 part(s).
#include "paged_attn_tc.cuh"

namespace nrc {
cudaError_t paged_attn_f16_2(pattn::Plan& p, int nt, cudaStream_t s) { return pattn::launch_hd<false, 2>(p, nt, s); }
}  // namespace nrc
