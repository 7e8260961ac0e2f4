// Attention of the newest tokens of many sequences over a paged KV cache.
#include "paged.cuh"

namespace nrc {
namespace {

__device__ unsigned g_attn_err;

constexpr int PA_THREADS = 128, PA_WARPS = PA_THREADS / 32;

// One CTA per (KV head, sequence): for each query row one pass over the positions, a warp per
// position, with the running maximum and sum of the softmax; where weights are wanted a second pass
// adds them in row order.
template <int PER>  // head_dim / 32
__global__ void __launch_bounds__(PA_THREADS) k_paged_attn(const PagedAttnArgs a) {
  constexpr int HD = 32 * PER;
  __shared__ float sm[PA_WARPS], sl[PA_WARPS], so[PA_WARPS][HD];
  const uint32_t h = blockIdx.x, b = blockIdx.y;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t gqa = a.n_heads / a.kv.n_kv_heads;
  const int32_t raw = a.lens[b];
  uint32_t len = raw < 0 ? 0u : (uint32_t)raw;
  const uint32_t most = a.weights && a.weights_len < a.max_len ? a.weights_len : a.max_len;
  if (raw < 0 || len > most) {
    if (threadIdx.x == 0) atomicOr(&g_attn_err, ERR_BAD_SLOT);
    len = raw < 0 ? 0u : most;
  }
  const uint16_t* kb = static_cast<const uint16_t*>(a.kv.k) + (int64_t)h * a.kv.head_stride;
  const uint16_t* vb = static_cast<const uint16_t*>(a.kv.v) + (int64_t)h * a.kv.head_stride;
  for (uint32_t r = 0; r < gqa * a.n_new; r++) {
    const uint32_t tok = r / gqa, head = h * gqa + r % gqa;
    const int64_t sees = (int64_t)len - (a.n_new - 1 - tok);
    const uint32_t n = sees > 0 ? (uint32_t)sees : 0u;
    float q[PER], acc[PER], m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < PER; i++) {
      q[i] = load_as_f32(a.q, (int64_t)b * a.q_seq + (int64_t)tok * a.q_token + (int64_t)head * a.q_head + lane + 32 * i,
                         a.dtype);
      acc[i] = 0.0f;
    }
    auto score = [&](uint32_t t, int64_t* row) {
      *row = paged_row(a.kv, b, t);
      if (*row < 0) {
        if (lane == 0) atomicOr(&g_attn_err, ERR_BAD_PAGE);
        return -INFINITY;
      }
      float s = 0.0f;
#pragma unroll
      for (int i = 0; i < PER; i++) s += q[i] * load_as_f32(kb, *row + lane + 32 * i, a.kv.dtype);
      return warp_sum(s) * a.scale;
    };
    for (uint32_t t = warp; t < n; t += PA_WARPS) {
      int64_t row;
      const float s = score(t, &row);
      if (row < 0 || s == -INFINITY) continue;
      const float mn = fmaxf(m, s), old = expf(m - mn), p = expf(s - mn);
      l = l * old + p;
#pragma unroll
      for (int i = 0; i < PER; i++) acc[i] = acc[i] * old + p * load_as_f32(vb, row + lane + 32 * i, a.kv.dtype);
      m = mn;
    }
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int i = 0; i < PER; i++) so[warp][lane + 32 * i] = acc[i];
    __syncthreads();
    float mx = -INFINITY, total = 0.0f;
    for (int w = 0; w < PA_WARPS; w++) mx = fmaxf(mx, sm[w]);
    for (int w = 0; w < PA_WARPS; w++) total += sl[w] == 0.0f ? 0.0f : sl[w] * expf(sm[w] - mx);
    const float inv = total == 0.0f ? 0.0f : 1.0f / total;
    for (int d = threadIdx.x; d < HD; d += PA_THREADS) {
      float o = 0.0f;
      for (int w = 0; w < PA_WARPS; w++) o += sl[w] == 0.0f ? 0.0f : so[w][d] * expf(sm[w] - mx);
      store_from_f32(a.out, (int64_t)b * a.o_seq + (int64_t)tok * a.o_token + (int64_t)head * a.o_head + d, a.dtype,
                     o * inv);
    }
    if (a.weights) {
      float* wr = a.weights + ((size_t)b * a.kv.n_kv_heads + h) * a.weights_len;
      for (uint32_t t = warp; t < n; t += PA_WARPS) {  // a position stays with its warp in every row
        int64_t row;
        const float s = score(t, &row);
        if (lane == 0 && row >= 0 && s != -INFINITY) wr[t] += expf(s - mx) * inv;
      }
    }
    __syncthreads();
  }
}

}  // namespace

size_t paged_attn_workspace(const nrc_paged_kv&, uint32_t, uint32_t, bool, uint32_t) { return 0; }

cudaError_t paged_attn_run(const PagedAttnArgs& a, cudaStream_t s) {
  PagedAttnArgs aa = a;
  void* args[] = {&aa};
  const void* fn = nullptr;
  switch (a.kv.head_dim) {
    case 32: fn = (const void*)k_paged_attn<1>; break;
    case 64: fn = (const void*)k_paged_attn<2>; break;
    case 96: fn = (const void*)k_paged_attn<3>; break;
    case 128: fn = (const void*)k_paged_attn<4>; break;
    default: return cudaErrorInvalidValue;
  }
  return launch_kernel(fn, dim3(a.kv.n_kv_heads, a.kv.n_seqs), dim3(PA_THREADS), 0, s, false, args);
}

cudaError_t paged_attn_take_errors(unsigned* bits) {
  cudaError_t e = cudaMemcpyFromSymbol(bits, g_attn_err, sizeof(unsigned));
  const unsigned zero = 0;
  if (e == cudaSuccess && *bits) e = cudaMemcpyToSymbol(g_attn_err, &zero, sizeof zero);
  return e;
}

}  // namespace nrc
