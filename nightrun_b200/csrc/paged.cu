// Rotary append and eviction over a paged KV cache.
#include "paged.cuh"

namespace nrc {
namespace {

__device__ unsigned g_paged_err;

// ------------------------------------------------------------ rotary append
// One thread per (token, head, pair): the pair's angle pos * freq is formed in 64 bits and reduced
// to a fraction of a turn there (a far position's angle has no correct digit left in 32 bits past
// 2^24 turns), its sine and cosine in f32.
__global__ void k_rope_append_paged(const RopeAppendArgs a) {
  const uint32_t hd = a.kv.head_dim, half_hd = hd / 2, nh = a.n_heads + 2 * a.kv.n_kv_heads;
  const size_t total = (size_t)a.tokens * nh * half_hd;
  for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (size_t)gridDim.x * blockDim.x) {
    const uint32_t pr = i % half_hd;
    const size_t th = i / half_hd;
    const uint32_t h = th % nh, t = th / nh;
    const uint32_t half = a.rot_dim / 2;
    const bool rotate = pr < half && h < a.n_heads + a.kv.n_kv_heads;
    // Pairs from rot_dim on are neighbours that pass unchanged.
    uint32_t ia, ib;
    if (pr < half && a.style == 1)
      ia = pr, ib = pr + half;
    else
      ia = 2 * pr, ib = 2 * pr + 1;
    const bool is_q = h < a.n_heads, is_k = !is_q && h < a.n_heads + a.kv.n_kv_heads;
    const uint32_t kh = is_q ? 0 : is_k ? h - a.n_heads : h - a.n_heads - a.kv.n_kv_heads;
    const void* src = is_q ? a.q : is_k ? a.k : a.v;
    const int64_t so = is_q   ? (int64_t)t * a.q_token + (int64_t)h * a.q_head
                       : is_k ? (int64_t)t * a.k_token + (int64_t)kh * a.k_head
                              : (int64_t)t * a.v_token + (int64_t)kh * a.v_head;
    float x = load_as_f32(src, so + ia, a.dtype), y = load_as_f32(src, so + ib, a.dtype);
    if (rotate) {
      const double turns = (double)a.pos[t] * (double)a.freqs[pr] * 0.15915494309189533577;
      float c, s;
      sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
      c *= a.mscale;
      s *= a.mscale;
      const float u = x * c - y * s, w = x * s + y * c;
      x = u;
      y = w;
    }
    if (is_q) {
      const int64_t o = (int64_t)t * a.qo_token + (int64_t)h * a.qo_head;
      store_from_f32(a.q_out, o + ia, a.dtype, x);
      store_from_f32(a.q_out, o + ib, a.dtype, y);
    } else {
      const int32_t slot = a.slot[t], seq = a.seq[t];
      if (slot < 0) continue;
      if (seq < 0 || (uint32_t)seq >= a.kv.n_seqs || (uint32_t)slot / a.kv.page_size >= a.kv.max_pages) {
        atomicOr(&g_paged_err, ERR_BAD_SLOT);
        continue;
      }
      const int64_t row = paged_row(a.kv, seq, slot);
      if (row < 0) {
        atomicOr(&g_paged_err, ERR_BAD_PAGE);
        continue;
      }
      void* dst = is_k ? a.kv.k : a.kv.v;
      const int64_t o = row + (int64_t)kh * a.kv.head_stride;
      store_from_f32(dst, o + ia, a.kv.dtype, x);
      store_from_f32(dst, o + ib, a.kv.dtype, y);
    }
  }
}

// ------------------------------------------------------------ eviction
constexpr int EV_THREADS = 1024;

// Weights ordered as unsigned keys: larger weight, larger key; both zeros alike; NaN the smallest.
NRC_DEV uint32_t weight_key(float v) {
  if (v != v) return 0u;
  const uint32_t b = __float_as_uint(v == 0.0f ? 0.0f : v);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

NRC_DEV uint32_t block_sum(uint32_t v, uint32_t* red) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if (lane == 0) red[warp] = v;
  __syncthreads();
  uint32_t s = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) s += red[w];
  return s;
}

// Exclusive prefix sum of v over the block; *total its sum.
NRC_DEV uint32_t block_scan(uint32_t v, uint32_t* red, uint32_t* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  uint32_t before = 0, all = 0;
  for (int w = 0; w < (int)(blockDim.x >> 5); w++) {
    if (w < warp) before += red[w];
    all += red[w];
  }
  *total = all;
  return before + x - v;
}

// The sequence's length, at most what its table and the weights hold.
NRC_DEV uint32_t evict_len(const EvictArgs& a, uint32_t b) {
  const int32_t raw = a.lens[b];
  const uint64_t slots = (uint64_t)a.kv.max_pages * a.kv.page_size;
  const uint32_t most = (uint32_t)(slots < a.weights_len ? slots : a.weights_len);
  if (raw < 0 || (uint32_t)raw > most) {
    if (threadIdx.x == 0) atomicOr(&g_paged_err, ERR_BAD_SLOT);
    return raw < 0 ? 0u : most;
  }
  return (uint32_t)raw;
}

// One CTA per (sequence, KV head): the key of the last position kept by its weight, found bit by bit
// from the top (the largest key that at least `want` keys reach); then one pass in position order
// writes the kept slots and their weights.
__global__ void __launch_bounds__(EV_THREADS) k_evict_select(const EvictArgs a) {
  __shared__ uint32_t red[32];
  const uint32_t h = blockIdx.x, b = blockIdx.y;
  const size_t row = (size_t)b * a.kv.n_kv_heads + h;
  const uint32_t n = evict_len(a, b);
  const float* w = a.weights + row * a.weights_len;
  float* nw = a.new_weights + row * a.weights_len;
  int32_t* kept = a.kept + row * a.budget;
  const uint32_t lo = a.sinks, hi = n > a.budget ? n - a.recent : n;  // chosen by weight: [lo, hi)
  uint32_t key = 0, ties = 0;
  if (n > a.budget) {
    const uint32_t want = a.budget - a.sinks - a.recent;
    if (want == 0) {
      key = 0xffffffffu;  // no weight's key
    } else {
      for (int bit = 31; bit >= 0; bit--) {
        const uint32_t probe = key | (1u << bit);
        uint32_t c = 0;
        for (uint32_t t = lo + threadIdx.x; t < hi; t += EV_THREADS) c += weight_key(w[t]) >= probe;
        if (block_sum(c, red) >= want) key = probe;
      }
      uint32_t c = 0;
      for (uint32_t t = lo + threadIdx.x; t < hi; t += EV_THREADS) c += weight_key(w[t]) > key;
      ties = want - block_sum(c, red);
    }
  }
  uint32_t at = 0, tied = 0;
  for (uint32_t t0 = 0; t0 < n; t0 += EV_THREADS) {
    const uint32_t t = t0 + threadIdx.x;
    bool keep = false, tie = false;
    float v = 0.0f;
    if (t < n) {
      v = w[t];
      if (n <= a.budget || t < lo || t >= hi) {
        keep = true;
      } else {
        const uint32_t k = weight_key(v);
        keep = k > key;
        tie = k == key;
      }
    }
    uint32_t all;
    const uint32_t nth = tied + block_scan(tie, red, &all);
    tied += all;
    keep = keep || (tie && nth < ties);
    const uint32_t to = at + block_scan(keep, red, &all);  // its barriers: w[t0..] is read before nw is written
    at += all;
    if (keep) {
      kept[to] = (int32_t)t;
      nw[to] = v;
    }
  }
  for (uint32_t i = at + threadIdx.x; i < a.budget; i += EV_THREADS) kept[i] = -1;
  __syncthreads();
  for (uint32_t i = at + threadIdx.x; i < a.weights_len; i += EV_THREADS) nw[i] = 0.0f;
}

// One CTA per (sequence, KV head, K or V): rows move down to their new slots in ascending order.
// Slot i receives slot kept[i] >= i, so a batch of rows that is read whole before it is written
// overwrites nothing that a later batch reads.
__global__ void __launch_bounds__(EV_THREADS) k_evict_move(const EvictArgs a) {
  const uint32_t h = blockIdx.x, b = blockIdx.y;
  const int32_t* kept = a.kept + ((size_t)b * a.kv.n_kv_heads + h) * a.budget;
  uint16_t* base = static_cast<uint16_t*>(blockIdx.z ? a.kv.v : a.kv.k) + (int64_t)h * a.kv.head_stride;
  const uint32_t vecs = a.kv.head_dim / 8, rows = EV_THREADS / vecs;
  const uint32_t r = threadIdx.x / vecs, c = threadIdx.x % vecs;
  for (uint32_t i0 = 0; i0 < a.budget; i0 += rows) {
    const uint32_t i = i0 + r;
    const int32_t src = r < rows && i < a.budget ? kept[i] : -1;
    uint4 x;
    int64_t to = -1;
    if (src >= 0) {
      if ((uint32_t)src != i) {
        const int64_t from = paged_row(a.kv, b, src);
        to = paged_row(a.kv, b, i);
        if (from < 0 || to < 0) {
          atomicOr(&g_paged_err, ERR_BAD_PAGE);
          to = -1;
        } else {
          x = reinterpret_cast<const uint4*>(base + from)[c];
        }
      }
    }
    __syncthreads();
    if (to >= 0) reinterpret_cast<uint4*>(base + to)[c] = x;
  }
  // new_lens may be lens: only this thread still reads that element.
  if (h == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
    const uint32_t n = evict_len(a, b);
    a.new_lens[b] = (int32_t)(n < a.budget ? n : a.budget);
  }
}

}  // namespace

cudaError_t rope_append_paged_run(const RopeAppendArgs& a, cudaStream_t s) {
  const size_t total = (size_t)a.tokens * (a.n_heads + 2 * a.kv.n_kv_heads) * (a.kv.head_dim / 2);
  const size_t blocks = (total + 255) / 256;
  k_rope_append_paged<<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t kv_evict_run(const EvictArgs& a, cudaStream_t s) {
  k_evict_select<<<dim3(a.kv.n_kv_heads, a.kv.n_seqs), EV_THREADS, 0, s>>>(a);
  if (cudaError_t e = cudaGetLastError()) return e;
  k_evict_move<<<dim3(a.kv.n_kv_heads, a.kv.n_seqs, 2), EV_THREADS, 0, s>>>(a);
  return cudaGetLastError();
}

cudaError_t paged_take_errors(unsigned* bits) {
  cudaError_t e = cudaMemcpyFromSymbol(bits, g_paged_err, sizeof(unsigned));
  const unsigned zero = 0;
  if (e == cudaSuccess && *bits) e = cudaMemcpyToSymbol(g_paged_err, &zero, sizeof zero);
  return e;
}

}  // namespace nrc
