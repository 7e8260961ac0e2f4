// Rotary append and eviction over a paged KV cache.
#include "paged.cuh"

namespace nrc {
namespace {

__device__ unsigned g_paged_err;

// ------------------------------------------------------------ rotary append
// y = mscale R(pos f) x on pairs of q and k, v as it is. One pass over the values: bound by HBM for many
// tokens, by latency for few.
//
// A block takes one token and up to ROPE_THREADS items of 2 W values of its heads: W neighbouring pairs
// (interleaved), or W values of the first half with their W partners in the second. Its first threads form the
// token's angles once for all heads, in 64 bits, reduced to a fraction of a turn there (in 32 bits a far
// position's angle has lost all its digits after 2^24 turns), sine and cosine in f32; the values are
// already on their way then. W is the widest access (16 bytes at most) that every pointer, stride and, for
// halves, half the rotated width allow. (Four items per thread, so that a token's angles are formed in one block instead of
// three: 59 against 47 us for 8192 tokens of 48 heads of 128, f16.)
constexpr int ROPE_THREADS = 128, ROPE_BLOCKS = 12;

struct RopeAppendArgs : nrc_rope_args {
  nrc_paged_kv kv;
};

template <int BYTES>
struct Bits;
template <>
struct Bits<16> { using T = uint4; };
template <>
struct Bits<8> { using T = uint2; };
template <>
struct Bits<4> { using T = uint32_t; };
template <>
struct Bits<2> { using T = uint16_t; };

// W values of type DT at element offset i, in registers of the widest access.
template <int DT, int W>
NRC_DEV void load_values(float (&x)[W], const void* p, int64_t i) {
  constexpr int SIZE = DT == NRC_F32 ? 4 : 2;
  using T = typename Bits<SIZE * W>::T;
  const T raw = *reinterpret_cast<const T*>(static_cast<const uint8_t*>(p) + i * SIZE);
#pragma unroll
  for (int e = 0; e < W; e++) x[e] = load_as_f32(&raw, e, DT);
}
template <int DT, int W>
NRC_DEV void store_values(const float (&x)[W], void* p, int64_t i) {
  constexpr int SIZE = DT == NRC_F32 ? 4 : 2;
  using T = typename Bits<SIZE * W>::T;
  T raw;
#pragma unroll
  for (int e = 0; e < W; e++) store_from_f32(&raw, e, DT, x[e]);
  *reinterpret_cast<T*>(static_cast<uint8_t*>(p) + i * SIZE) = raw;
}

// One pair of values turned by (cos, sin).
NRC_DEV void turn(float& x, float& y, float2 r) {
  const float u = x * r.x - y * r.y;
  y = x * r.y + y * r.x;
  x = u;
}

template <int DT, int W>
__global__ void __launch_bounds__(ROPE_THREADS, ROPE_BLOCKS) k_rope_append_paged(const RopeAppendArgs a) {
  // Cosine and sine of each pair (head_dim <= 128): pair W c + e at [e][c], so that neighbouring items read neighbours.
  __shared__ float2 cs[W][64 / W];
  const uint32_t t = blockIdx.x, hd = a.kv.head_dim, half = (uint32_t)a.rot_dim / 2, hq = (uint32_t)a.n_heads, hk = a.kv.n_kv_heads;
  // The item's head (query heads, then K's, then V's), its place in it, and its two groups of W values: halves pair their
  // first half / W items, the others hold what is not rotated.
  const uint32_t per_head = hd / (2 * W), item = blockIdx.y * ROPE_THREADS + threadIdx.x;
  const uint32_t hh = item / per_head, c = item - hh * per_head;
  const bool live = hh < hq + 2 * hk, is_q = hh < hq, is_k = !is_q && hh < hq + hk;
  const uint32_t h = is_q ? hh : is_k ? hh - hq : hh - hq - hk;
  const bool split = a.style == 1 && c * W < half;
  const uint32_t i0 = split ? c * W : 2 * W * c, i1 = split ? i0 + half : i0 + W;
  float x[W], y[W];
  int32_t slot = -1, seq = 0;
  if (live) {
    const void* src = is_q ? a.q : is_k ? a.k : a.v;
    const int64_t from = is_q   ? (int64_t)t * a.q_token + (int64_t)h * a.q_head
                         : is_k ? (int64_t)t * a.k_token + (int64_t)h * a.k_head
                                : (int64_t)t * a.v_token + (int64_t)h * a.v_head;
    load_values<DT, W>(x, src, from + i0);
    load_values<DT, W>(y, src, from + i1);
    if (!is_q) slot = a.slot[t], seq = a.seq[t];
  }
  for (uint32_t i = threadIdx.x; i < half; i += ROPE_THREADS) {
    const double turns = (double)a.pos[t] * (double)a.freqs[i] * 0.15915494309189533577;
    float sn, co;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &co);
    cs[i % W][i / W] = make_float2(co * a.mscale, sn * a.mscale);
  }
  __syncthreads();
  if (!live) return;
  if (is_q || is_k) {
    if (split) {
#pragma unroll
      for (int i = 0; i < W; i++) turn(x[i], y[i], cs[i][c]);
    } else if (a.style == 0 && W == 1) {
      if (c < half) turn(x[0], y[0], cs[0][c]);
    } else if (a.style == 0) {
#pragma unroll
      for (int i = 0; i < W; i += 2) {
        if (W * c + i / 2 < half) turn(x[i], x[(i + 1) % W], cs[i / 2][c]);
        if (W * c + W / 2 + i / 2 < half) turn(y[i], y[(i + 1) % W], cs[W / 2 + i / 2][c]);
      }
    }
  }
  if (is_q) {
    const int64_t to = (int64_t)t * a.qo_token + (int64_t)h * a.qo_head;
    store_values<DT, W>(x, a.q_out, to + i0);
    store_values<DT, W>(y, a.q_out, to + i1);
    return;
  }
  if (slot < 0) return;
  if (seq < 0 || (uint32_t)seq >= a.kv.n_seqs || (uint32_t)slot / a.kv.page_size >= a.kv.max_pages) {
    atomicOr(&g_paged_err, ERR_BAD_SLOT);
    return;
  }
  const int64_t row = paged_row(a.kv, seq, slot);
  if (row < 0) {
    atomicOr(&g_paged_err, ERR_BAD_PAGE);
    return;
  }
  void* dst = is_k ? a.kv.k : a.kv.v;
  const int64_t to = row + (int64_t)h * a.kv.head_stride;
  if (a.kv.dtype == NRC_F16) {
    store_values<NRC_F16, W>(x, dst, to + i0);
    store_values<NRC_F16, W>(y, dst, to + i1);
  } else {
    store_values<NRC_BF16, W>(x, dst, to + i0);
    store_values<NRC_BF16, W>(y, dst, to + i1);
  }
}

template <int DT, int W>
cudaError_t launch_rope(const RopeAppendArgs& a, cudaStream_t s) {
  const uint32_t items = ((uint32_t)a.n_heads + 2 * a.kv.n_kv_heads) * (a.kv.head_dim / (2 * W));
  k_rope_append_paged<DT, W><<<dim3((uint32_t)a.tokens, (items + ROPE_THREADS - 1) / ROPE_THREADS), ROPE_THREADS, 0, s>>>(a);
  return cudaGetLastError();
}
template <int DT>
cudaError_t launch_rope_w(const RopeAppendArgs& a, uint32_t w, cudaStream_t s) {
  if constexpr (DT != NRC_F32)
    if (w == 8) return launch_rope<DT, 8>(a, s);
  return w >= 4 ? launch_rope<DT, 4>(a, s) : w == 2 ? launch_rope<DT, 2>(a, s) : launch_rope<DT, 1>(a, s);
}

// ------------------------------------------------------------ eviction
// The kept positions of a (sequence, KV head): the largest key that `want` weights reach, found by three radix passes,
// then one pass in position order. One block per row, bound by its instructions and barriers over a row that stays in L1
// and L2: 28 us for 24 sequences up to 20000 positions and 8 KV heads. (A cluster of four blocks per row: 71 us, adding up
// its histograms took longer than counting them; four counters per bin: 27 against 24 us without the weights' moves; keys
// kept in registers: 32 us, they do not fit; one scan of warp counts per 32768 positions: 27 us.)
constexpr int EV_THREADS = 1024, EV_BINS = 2048, EV_EACH = 4;

// Weights ordered as unsigned keys: larger weight, larger key; both zeros alike; NaN the smallest.
NRC_DEV uint32_t weight_key(float v) {
  const uint32_t b = __float_as_uint(v + 0.0f);  // -0 becomes +0
  return v == v ? b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u) : 0u;
}

// Exclusive prefix sum of v over the EV_THREADS threads; *total its sum. Two barriers.
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
  uint32_t w = red[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t y = __shfl_up_sync(0xffffffffu, w, o);
    if (lane >= o) w += y;
  }
  *total = __shfl_sync(0xffffffffu, w, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
  return (warp ? before : 0) + x - v;
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

__global__ void __launch_bounds__(EV_THREADS) k_evict_select(const EvictArgs a) {
  __shared__ uint32_t red[32], hist[EV_BINS], found[2];
  const uint32_t h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const size_t row = (size_t)b * a.kv.n_kv_heads + h;
  const uint32_t n = evict_len(a, b);
  const float* w = a.weights + row * a.weights_len;
  float* nw = a.new_weights + row * a.weights_len;
  int32_t* kept = a.kept + row * a.budget;
  const bool all = n <= a.budget;
  const uint32_t lo = a.sinks, hi = all ? n : n - a.recent;  // chosen by weight: [lo, hi)
  // Positions of [lo, hi) whose key is above `key` are kept, and the first `ties` of those that equal it.
  uint32_t key = 0xffffffffu, ties = 0;  // no weight's key
  if (!all && a.budget > a.sinks + a.recent) {
    uint32_t need = a.budget - a.sinks - a.recent, prefix = 0, mask = 0;
    for (int pass = 0; pass < 3; pass++) {
      const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
      const uint32_t bins = pass < 2 ? 2048u : 1024u;
      for (uint32_t i = tid; i < EV_BINS; i += EV_THREADS) hist[i] = 0;
      __syncthreads();
#pragma unroll 8
      for (uint32_t t = lo + tid; t < hi; t += EV_THREADS) {
        const uint32_t k = weight_key(w[t]);
        if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
      }
      __syncthreads();
      // Bins from the largest on, two a thread: where the count reaches `need`.
      const uint32_t c0 = hist[EV_BINS - 1 - 2 * tid], c1 = hist[EV_BINS - 2 - 2 * tid];
      uint32_t total;
      const uint32_t above = block_scan(c0 + c1, red, &total);
      if (above < need && above + c0 + c1 >= need) {
        const bool first = above + c0 >= need;
        found[0] = EV_BINS - 1 - 2 * tid - (first ? 0 : 1);
        found[1] = need - above - (first ? 0 : c0);
      }
      __syncthreads();
      prefix |= found[0] << shift;
      mask |= (bins - 1) << shift;
      need = found[1];
    }
    key = prefix;
    ties = need;
  }
  uint32_t above = 0, tied = 0;
  for (uint32_t t0 = 0; t0 < n; t0 += EV_THREADS * EV_EACH) {
    float v[EV_EACH];
    uint32_t keep = 0, tie = 0;
    const uint32_t t1 = t0 + tid * EV_EACH;
#pragma unroll
    for (int e = 0; e < EV_EACH; e++) {
      const uint32_t t = t1 + e;
      if (t < n) {
        v[e] = w[t];
        const uint32_t k = weight_key(v[e]);
        const bool fixed = all || t < lo || t >= hi;
        keep |= (fixed || k > key ? 1u : 0u) << e;
        tie |= (!fixed && k == key ? 1u : 0u) << e;
      }
    }
    uint32_t sum;
    // Its barriers stand between the reads of these positions and the writes below (new_weights may be weights).
    const uint32_t before = block_scan((uint32_t)__popc(keep) << 16 | (uint32_t)__popc(tie), red, &sum);
    uint32_t g = above + (before >> 16), q = tied + (before & 0xffffu);
#pragma unroll
    for (int e = 0; e < EV_EACH; e++) {
      const bool is_tie = (tie >> e) & 1, kp = ((keep >> e) & 1) || (is_tie && q < ties);
      const uint32_t to = g + min(q, ties);
      if (kp) {
        kept[to] = (int32_t)(t1 + e);
        nw[to] = v[e];
      }
      g += (keep >> e) & 1;
      q += is_tie;
    }
    above += sum >> 16;
    tied += sum & 0xffffu;
  }
  const uint32_t count = above + min(tied, ties);
  for (uint32_t i = count + tid; i < a.budget; i += EV_THREADS) kept[i] = -1;
  __syncthreads();
  for (uint32_t i = count + tid; i < a.weights_len; i += EV_THREADS) nw[i] = 0.0f;
  pdl_trigger();
}

// Rows move down to their new slots in ascending order. Slot i receives slot kept[i] >= i, so a batch of rows that is
// read whole before it is written overwrites nothing that a later batch reads. One block takes a column of 64 bytes of
// all the rows of a (sequence, KV head, K or V): columns are independent, and there are enough of them to fill the GPU.
// A warp takes 32 rows of a batch: each lane looks up where one of them lies and goes, then 4 lanes move a row.
// Bound by HBM.
constexpr int MV_PIECES = 4, MV_EACH = MV_PIECES;

__global__ void __launch_bounds__(1024) k_evict_move(const EvictArgs a) {
  pdl_wait();
  const uint32_t cols = a.kv.head_dim / (8 * MV_PIECES), h = blockIdx.x / cols, b = blockIdx.y;
  const uint32_t lane = threadIdx.x & 31;
  // new_lens may be lens: only this thread reads that element here.
  if (blockIdx.x == 0 && blockIdx.z == 0 && threadIdx.x == 0) {
    const uint32_t n = evict_len(a, b);
    a.new_lens[b] = (int32_t)(n < a.budget ? n : a.budget);
  }
  if (a.budget == 0) return;
  const int32_t* kept = a.kept + ((size_t)b * a.kv.n_kv_heads + h) * a.budget;
  const int32_t end = kept[a.budget - 1];
  if (end < 0 || (uint32_t)end == a.budget - 1) return;  // every row is where it belongs
  uint16_t* base = static_cast<uint16_t*>(blockIdx.z ? a.kv.v : a.kv.k) + (int64_t)h * a.kv.head_stride +
                   (blockIdx.x % cols) * MV_PIECES * 8 + (lane % MV_PIECES) * 8;
  // The row of this thread in the batch from i0 on: where it lies (-1: it stays) and goes.
  auto locate = [&](uint32_t i0, int64_t& from, int64_t& to) {
    const uint32_t i = i0 + threadIdx.x;
    const int32_t src = i < a.budget ? kept[i] : -1;
    from = to = -1;
    if (src < 0 || (uint32_t)src == i) return;
    from = paged_row(a.kv, b, src);
    to = paged_row(a.kv, b, i);
    if (from < 0 || to < 0) {
      atomicOr(&g_paged_err, ERR_BAD_PAGE);
      from = -1;
    }
  };
  int64_t from, to;
  locate(0, from, to);
  for (uint32_t i0 = 0; i0 < a.budget; i0 += blockDim.x) {
    uint4 x[MV_EACH];
    int64_t into[MV_EACH];
#pragma unroll
    for (int e = 0; e < MV_EACH; e++) {
      const int who = e * (32 / MV_PIECES) + lane / MV_PIECES;
      const int64_t f = __shfl_sync(0xffffffffu, from, who);
      into[e] = __shfl_sync(0xffffffffu, to, who);
      if (f < 0) into[e] = -1;
      if (f >= 0) x[e] = *reinterpret_cast<const uint4*>(base + f);
    }
    locate(i0 + blockDim.x, from, to);
    __syncthreads();
#pragma unroll
    for (int e = 0; e < MV_EACH; e++)
      if (into[e] >= 0) *reinterpret_cast<uint4*>(base + into[e]) = x[e];
  }
}

}  // namespace

cudaError_t rope_append_paged_run(const nrc_paged_kv& kv, const nrc_rope_args& r, cudaStream_t s) {
  RopeAppendArgs a;
  static_cast<nrc_rope_args&>(a) = r;
  a.kv = kv;
  const uint32_t size = a.dtype == NRC_F32 ? 4 : 2;
  // Every bit below the access width is 0 in what all accesses start from (the pages' strides are checked already).
  uint64_t low = reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                 reinterpret_cast<uintptr_t>(a.q_out);
  for (int64_t stride : {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head, a.qo_token, a.qo_head})
    low |= (uint64_t)stride * size;
  if (a.style == 1) low |= (uint64_t)(a.rot_dim / 2) * size;
  uint32_t w = 16 / size;
  while (w > 1 && low % (w * size)) w /= 2;
  return a.dtype == NRC_F32   ? launch_rope_w<NRC_F32>(a, w, s)
         : a.dtype == NRC_F16 ? launch_rope_w<NRC_F16>(a, w, s)
                              : launch_rope_w<NRC_BF16>(a, w, s);
}

cudaError_t kv_evict_run(const EvictArgs& a, cudaStream_t s) {
  k_evict_select<<<dim3(a.kv.n_kv_heads, a.kv.n_seqs), EV_THREADS, 0, s>>>(a);
  if (cudaError_t e = cudaGetLastError()) return e;
  // Few columns: all the rows that a block can hold in flight. Many: smaller blocks, which wait less for one another. Both
  // kernels, us with blocks of 256, 512 and 1024 threads: 32 columns (one sequence of 1500 to 1024, 64 wide) 11.6, 10.5, 10.2; 256 (4 of
  // 8000 to 4096, 128 wide) 51.3, 44.3, 48.3; 512 (8 of them) 65.3, 70.3, 76.9; 1536 (24 of 1000..20000) 167, 165, 180; 2048 (64 of
  // 2000 to 1000, 64 wide) 71.9, 77.5, 89.7.
  const uint64_t blocks = (uint64_t)a.kv.n_kv_heads * (a.kv.head_dim / (8 * MV_PIECES)) * a.kv.n_seqs * 2;
  const uint32_t threads = blocks < 296 ? 1024 : blocks < 1184 ? 512 : 256;
  EvictArgs aa = a;
  void* args[] = {&aa};
  return launch_kernel((const void*)k_evict_move, dim3(a.kv.n_kv_heads * (a.kv.head_dim / (8 * MV_PIECES)), a.kv.n_seqs, 2),
                       dim3(threads), 0, s, true, args);
}

cudaError_t paged_take_errors(unsigned* bits) {
  cudaError_t e = cudaMemcpyFromSymbol(bits, g_paged_err, sizeof(unsigned));
  const unsigned zero = 0;
  if (e == cudaSuccess && *bits) e = cudaMemcpyToSymbol(g_paged_err, &zero, sizeof zero);
  return e;
}

}  // namespace nrc
