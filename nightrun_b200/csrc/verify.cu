// Verification of drafted tokens against the target's probabilities.
//
// Draft x_i is taken while u_i q_i(x_i) < p_i(x_i), an exact comparison in 64 bits (products of two f32 values); the
// token behind the taken ones is the first index whose running sum of r = max(p - q, 0) (or of p) exceeds u times the
// whole sum. The running sums are taken in 64 bits: in 32 the order of the additions would move the drawn token.
//
// Bound by reading one row of p (and of q): HBM for many sequences, latency for few. A cluster of blocks takes a
// sequence, each warp a contiguous span of the row; the span sums are exchanged through distributed shared memory, and
// only the span that holds the goal is read again, by one warp.
#include <cooperative_groups.h>

#include "paged.cuh"

namespace nrc {
namespace {

namespace cg = cooperative_groups;

constexpr int VD_THREADS = 512, VD_WARPS = VD_THREADS / 32, VD_MAX_CLUSTER = 8;

// What is left of p at one token: max(p - q, 0) after a refusal, p itself otherwise; NaN and
// negative values count as nothing. The difference of two f32 values is formed in 64 bits.
NRC_DEV double left_of(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0.0 ? d : 0.0;
}

template <int DT>
struct Row {
  const void *p, *q;   // q null: nothing is taken from p, or (certain >= 0) all of one token
  int32_t certain;
  NRC_DEV double at(uint32_t t) const {
    return left_of(load_as_f32(p, t, DT), q ? load_as_f32(q, t, DT) : (int32_t)t == certain ? 1.0f : 0.0f);
  }
};

// Sum of [t0, t1) over the warp. Rows may start anywhere: single values up to a 16-byte border of p, then 16-byte
// pieces where q is aligned like p, single values otherwise.
template <int DT>
NRC_DEV double span_sum(const Row<DT>& r, uint32_t t0, uint32_t t1, int lane) {
  constexpr uint32_t SIZE = DT == NRC_F32 ? 4 : 2, W = 16 / SIZE;
  double s0 = 0.0, s1 = 0.0;
  const uintptr_t pa = reinterpret_cast<uintptr_t>(r.p), qa = reinterpret_cast<uintptr_t>(r.q);
  if (pa % SIZE == 0 && (!r.q || (pa - qa) % 16 == 0)) {
    const uint32_t ahead = min((uint32_t)((16 - (pa + (uint64_t)t0 * SIZE) % 16) % 16) / SIZE, t1 - t0);
    if ((uint32_t)lane < ahead) s0 += r.at(t0 + lane);
    t0 += ahead;
    const uint32_t pieces = (t1 - t0) / W;
    const uint4* pv = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(r.p) + (uint64_t)t0 * SIZE);
    const uint4* qv = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(r.q) + (uint64_t)t0 * SIZE);
    constexpr int U = 4;
    for (uint32_t i0 = lane; i0 < pieces; i0 += 32 * U) {
      uint4 x[U], y[U];
#pragma unroll
      for (int k = 0; k < U; k++) {
        const uint32_t i = i0 + 32 * k;
        x[k] = y[k] = make_uint4(0, 0, 0, 0);
        if (i < pieces) {
          x[k] = __ldg(pv + i);
          if (r.q) y[k] = __ldg(qv + i);
        }
      }
#pragma unroll
      for (int k = 0; k < U; k++) {
        const uint32_t first = t0 + (i0 + 32 * k) * W;
#pragma unroll
        for (uint32_t e = 0; e < W; e++) {
          const float q = r.q ? load_as_f32(&y[k], e, DT) : (int32_t)(first + e) == r.certain ? 1.0f : 0.0f;
          const double d = left_of(load_as_f32(&x[k], e, DT), q);
          if (e & 1)
            s1 += d;
          else
            s0 += d;
        }
      }
    }
    t0 += pieces * W;
    if (t0 + lane < t1) s0 += r.at(t0 + lane);
  } else {
    constexpr int U = 8;
    for (uint32_t i0 = t0 + lane; i0 < t1; i0 += 32 * U)
#pragma unroll
      for (int k = 0; k < U; k++)
        if (i0 + 32 * k < t1) s0 += r.at(i0 + 32 * k);
  }
  double s = s0 + s1;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// First index of [t0, t1) whose running sum, begun at `before`, exceeds goal; where rounding leaves none, the last one
// that holds anything.
template <int DT>
NRC_DEV uint32_t span_find(const Row<DT>& r, uint32_t t0, uint32_t t1, double before, double goal, int lane) {
  const uint32_t per = (t1 - t0 + 31) / 32, a = min(t0 + lane * per, t1), b = min(a + per, t1);
  double s = 0.0;
  int last = -1;
#pragma unroll 8
  for (uint32_t t = a; t < b; t++) {
    const double d = r.at(t);
    s += d;
    if (d > 0.0) last = (int)t;
  }
  double run = s;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += y;
  }
  run += before;
  const unsigned over = __ballot_sync(0xffffffffu, run > goal), some = __ballot_sync(0xffffffffu, last >= 0);
  if (over) {
    const int who = __ffs(over) - 1;
    double prev = __shfl_up_sync(0xffffffffu, run, 1);
    if (lane == 0) prev = before;
    int found = last;
    if (lane == who)
      for (uint32_t t = a; t < b; t++) {
        prev += r.at(t);
        if (prev > goal) {
          found = (int)t;
          break;
        }
      }
    found = __shfl_sync(0xffffffffu, found, who);
    if (found >= 0) return (uint32_t)found;
  }
  return some ? (uint32_t)__shfl_sync(0xffffffffu, last, 31 - __clz(some)) : 0u;
}

template <int DT>
__global__ void __launch_bounds__(VD_THREADS) k_verify_draft(const VerifyArgs a) {
  constexpr uint32_t SIZE = DT == NRC_F32 ? 4 : 2;
  __shared__ double sums[2][VD_MAX_CLUSTER * VD_WARPS];  // every span's, in each block of the cluster
  __shared__ uint32_t taken_s;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const uint32_t b = blockIdx.x / blocks, m = a.n_max;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) {
    // All drafts at once; the first that is refused counts.
    int nd = a.n_draft ? a.n_draft[b] : (int)m;
    nd = nd < 0 ? 0 : nd > (int)m ? (int)m : nd;
    int taken = nd;
    for (int i0 = 0; i0 < nd; i0 += 32) {
      const int i = i0 + lane;
      bool refuse = false;
      if (i < nd) {
        const int32_t x = a.draft[(size_t)b * m + i];
        refuse = true;
        if (x >= 0 && (uint32_t)x < a.vocab) {
          const float px = load_as_f32(a.p, (int64_t)b * a.p_seq + (int64_t)i * a.p_token + x, DT);
          const float qx = a.q ? load_as_f32(a.q, (int64_t)b * a.q_seq + (int64_t)i * a.q_token + x, DT) : 1.0f;
          refuse = !((double)a.u[(size_t)b * (m + 1) + i] * (double)qx < (double)px);
        }
      }
      const unsigned no = __ballot_sync(0xffffffffu, refuse);
      if (no) {
        taken = i0 + __ffs(no) - 1;
        break;
      }
    }
    if (lane == 0) taken_s = (uint32_t)taken | (taken < nd ? 0x80000000u : 0u);
  }
  __syncthreads();
  const uint32_t taken = taken_s & 0x7fffffffu;
  const bool refused = taken_s >> 31;
  Row<DT> row;
  row.p = static_cast<const uint8_t*>(a.p) + ((int64_t)b * a.p_seq + (int64_t)taken * a.p_token) * SIZE;
  row.q = refused && a.q ? static_cast<const uint8_t*>(a.q) + ((int64_t)b * a.q_seq + (int64_t)taken * a.q_token) * SIZE
                         : nullptr;
  row.certain = refused && !a.q ? a.draft[(size_t)b * m + taken] : -1;

  // Spans of whole 16-byte pieces (counted from the row's start), in index order over blocks and warps.
  const uint32_t spans = blocks * VD_WARPS;
  uint32_t per = (a.vocab + spans - 1) / spans;
  per = (per + 7) & ~7u;
  auto begin = [&](uint32_t i) { return (uint32_t)min((uint64_t)i * per, (uint64_t)a.vocab); };
  const uint32_t mine = rank * VD_WARPS + warp;
  for (int round = 0;; round++) {
    const double s = span_sum<DT>(row, begin(mine), begin(mine + 1), lane);
    if ((uint32_t)lane < blocks) *cluster.map_shared_rank(&sums[round][mine], lane) = s;
    cluster.sync();
    if (warp != 0 && round == 1) return;
    // Each block's warps look for the goal alike: the running sums of the spans, `each` of them per lane.
    const uint32_t each = (spans + 31) / 32;
    double t = 0.0;
    for (uint32_t i = lane * each; i < min((lane + 1) * each, spans); i++) t += sums[round][i];
    double run = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    const double total = __shfl_sync(0xffffffffu, run, 31);
    if (!(total > 0.0) && refused && round == 0) {  // the difference leaves nothing: p itself (every block agrees)
      row.q = nullptr;
      row.certain = -1;
      continue;
    }
    if (warp != 0) return;
    const double goal = (double)a.u[(size_t)b * (m + 1) + m] * total;
    double before = run - t;
    // The lane's spans one by one: the first whose running sum exceeds the goal, and the last that holds anything.
    int over = -1, last = -1;
    double at_over = 0.0, x = __shfl_up_sync(0xffffffffu, run, 1);
    before = lane ? x : 0.0;
    for (uint32_t i = lane * each; i < min((lane + 1) * each, spans); i++) {
      const double v = sums[round][i];
      if (over < 0 && before + v > goal) over = (int)i, at_over = before;
      if (v > 0.0) last = (int)i;
      before += v;
    }
    const unsigned any_over = __ballot_sync(0xffffffffu, over >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
    uint32_t token = 0, owner = 0;
    if (any_over) {
      const int who = __ffs(any_over) - 1;
      owner = (uint32_t)__shfl_sync(0xffffffffu, over, who);
      at_over = __shfl_sync(0xffffffffu, at_over, who);
    } else if (any) {  // rounding, or u not below 1: the last token that holds anything
      owner = (uint32_t)__shfl_sync(0xffffffffu, last, 31 - __clz(any));
      at_over = -INFINITY;
    }
    if (owner / VD_WARPS != rank) return;
    if (any_over || any) token = span_find<DT>(row, begin(owner), begin(owner + 1), at_over, goal, lane);
    for (uint32_t i = lane; i <= m; i += 32)
      a.tokens[(size_t)b * (m + 1) + i] = i < taken ? a.draft[(size_t)b * m + i] : i == taken ? (int32_t)token : -1;
    if (lane == 0) a.accepted[b] = (int32_t)taken;
    return;
  }
}

}  // namespace

cudaError_t verify_draft_run(const VerifyArgs& a, cudaStream_t s) {
  // Blocks per sequence: as many as give each warp some 512 tokens.
  uint32_t blocks = 1;
  while (blocks < VD_MAX_CLUSTER && (uint64_t)blocks * VD_WARPS * 512 < a.vocab) blocks *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.n_seqs * blocks);
  cfg.blockDim = dim3(VD_THREADS);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  VerifyArgs aa = a;
  void* args[] = {&aa};
  const void* fn = a.dtype == NRC_F32   ? (const void*)k_verify_draft<NRC_F32>
                   : a.dtype == NRC_F16 ? (const void*)k_verify_draft<NRC_F16>
                                        : (const void*)k_verify_draft<NRC_BF16>;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace nrc
