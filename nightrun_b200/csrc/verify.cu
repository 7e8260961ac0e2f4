// Verification of drafted tokens against the target's probabilities.
//
// Draft x_i is taken while u_i q_i(x_i) < p_i(x_i), an exact comparison in 64 bits (products of two f32 values); the
// token behind the taken ones is the first index whose running sum of r = max(p - q, 0) (or of p) exceeds u times the
// whole sum. The running sums are taken in 64 bits: in 32 the order of the additions would move the drawn token. (Pairs of
// f32 with error-free sums, to save the conversions: 47 against 44 us for 160 rows of 151936. It is not the arithmetic.)
//
// Bound by reading one row of p (and of q): HBM for many sequences, latency for few. A cluster of blocks takes a
// sequence, each warp a contiguous span of the row; the span sums are exchanged through distributed shared memory, and
// only the group of a span's tokens that holds the goal is read again, by the warp that summed it.
#include <cooperative_groups.h>
#include <float.h>

#include "paged.cuh"

namespace nrc {
namespace {

namespace cg = cooperative_groups;

constexpr int VD_MAX_CLUSTER = 8;

// What is left of p at one token: max(p - q, 0) after a refusal, p itself otherwise; NaN, infinities (of p or q) and negative
// differences count as nothing. The difference of two f32 values is formed in 64 bits.
NRC_DEV double left_of(float p, float q) { return p > q && fmaxf(p, -q) <= FLT_MAX ? (double)p - (double)q : 0.0; }

// Two running sums of what is left.
struct Sums {
  double a = 0.0, b = 0.0;
  NRC_DEV void add(float2 p, float2 q) {
    a += left_of(p.x, q.x);
    b += left_of(p.y, q.y);
  }
  NRC_DEV double value() const { return a + b; }
};

template <int DT>
struct Row {
  const void *p, *q;   // q null: nothing is taken from p, or (certain >= 0) all of one token
  int32_t certain;
  NRC_DEV double at(uint32_t t) const {
    return left_of(load_as_f32(p, t, DT), q ? load_as_f32(q, t, DT) : (int32_t)t == certain ? 1.0f : 0.0f);
  }
};

NRC_DEV double warp_sum(double s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// How a warp walks a span of tokens: single values up to the first 16-byte border of p (`ahead` of them), then batches of
// 32 * U pieces of 16 bytes where q is aligned like p, of 64 * U single values otherwise, then what is left over.
// FINE groups of `group` batches keep sums of their own, the first with what is ahead, the last with the rest.
constexpr int FINE = 8;
template <int DT, int U>
struct Span {
  static constexpr uint32_t SIZE = DT == NRC_F32 ? 4 : 2, W = 16 / SIZE;
  uint32_t t0, t1, ahead, batch, batches, group;
  bool wide;
  NRC_DEV Span(const Row<DT>& r, uint32_t a, uint32_t b) : t0(a), t1(b) {
    const uintptr_t pa = reinterpret_cast<uintptr_t>(r.p) + (uint64_t)t0 * SIZE, qa = reinterpret_cast<uintptr_t>(r.q);
    wide = !r.q || (reinterpret_cast<uintptr_t>(r.p) - qa) % 16 == 0;
    ahead = wide ? min((uint32_t)((16 - pa % 16) % 16) / SIZE, t1 - t0) : 0;
    batch = wide ? 32 * U * W : 64 * U;
    batches = (t1 - t0 - ahead + batch - 1) / batch;
    group = (batches + FINE - 1) / FINE;
  }
  // The tokens of group f.
  NRC_DEV uint32_t begin(uint32_t f) const {
    return f == 0 ? t0 : (uint32_t)min((uint64_t)t0 + ahead + (uint64_t)f * group * batch, (uint64_t)t1);
  }
};

// Sums of a span's groups into fine[], and of the whole.
template <int DT, int U>
NRC_DEV double span_sum(const Row<DT>& r, const Span<DT, U>& sp, double* fine, int lane) {
  constexpr uint32_t W = Span<DT, U>::W;
  double all = 0.0, edge = (uint32_t)lane < sp.ahead ? r.at(sp.t0 + lane) : 0.0;
  const uint32_t a0 = sp.t0 + sp.ahead;
  const uint4* pv = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(r.p) + (uint64_t)a0 * Span<DT, U>::SIZE);
  const uint4* qv = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(r.q) + (uint64_t)a0 * Span<DT, U>::SIZE);
  Sums s;
  uint32_t f = 0, in_group = 0;
  for (uint32_t i = 0; i < sp.batches; i++) {
    const uint32_t a = a0 + i * sp.batch;
    if (sp.wide) {
      uint4 x[U], y[U];
#pragma unroll
      for (int k = 0; k < U; k++) {
        const uint32_t piece = (i * U + k) * 32 + lane;
        x[k] = y[k] = make_uint4(0, 0, 0, 0);
        if (a0 + (piece + 1) * W <= sp.t1) {
          x[k] = __ldg(pv + piece);
          if (r.q) y[k] = __ldg(qv + piece);
        }
      }
#pragma unroll
      for (int k = 0; k < U; k++) {
        const uint32_t t = a + (lane + 32 * k) * W;
#pragma unroll
        for (uint32_t e = 0; e < W; e += 2) {
          float2 q = make_float2(load_as_f32(&y[k], e, DT), load_as_f32(&y[k], e + 1, DT));
          if (!r.q) q = make_float2((int32_t)(t + e) == r.certain ? 1.0f : 0.0f, (int32_t)(t + e + 1) == r.certain ? 1.0f : 0.0f);
          s.add(make_float2(load_as_f32(&x[k], e, DT), load_as_f32(&x[k], e + 1, DT)), q);
        }
        if (t < sp.t1 && t + W > sp.t1)  // the piece that the span cuts
          for (uint32_t u = t; u < sp.t1; u++) edge += r.at(u);
      }
    } else {
      float p[2 * U], q[2 * U];
#pragma unroll
      for (int k = 0; k < 2 * U; k++) {
        const uint32_t t = a + lane + 32 * k;
        p[k] = t < sp.t1 ? load_as_f32(r.p, t, DT) : 0.0f;
        q[k] = t < sp.t1 ? load_as_f32(r.q, t, DT) : 0.0f;
      }
#pragma unroll
      for (int k = 0; k < 2 * U; k += 2) s.add(make_float2(p[k], p[k + 1]), make_float2(q[k], q[k + 1]));
    }
    if (++in_group == sp.group || i + 1 == sp.batches) {
      const double g = warp_sum(s.value() + edge);
      if (lane == 0) fine[f] = g;
      all += g;
      s = Sums();
      edge = 0.0;
      in_group = 0;
      f++;
    }
  }
  if (sp.batches == 0) {
    all = warp_sum(edge);
    if (lane == 0) fine[0] = all;
    f = 1;
  }
  if ((uint32_t)lane >= f && lane < FINE) fine[lane] = 0.0;
  __syncwarp();
  return all;
}

// First index of [t0, t1) whose running sum, begun at `before`, exceeds goal; where rounding leaves none, the last one
// that holds anything. A lane takes 4 neighbours at a time, the next ones on their way.
template <int DT>
NRC_DEV uint32_t span_find(const Row<DT>& r, uint32_t t0, uint32_t t1, double before, double goal, int lane) {
  float p[4], q[4];
  auto fetch = [&](uint32_t t) {
#pragma unroll
    for (int e = 0; e < 4; e++, t++) {
      p[e] = t < t1 ? load_as_f32(r.p, t, DT) : 0.0f;
      q[e] = t < t1 && r.q ? load_as_f32(r.q, t, DT) : (int32_t)t == r.certain ? 1.0f : 0.0f;
    }
  };
  int last = 0;
  fetch(t0 + 4 * lane);
  for (; t0 < t1; t0 += 128) {
    const int t = (int)(t0 + 4 * lane);
    double v[4], own = 0.0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      v[e] = left_of(p[e], q[e]);
      own += v[e];
    }
    fetch(t0 + 128 + 4 * lane);
    double run = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    double prev = __shfl_up_sync(0xffffffffu, run, 1);
    prev = before + (lane ? prev : 0.0);
    int found = -1, mine = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      prev += v[e];
      if (v[e] > 0.0) mine = t + e;
      if (found < 0 && v[e] > 0.0 && prev > goal) found = t + e;
    }
    const unsigned over = __ballot_sync(0xffffffffu, found >= 0), some = __ballot_sync(0xffffffffu, own > 0.0);
    if (over) return (uint32_t)__shfl_sync(0xffffffffu, found, __ffs(over) - 1);
    if (some) last = __shfl_sync(0xffffffffu, mine, 31 - __clz(some));
    before += __shfl_sync(0xffffffffu, run, 31);
  }
  return (uint32_t)last;
}

// The span that holds something and whose running sum first exceeds goal, and the running sum before it; where rounding
// leaves none, the last that holds anything (before: -inf); -1 if none does. (A lane's running sum begins with the scan's, which
// may be a rounding above the lane's before it: without the first condition a goal between the two would pick a span of
// zeros.) One warp; sums in index order, each lane `n / 32` of them.
NRC_DEV int pick_span(const double* sums, uint32_t n, double goal_of_total, double* total, double* before, int lane) {
  const uint32_t each = (n + 31) / 32, i0 = min(lane * each, n), i1 = min(i0 + each, n);
  double t = 0.0;
  for (uint32_t i = i0; i < i1; i++) t += sums[i];
  double run = t;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, run, o);
    if (lane >= o) run += y;
  }
  *total = __shfl_sync(0xffffffffu, run, 31);
  const double goal = goal_of_total * *total;
  double at = __shfl_up_sync(0xffffffffu, run, 1);
  if (lane == 0) at = 0.0;
  int over = -1, last = -1;
  double at_over = 0.0;
  for (uint32_t i = i0; i < i1; i++) {
    const double v = sums[i];
    if (over < 0 && v > 0.0 && at + v > goal) over = (int)i, at_over = at;
    if (v > 0.0) last = (int)i;
    at += v;
  }
  const unsigned any_over = __ballot_sync(0xffffffffu, over >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
  if (any_over) {
    const int who = __ffs(any_over) - 1;
    *before = __shfl_sync(0xffffffffu, at_over, who);
    return __shfl_sync(0xffffffffu, over, who);
  }
  *before = -INFINITY;
  return any ? __shfl_sync(0xffffffffu, last, 31 - __clz(any)) : -1;
}

// U: 16-byte pieces of each row that a lane keeps in flight.
template <int DT, int WARPS, int U>
__global__ void __launch_bounds__(32 * WARPS, WARPS == 8 ? 5 : 2) k_verify_draft(const VerifyArgs a) {
  constexpr uint32_t SIZE = DT == NRC_F32 ? 4 : 2;
  __shared__ double sums[2][VD_MAX_CLUSTER * WARPS];  // every span's, in each block of the cluster
  __shared__ double fine[WARPS][FINE];                // the groups of this block's spans
  __shared__ uint32_t taken_s;
  cg::cluster_group cluster = cg::this_cluster();
  const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
  const uint32_t b = blockIdx.x / blocks, m = a.n_max;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this block has started
  if (warp == 0) {
    // All drafts at once; the first that is refused counts.
    const int asked = a.n_draft ? a.n_draft[b] : (int)m, nd = asked < 0 ? 0 : asked > (int)m ? (int)m : asked;
    int taken = nd;
    for (int i0 = 0; i0 < (int)m; i0 += 32) {
      const int i = i0 + lane;
      bool refuse = false;
      if (i < (int)m) {
        const int32_t x = a.draft[(size_t)b * m + i];
        const float u = a.u[(size_t)b * (m + 1) + i];
        refuse = i < nd;
        if (refuse && x >= 0 && (uint32_t)x < a.vocab) {
          const float px = load_as_f32(a.p, (int64_t)b * a.p_seq + (int64_t)i * a.p_token + x, DT);
          const float qx = a.q ? load_as_f32(a.q, (int64_t)b * a.q_seq + (int64_t)i * a.q_token + x, DT) : 1.0f;
          refuse = !((double)u * (double)qx < (double)px);
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
  const float u = a.u[(size_t)b * (m + 1) + m];

  __syncwarp();
  asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // all have: their shared memory may be written

  // Spans of whole 16-byte pieces (counted from the row's start), in index order over blocks and warps.
  const uint32_t spans = blocks * WARPS, per = ((a.vocab + spans - 1) / spans + 7) & ~7u;
  auto begin = [&](uint32_t i) { return (uint32_t)min((uint64_t)i * per, (uint64_t)a.vocab); };
  const uint32_t mine = rank * WARPS + warp;
  double total, before;
  int owner;
  for (int round = 0;; round++) {
    const double s = span_sum<DT, U>(row, Span<DT, U>(row, begin(mine), begin(mine + 1)), fine[warp], lane);
    if ((uint32_t)lane < blocks) *cluster.map_shared_rank(&sums[round][mine], lane) = s;
    cluster.sync();
    // Every warp of the cluster reads the same sums and decides alike.
    owner = pick_span(sums[round], spans, (double)u, &total, &before, lane);
    if (owner >= 0 || !refused || round) break;
    row.q = nullptr;  // the difference leaves nothing: p itself
    row.certain = -1;
  }
  uint32_t token = 0;
  if (owner < 0) {
    if (rank || warp) return;  // p holds nothing either
  } else {
    if ((uint32_t)owner != mine) return;
    // The owner's groups, then the tokens of the one that holds the goal.
    const Span<DT, U> sp(row, begin(mine), begin(mine + 1));
    const double goal = (double)u * total;
    const double f = lane < FINE ? fine[warp][lane] : 0.0;
    double run = f;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const double y = __shfl_up_sync(0xffffffffu, run, o);
      if (lane >= o) run += y;
    }
    run += before;
    const unsigned over = __ballot_sync(0xffffffffu, f > 0.0 && run > goal), some = __ballot_sync(0xffffffffu, f > 0.0);
    const int pick = over ? __ffs(over) - 1 : 31 - __clz(some);
    double at = __shfl_up_sync(0xffffffffu, run, 1);
    if (lane == 0) at = before;
    at = over ? __shfl_sync(0xffffffffu, at, pick) : -INFINITY;
    token = span_find<DT>(row, sp.begin(pick), sp.begin(pick + 1), at, goal, lane);
  }
  for (uint32_t i = lane; i <= m; i += 32)
    a.tokens[(size_t)b * (m + 1) + i] = i < taken ? a.draft[(size_t)b * m + i] : i == taken ? (int32_t)token : -1;
  if (lane == 0) a.accepted[b] = (int32_t)taken;
}

template <int DT>
const void* variant(bool many) {
  return many ? (const void*)k_verify_draft<DT, 8, 2> : (const void*)k_verify_draft<DT, 16, 4>;
}

}  // namespace

cudaError_t verify_draft_run(const VerifyArgs& a, cudaStream_t s) {
  // All blocks should be resident at once, or the fixed latency of a block (four dependent reads and the cluster's
  // barrier, some 5 us) is paid again: up to 18 sequences in clusters of 8 wide blocks, at most one per SM; more in
  // narrower blocks, five per SM, in clusters that shrink as the sequences grow in number (640 of the 740 places: clusters
  // do not straddle the SM groups). 37 sequences of 100352, f16: 17.5 us in wide blocks, 13.7 us in narrow ones; 160
  // of 151936, f32: 56 us in clusters of 8, 44 us of 4.
  const bool many = (uint64_t)a.n_seqs * VD_MAX_CLUSTER > 148;
  const uint32_t warps = many ? 8 : 16;
  uint32_t blocks = 1;
  while (blocks < VD_MAX_CLUSTER && (uint64_t)blocks * warps * 512 < a.vocab && (uint64_t)a.n_seqs * blocks * 2 <= 640)
    blocks *= 2;  // and a warp has some 512 tokens
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(a.n_seqs * blocks);
  cfg.blockDim = dim3(32 * warps);
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
  const void* fn = a.dtype == NRC_F32 ? variant<NRC_F32>(many) : a.dtype == NRC_F16 ? variant<NRC_F16>(many) : variant<NRC_BF16>(many);
  return cudaLaunchKernelExC(&cfg, fn, args);
}

}  // namespace nrc
