// Attention of the newest tokens of many sequences over a paged KV cache:
// the kernels, instantiated per cache type by paged_attn_f16.cu and
// paged_attn_bf16.cu and launched by paged_attn.cu.
//
// Mathematics. For query row r (head r % gqa of the KV head's group, new token r / gqa) over the
// cached positions t: s_t = f_r (q_r . K_t) with f_r = scale log2(e), m = max s_t, and
//   out_r = sum_t 2^(s_t - m) V_t / sum_t 2^(s_t - m),
// taken in one pass with the running maximum, sum and accumulators (all f32) rescaled when the
// maximum grows, and joined across warps and blocks by the same rule.
//
// What bounds it: every K and V row is read once and serves 2 FLOPs per query row and value; with up to 32 rows
// that is far below the ratio of tensor to memory rate, so the kernel has to keep HBM busy.
//
// Layout. Both products run transposed, with the cache as the 16-row operand A of mma.m16n8k16 and the query rows as
// its 8 columns: S^T = K Q^T (16 positions x 8 rows) and O^T += V^T P^T (16 values x 8 rows), so that 1..8 rows waste
// nothing more than their tile. The order of the contracted index is free, and A's fragment can be loaded straight
// from global memory in 16-byte pieces:
//   K: lane (g, t) = (lane / 4, lane % 4) reads the values 32 c + 8 t .. + 7 of the positions g and g + 8: two k-steps
//      of A, whose k index 2 t + {0, 1} stands for value 32 c + 8 t + 4 s + {0, 1} and 2 t + 8 + {0, 1} for the two
//      behind them. Q's fragment in shared memory is laid out for the same order.
//   V: lane (g, t) reads the values 64 c + 8 g .. + 7 of the positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9; byte permutes
//      pair neighbouring positions, and row g of the tile j of chunk c stands for value 64 c + 8 g + 2 j, row g + 8 for
//      the one behind it.
// P^T's operand is the transposed accumulator of S^T, turned by movmatrix. No tile passes through shared memory, and a
// warp has 16 positions of K and V in flight while it computes on the ones before. tcgen05 would need the tiles in
// shared memory and 64 or more rows of queries to be fed; here its rate is not what is missing.
//
// Split parts. The tensor cores take operands of the cache's type. q (scaled by a power of two to at most 2 per row) and
// p enter as PARTS values of that type whose sum holds the bits that the output's type can show: one where the output is
// no wider than the cache, two f16 (22 bits) or three bf16 (24 bits) for f32, two bf16 for f16. Products of the parts go to
// the same f32 accumulators.
#pragma once
#include "paged.cuh"

namespace nrc {
namespace pattn {

constexpr int THREADS = 128, WARPS = 4;
constexpr int TILE = 16;             // positions per warp and step
constexpr int UNIT = TILE * WARPS;   // positions per block and step: the unit of the schedule
constexpr int MAX_HD_NT4 = 64;       // 32 query rows at once: wider heads' accumulators do not fit the registers

// What one launch needs beside the arguments.
struct Plan {
  PagedAttnArgs a;
  uint32_t gqa, rows, row_blocks;  // query rows per KV head (gqa * n_new), blocks of 8 * NT of them
  uint32_t blocks;                 // blocks of the attention kernel
  uint32_t direct;                 // one (sequence, KV head, row block) per block: nothing is split
  uint32_t min_units;
  int4* cut;                       // [blocks]: the work that starts in this block and ends in a later one
  float* lse;                      // [n_seqs][n_heads * n_new] (row order), for the weights
  float2* part_ml;                 // [2 * blocks][8 * NT]
  float* part_o;                   // [2 * blocks][8 * NT][head_dim]
  unsigned* err;
};

template <bool BF>
NRC_DEV void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (BF)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
NRC_DEV uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
NRC_DEV float exp2_fast(float x) {  // within 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <bool BF>
NRC_DEV uint32_t pack2(float lo, float hi) {
  if (BF) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
template <bool BF>
NRC_DEV float2 unpack2(uint32_t x) {
  if (BF) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
// PARTS packed pairs whose sums are (x, y).
template <bool BF, int PARTS>
NRC_DEV void split2(float x, float y, uint32_t (&out)[PARTS]) {
#pragma unroll
  for (int i = 0; i < PARTS; i++) {
    out[i] = pack2<BF>(x, y);
    if (i + 1 < PARTS) {
      const float2 v = unpack2<BF>(out[i]);
      x -= v.x;
      y -= v.y;
    }
  }
}

NRC_DEV uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
NRC_DEV uint2 ld_stream8(const void* p) {
  uint2 v;
  asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
  return v;
}

// Cached positions of a sequence, at most max_len (and what the weights hold).
NRC_DEV uint32_t seq_len(const Plan& p, uint32_t b) {
  const int32_t raw = p.a.lens[b];
  const uint32_t most = p.a.weights && p.a.weights_len < p.a.max_len ? p.a.weights_len : p.a.max_len;
  if (raw < 0 || (uint32_t)raw > most) {
    atomicOr(p.err, ERR_BAD_SLOT);
    return raw < 0 ? 0u : most;
  }
  return (uint32_t)raw;
}
// Units of a sequence; an empty one has a unit too, whose block writes its zeros.
NRC_DEV uint32_t units_of(uint32_t len) { return len ? (len + UNIT - 1) / UNIT : 1u; }

// The positions of one tile: element offset of each lane's position (lane & 15), and which of the 16 can be read.
struct TileRows {
  int64_t off;
  uint32_t ok;  // bit r: position r of the tile is cached
};
NRC_DEV TileRows tile_rows(const Plan& p, uint32_t b, int64_t head_off, uint32_t tile, uint32_t len, int lane) {
  const uint32_t pos = tile * TILE + (lane & 15);
  TileRows t;
  t.off = -1;
  if (pos < len) {
    t.off = paged_row(p.a.kv, b, pos);
    if (t.off < 0)
      atomicOr(p.err, ERR_BAD_PAGE);
    else
      t.off += head_off;
  }
  t.ok = __ballot_sync(0xffffffffu, t.off >= 0) & 0xffffu;
  return t;
}

template <int HD>
NRC_DEV void load_k(uint4 (&k)[HD / 32][2], const uint16_t* base, const TileRows& r, int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int64_t off = __shfl_sync(0xffffffffu, r.off, g + 8 * i);
    const uint16_t* p = base + off + 8 * t;
#pragma unroll
    for (int c = 0; c < HD / 32; c++) k[c][i] = off >= 0 ? ld_stream16(p + 32 * c) : make_uint4(0, 0, 0, 0);
  }
}

// V: whole chunks of 64 values as 16-byte pieces, a last chunk of 32 as 8-byte pieces.
template <int HD>
struct VRegs {
  uint4 w[HD / 64 > 0 ? HD / 64 : 1][4];
  uint2 h[4];
};
template <int HD>
NRC_DEV void load_v(VRegs<HD>& v, const uint16_t* base, const TileRows& r, int lane) {
  const int g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int64_t off = __shfl_sync(0xffffffffu, r.off, 2 * t + (i & 1) + 8 * (i >> 1));
    const uint16_t* p = base + off;
#pragma unroll
    for (int c = 0; c < HD / 64; c++) v.w[c][i] = off >= 0 ? ld_stream16(p + 64 * c + 8 * g) : make_uint4(0, 0, 0, 0);
    if (HD % 64) v.h[i] = off >= 0 ? ld_stream8(p + HD - 32 + 4 * g) : make_uint2(0, 0);
  }
}
// Operand A of value tile mt: rows g, g + 8 (two neighbouring values), k = positions.
template <int HD>
NRC_DEV void v_operand(uint32_t (&a)[4], const VRegs<HD>& v, int mt) {
  uint32_t x[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (mt < HD / 64 * 4) {
      const uint4& w = v.w[mt / 4][i];
      x[i] = mt % 4 == 0 ? w.x : mt % 4 == 1 ? w.y : mt % 4 == 2 ? w.z : w.w;
    } else {
      x[i] = mt % 2 == 0 ? v.h[i].x : v.h[i].y;
    }
  }
  a[0] = __byte_perm(x[0], x[1], 0x5410);
  a[1] = __byte_perm(x[0], x[1], 0x7632);
  a[2] = __byte_perm(x[2], x[3], 0x5410);
  a[3] = __byte_perm(x[2], x[3], 0x7632);
}
// The first of the two neighbouring values that rows g and g + 8 of tile mt stand for.
template <int HD>
NRC_DEV int value_of(int mt, int g) {
  return mt < HD / 64 * 4 ? 64 * (mt / 4) + 8 * g + 2 * (mt % 4) : HD - 32 + 4 * g + 2 * (mt % 2);
}

// The row block's queries as operand B of S^T, per k-step and part, and the factor of each row.
template <int HD, int PARTS, int NT>
struct Queries {
  uint2 frag[PARTS][HD / 16][NT][32];
  float factor[8 * NT];
};
template <bool BF, int HD, int PARTS, int NT>
NRC_DEV void load_queries(const Plan& p, uint32_t b, uint32_t h, uint32_t rb, Queries<HD, PARTS, NT>& qs) {
  constexpr int PER_ROW = THREADS / (8 * NT);  // threads of a row (16, 8 or 4), HD / PER_ROW values each
  constexpr int VALUES = HD / PER_ROW;
  const int row = threadIdx.x / PER_ROW, part = threadIdx.x % PER_ROW;
  const uint32_t r = rb * 8 * NT + row;
  const bool real = r < p.rows;
  const uint32_t tok = real ? r / p.gqa : 0, head = h * p.gqa + (real ? r % p.gqa : 0);
  const int64_t at = (int64_t)b * p.a.q_seq + (int64_t)tok * p.a.q_token + (int64_t)head * p.a.q_head + part * VALUES;
  float x[VALUES], big = 0.0f;
#pragma unroll
  for (int i = 0; i < VALUES; i++) {
    x[i] = real ? load_as_f32(p.a.q, at + i, p.a.dtype) : 0.0f;
    big = fmaxf(big, fabsf(x[i]));
  }
#pragma unroll
  for (int o = 1; o < PER_ROW; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
  int e = 0;  // |x| 2^-e < 2; infinities and zeros as they are
  if (big > 0.0f && big < INFINITY) e = ilogbf(big);
#pragma unroll
  for (int i = 0; i < VALUES; i += 2) {
    const float lo = ldexpf(x[i], -e), hi = ldexpf(x[i + 1], -e);
    uint32_t w[PARTS];
    split2<BF, PARTS>(lo, hi, w);
    const int d = part * VALUES + i;  // 32 c + 8 t + 4 s + 2 word
    const int ks = 2 * (d / 32) + (d / 4) % 2, t = (d / 8) % 4, word = (d / 2) % 2;
#pragma unroll
    for (int j = 0; j < PARTS; j++)
      reinterpret_cast<uint32_t*>(&qs.frag[j][ks][row / 8][(row % 8) * 4 + t])[word] = w[j];
  }
  if (part == 0) qs.factor[row] = ldexpf(p.a.scale * 1.44269504088896340736f, e);
}

// S^T of one tile.
template <bool BF, int HD, int PARTS, int NT>
NRC_DEV void scores(float (&s)[NT][4], const uint4 (&k)[HD / 32][2], const Queries<HD, PARTS, NT>& qs, int lane) {
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int i = 0; i < 4; i++) s[n][i] = 0.0f;
#pragma unroll
  for (int c = 0; c < HD / 32; c++)
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint32_t a[4] = {u ? k[c][0].z : k[c][0].x, u ? k[c][1].z : k[c][1].x, u ? k[c][0].w : k[c][0].y,
                             u ? k[c][1].w : k[c][1].y};
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < PARTS; j++) {
          const uint2 q = qs.frag[j][2 * c + u][n][lane];
          mma<BF>(s[n], a, q.x, q.y);
        }
    }
}

// Where block `i` starts, and the units each block takes: sequences in order, in each the (KV head, row
// block) pairs in order, in each its units. Every block finds its start alone, from the lengths.
struct Start {
  uint32_t b, hb, unit;  // sequence, KV head * row_blocks + row block, first unit
  uint64_t left;         // units of work of this block
  uint64_t share, total;
};
NRC_DEV Start find_start(const Plan& p, uint64_t* warp_sums, Start* found) {
  const uint32_t hbs = p.a.kv.n_kv_heads * p.row_blocks, n = p.a.kv.n_seqs;
  const uint32_t per = (n + THREADS - 1) / THREADS, b0 = min(threadIdx.x * per, n), b1 = min(b0 + per, n);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t sum = 0;
  for (uint32_t b = b0; b < b1; b++) sum += units_of(seq_len(p, b));
  uint64_t x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint64_t before = x - sum, all = 0;
  for (int w = 0; w < WARPS; w++) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  const uint64_t total = all * hbs;
  uint64_t share = (total + gridDim.x - 1) / gridDim.x;
  if (share < p.min_units) share = p.min_units;
  const uint64_t start = share * blockIdx.x;
  if (threadIdx.x == 0) found->left = 0, found->share = share, found->total = total;
  __syncthreads();
  if (start < total && start >= before * hbs && start < (before + sum) * hbs) {
    uint64_t at = start - before * hbs;
    uint32_t b = b0, u = units_of(seq_len(p, b));
    while (at >= (uint64_t)u * hbs) {
      at -= (uint64_t)u * hbs;
      u = units_of(seq_len(p, ++b));
    }
    found->b = b;
    found->hb = (uint32_t)(at / u);
    found->unit = (uint32_t)(at % u);
    found->left = min(share, total - start);
  }
  __syncthreads();
  return *found;
}

template <bool BF, int HD, int PARTS, int NT>
__global__ void __launch_bounds__(THREADS, NT == 1 ? 3 : 2) k_attn(const Plan p) {
  constexpr int MT = HD / 16, COLS = 8 * NT;
  // A running sum of p, whose f16 operand has no bits below 2^-24: p is kept 2^14 times larger.
  constexpr float LIFT = BF ? 0.0f : 14.0f;
  __shared__ Queries<HD, PARTS, NT> qs;
  __shared__ __align__(16) float o_s[WARPS][COLS][HD + 2];
  __shared__ float m_s[WARPS][COLS], l_s[WARPS][COLS];
  __shared__ uint64_t warp_sums[WARPS];
  __shared__ Start start_s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t hbs = p.a.kv.n_kv_heads * p.row_blocks;
  Start st;
  if (p.direct) {
    st.b = blockIdx.x / hbs;
    st.hb = blockIdx.x % hbs;
    st.unit = 0;
    st.left = units_of(seq_len(p, st.b));
    st.share = st.left;
  } else {
    st = find_start(p, warp_sums, &start_s);
    if (threadIdx.x == 0) p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  bool first = true;
  while (st.left) {
    const uint32_t b = st.b, h = st.hb / p.row_blocks, rb = st.hb % p.row_blocks;
    const uint32_t len = seq_len(p, b), units = units_of(len), u0 = st.unit;
    const uint32_t u1 = (uint32_t)min((uint64_t)units, u0 + st.left);
    __syncthreads();  // the queries and sums of the work before are read
    load_queries<BF, HD, PARTS, NT>(p, b, h, rb, qs);
    __syncthreads();
    const uint16_t* kb = static_cast<const uint16_t*>(p.a.kv.k);
    const uint16_t* vb = static_cast<const uint16_t*>(p.a.kv.v);
    const int64_t head_off = (int64_t)h * p.a.kv.head_stride;
    float acc[MT][NT][4], m[NT][2], l[NT][2], fac[NT][2];
    uint32_t sees[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint32_t r = rb * COLS + 8 * n + 2 * t + i;
        const uint32_t behind = r < p.rows ? p.a.n_new - 1 - r / p.gqa : 0;
        sees[n][i] = len > behind ? len - behind : 0;
        fac[n][i] = qs.factor[8 * n + 2 * t + i];
        m[n][i] = -INFINITY;
        l[n][i] = 0.0f;
      }
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[j][n][i] = 0.0f;
    const uint32_t all_see = len > p.a.n_new - 1 ? len - (p.a.n_new - 1) : 0;  // every row sees these

    uint4 k[HD / 32][2];
    VRegs<HD> v;
    const uint32_t tiles = min(u1 * WARPS, (len + TILE - 1) / TILE);
    uint32_t tile = u0 * WARPS + warp;
    TileRows now = tile_rows(p, b, head_off, tile, tile < tiles ? len : 0, lane);
    load_k<HD>(k, kb, now, lane);
    load_v<HD>(v, vb, now, lane);
    TileRows next = tile_rows(p, b, head_off, tile + WARPS, tile + WARPS < tiles ? len : 0, lane);
    for (; tile < tiles; tile += WARPS) {
      float s[NT][4];
      scores<BF, HD, PARTS, NT>(s, k, qs, lane);
      load_k<HD>(k, kb, next, lane);
      const uint32_t p0 = tile * TILE;
      const bool whole = now.ok == 0xffffu && p0 + TILE <= all_see;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          s[n][i] *= fac[n][i & 1];
          const uint32_t r = g + 8 * (i >> 1);
          if (!whole && (!((now.ok >> r) & 1) || p0 + r >= sees[n][i & 1])) s[n][i] = -INFINITY;
        }
      float top[NT][2];
      bool grows = false;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          float x = fmaxf(s[n][i], s[n][i + 2]);
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
          x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
          top[n][i] = x;
          grows = grows || x > m[n][i];
        }
      if (__any_sync(0xffffffffu, grows)) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          float f[2];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const float mn = fmaxf(m[n][i], top[n][i]);
            f[i] = m[n][i] == -INFINITY ? 0.0f : exp2_fast(m[n][i] - mn);
            m[n][i] = mn;
            l[n][i] *= f[i];
          }
#pragma unroll
          for (int j = 0; j < MT; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[j][n][i] *= f[i & 1];
        }
      }
      uint32_t pb[NT][PARTS][2];
#pragma unroll
      for (int n = 0; n < NT; n++) {
        float e[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          // A row that has seen nothing yet: its scores are all -inf, any finite maximum gives 0.
          const float ref = m[n][i & 1] == -INFINITY ? 0.0f : m[n][i & 1] - LIFT;
          e[i] = exp2_fast(s[n][i] - ref);
          l[n][i & 1] += e[i];
        }
        uint32_t lo[PARTS], hi[PARTS];
        split2<BF, PARTS>(e[0], e[1], lo);
        split2<BF, PARTS>(e[2], e[3], hi);
#pragma unroll
        for (int j = 0; j < PARTS; j++) {
          pb[n][j][0] = transpose8x8(lo[j]);
          pb[n][j][1] = transpose8x8(hi[j]);
        }
      }
      if (p0 + TILE <= all_see || p.a.n_new == 1) {
#pragma unroll
        for (int j = 0; j < MT; j++) {
          uint32_t a[4];
          v_operand<HD>(a, v, j);
#pragma unroll
          for (int n = 0; n < NT; n++)
#pragma unroll
            for (int i = 0; i < PARTS; i++) mma<BF>(acc[j][n], a, pb[n][i][0], pb[n][i][1]);
        }
      } else {
        // Positions that only some of the new tokens see: 0 times an infinite value must not reach the others, so
        // each token's rows are taken from a product with the values behind it cleared.
        const uint32_t tok0 = rb * COLS / p.gqa, tok1 = min(p.a.n_new, (rb * COLS + COLS - 1) / p.gqa + 1);
        for (uint32_t tok = tok0; tok < tok1; tok++) {
          const uint32_t behind = p.a.n_new - 1 - tok, end = len > behind ? len - behind : 0;
          const uint32_t at = p0 + 2 * t;
          const uint32_t mask0 = (at < end ? 0xffffu : 0u) | (at + 1 < end ? 0xffff0000u : 0u);
          const uint32_t mask1 = (at + 8 < end ? 0xffffu : 0u) | (at + 9 < end ? 0xffff0000u : 0u);
#pragma unroll
          for (int j = 0; j < MT; j++) {
            uint32_t a[4];
            v_operand<HD>(a, v, j);
            a[0] &= mask0, a[1] &= mask0, a[2] &= mask1, a[3] &= mask1;
#pragma unroll
            for (int n = 0; n < NT; n++) {
              float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int i = 0; i < PARTS; i++) mma<BF>(d, a, pb[n][i][0], pb[n][i][1]);
#pragma unroll
              for (int i = 0; i < 4; i++)
                if ((rb * COLS + 8 * n + 2 * t + (i & 1)) / p.gqa == tok) acc[j][n][i] += d[i];
            }
          }
        }
      }
      load_v<HD>(v, vb, next, lane);
      now = next;
      next = tile_rows(p, b, head_off, tile + 2 * WARPS, tile + 2 * WARPS < tiles ? len : 0, lane);
    }

    // Join the warps.
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], o);
        if (g == 0) {
          m_s[warp][8 * n + 2 * t + i] = m[n][i];
          l_s[warp][8 * n + 2 * t + i] = l[n][i];
        }
      }
#pragma unroll
      for (int j = 0; j < MT; j++) {
        const int d = value_of<HD>(j, g);
#pragma unroll
        for (int i = 0; i < 2; i++)
          *reinterpret_cast<float2*>(&o_s[warp][8 * n + 2 * t + i][d]) = make_float2(acc[j][n][i], acc[j][n][i + 2]);
      }
    }
    __syncthreads();
    const bool complete = u0 == 0 && u1 == units;
    const uint32_t slot = 2 * blockIdx.x + (first && u0 ? 0 : 1);
    for (uint32_t i = threadIdx.x; i < COLS * HD; i += THREADS) {
      const uint32_t col = i / HD, d = i % HD, r = rb * COLS + col;
      if (r >= p.rows) break;
      float mx = -INFINITY, o = 0.0f, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < WARPS; w++) mx = fmaxf(mx, m_s[w][col]);
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float f = m_s[w][col] == -INFINITY ? 0.0f : exp2_fast(m_s[w][col] - mx);
        sum += f * l_s[w][col];
        o += f * o_s[w][col][d];
      }
      if (complete) {
        const uint32_t tok = r / p.gqa, head = h * p.gqa + r % p.gqa;
        store_from_f32(p.a.out, (int64_t)b * p.a.o_seq + (int64_t)tok * p.a.o_token + (int64_t)head * p.a.o_head + d,
                       p.a.dtype, mx == -INFINITY ? 0.0f : o / sum);
        if (d == 0 && p.lse) p.lse[((size_t)b * p.a.kv.n_kv_heads + h) * p.rows + r] = mx - LIFT + log2f(sum);
      } else {
        p.part_o[((size_t)slot * COLS + col) * HD + d] = o;
        if (d == 0) p.part_ml[(size_t)slot * COLS + col] = make_float2(mx, sum);
      }
    }
    // Work that starts here and goes on: the join kernel's item, with the blocks that hold its parts.
    if (u1 < units && !(first && u0) && threadIdx.x == 0) {
      const uint64_t rest = units - u1;
      p.cut[blockIdx.x] = make_int4((int)b, (int)st.hb, (int)(1 + (rest + st.share - 1) / st.share), 0);
    }
    first = false;
    st.left -= u1 - u0;
    st.unit = 0;
    if (++st.hb == hbs) {
      st.hb = 0;
      st.b++;
    }
  }
  pdl_trigger();
}

// One block per (attention block whose last work goes on, row): the parts' running maxima and sums joined.
template <int HD>
__global__ void __launch_bounds__(HD) k_join(const Plan p, int cols, float lift) {
  pdl_wait();
  const int4 cut = p.cut[blockIdx.x];
  const uint32_t b = cut.x, h = cut.y / p.row_blocks, rb = cut.y % p.row_blocks, n = cut.z;
  const uint32_t col = blockIdx.y, r = rb * cols + col;
  if (n == 0 || r >= p.rows) return;
  // The first part is the last work of its block, the others the first of theirs.
  auto slot = [&](uint32_t i) { return ((size_t)2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * cols + col; };
  float mx = -INFINITY;
  for (uint32_t i = 0; i < n; i++) mx = fmaxf(mx, p.part_ml[slot(i)].x);
  float o = 0.0f, sum = 0.0f;
#pragma unroll 4
  for (uint32_t i = 0; i < n; i++) {
    const float2 ml = p.part_ml[slot(i)];
    const float f = ml.x == -INFINITY ? 0.0f : exp2_fast(ml.x - mx);
    sum += f * ml.y;
    o += f * p.part_o[slot(i) * HD + threadIdx.x];
  }
  const uint32_t tok = r / p.gqa, head = h * p.gqa + r % p.gqa;
  store_from_f32(p.a.out, (int64_t)b * p.a.o_seq + (int64_t)tok * p.a.o_token + (int64_t)head * p.a.o_head + threadIdx.x,
                 p.a.dtype, mx == -INFINITY ? 0.0f : o / sum);
  if (threadIdx.x == 0 && p.lse) p.lse[((size_t)b * p.a.kv.n_kv_heads + h) * p.rows + r] = mx - lift + log2f(sum);
}

// Weights: the scores again (the same products, the same bits), 2^(s - lse) summed over the query rows in
// a fixed order and added. One warp per tile of 16 positions of a (sequence, KV head); a block's tiles are
// the units x, x + gridDim.x, ...
template <bool BF, int HD, int PARTS, int NT>
__global__ void __launch_bounds__(THREADS) k_weights(const Plan p) {
  constexpr int COLS = 8 * NT;
  __shared__ Queries<HD, PARTS, NT> qs;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  pdl_wait();
  const uint32_t h = blockIdx.y, b = blockIdx.z;
  const uint32_t len = seq_len(p, b), units = (len + UNIT - 1) / UNIT;
  const uint16_t* kb = static_cast<const uint16_t*>(p.a.kv.k);
  float* w = p.a.weights + ((size_t)b * p.a.kv.n_kv_heads + h) * p.a.weights_len;
  for (uint32_t rb = 0; rb < p.row_blocks; rb++) {
    if (blockIdx.x >= units) return;
    __syncthreads();
    load_queries<BF, HD, PARTS, NT>(p, b, h, rb, qs);
    __syncthreads();
    float fac[NT][2], lse[NT][2];
    uint32_t sees[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        const uint32_t r = rb * COLS + 8 * n + 2 * t + i;
        const uint32_t behind = r < p.rows ? p.a.n_new - 1 - r / p.gqa : 0;
        sees[n][i] = r < p.rows && len > behind ? len - behind : 0;
        fac[n][i] = qs.factor[8 * n + 2 * t + i];
        lse[n][i] = sees[n][i] ? p.lse[((size_t)b * p.a.kv.n_kv_heads + h) * p.rows + r] : 0.0f;
      }
    for (uint32_t unit = blockIdx.x; unit < units; unit += gridDim.x) {
      const uint32_t tile = unit * WARPS + warp, p0 = tile * TILE;
      const TileRows now = tile_rows(p, b, (int64_t)h * p.a.kv.head_stride, tile, len, lane);
      uint4 k[HD / 32][2];
      load_k<HD>(k, kb, now, lane);
      float s[NT][4], sum[2] = {0.0f, 0.0f};
      scores<BF, HD, PARTS, NT>(s, k, qs, lane);
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) {
          const uint32_t r = g + 8 * (i >> 1);
          if (((now.ok >> r) & 1) && p0 + r < sees[n][i & 1] && lse[n][i & 1] != -INFINITY)
            sum[i >> 1] += exp2_fast(s[n][i] * fac[n][i & 1] - lse[n][i & 1]);
        }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
        const uint32_t r = g + 8 * i;
        if (t == 0 && ((now.ok >> r) & 1)) w[p0 + r] += sum[i];
      }
    }
  }
}

template <bool BF, int HD, int PARTS, int NT>
cudaError_t launch(Plan& p, cudaStream_t s) {
  void* args[] = {&p};
  if (cudaError_t e = launch_kernel((const void*)k_attn<BF, HD, PARTS, NT>, dim3(p.blocks), dim3(THREADS), 0, s, false, args))
    return e;
  if (!p.direct) {
    int cols = 8 * NT;
    float lift = BF ? 0.0f : 14.0f;
    void* jargs[] = {&p, &cols, &lift};
    const uint32_t rows = p.rows < (uint32_t)cols ? p.rows : (uint32_t)cols;
    if (cudaError_t e = launch_kernel((const void*)k_join<HD>, dim3(p.blocks, rows), dim3(HD), 0, s, true, jargs)) return e;
  }
  if (p.a.weights) {
    const uint32_t units = (p.a.max_len + UNIT - 1) / UNIT, pairs = p.a.kv.n_kv_heads * p.a.kv.n_seqs;
    uint32_t x = (16 * 148 + pairs - 1) / pairs;
    if (x > units) x = units;
    if (x == 0) return cudaSuccess;
    return launch_kernel((const void*)k_weights<BF, HD, PARTS, NT>, dim3(x, p.a.kv.n_kv_heads, p.a.kv.n_seqs), dim3(THREADS), 0,
                         s, true, args);
  }
  return cudaSuccess;
}
template <bool BF, int HD, int PARTS>
cudaError_t launch_nt(Plan& p, int nt, cudaStream_t s) {
  if (nt == 1) return launch<BF, HD, PARTS, 1>(p, s);
  if constexpr (HD <= MAX_HD_NT4)
    if (nt == 4) return launch<BF, HD, PARTS, 4>(p, s);
  return launch<BF, HD, PARTS, 2>(p, s);
}
template <bool BF, int PARTS>
cudaError_t launch_hd(Plan& p, int nt, cudaStream_t s) {
  switch (p.a.kv.head_dim) {
    case 32: return launch_nt<BF, 32, PARTS>(p, nt, s);
    case 64: return launch_nt<BF, 64, PARTS>(p, nt, s);
    case 96: return launch_nt<BF, 96, PARTS>(p, nt, s);
    case 128: return launch_nt<BF, 128, PARTS>(p, nt, s);
  }
  return cudaErrorInvalidValue;
}

}  // namespace pattn

// One per cache type and number of parts.
cudaError_t paged_attn_f16_1(pattn::Plan& p, int nt, cudaStream_t s);
cudaError_t paged_attn_f16_2(pattn::Plan& p, int nt, cudaStream_t s);
cudaError_t paged_attn_bf16_1(pattn::Plan& p, int nt, cudaStream_t s);
cudaError_t paged_attn_bf16_2(pattn::Plan& p, int nt, cudaStream_t s);
cudaError_t paged_attn_bf16_3(pattn::Plan& p, int nt, cudaStream_t s);

}  // namespace nrc
