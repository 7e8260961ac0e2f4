// Attention of the newest tokens of many sequences over a paged KV cache:
// the kernels for up to 8 query rows per KV head (and for shapes that
// paged_attn_tc.cuh does not take), instantiated per cache type and number of
// parts by paged_attn_*_*.cu and launched by paged_attn.cu.
//
// Mathematics. For query row r (head r % gqa of the KV head's group, new token r / gqa) over the
// cached positions t: s_t = f_r (q_r . K_t) with f_r = scale log2(e), m = max s_t, and
//   out_r = sum_t 2^(s_t - m) V_t / sum_t 2^(s_t - m),
// taken in one pass with the running maximum, sum and accumulators (all f32) rescaled when the
// maximum grows, and joined across warps and blocks by the same rule.
//
// What bounds it: every K and V row is read once and serves 2 FLOPs per query row and value; that is far below the ratio
// of tensor to memory rate, so the kernel has to keep HBM busy.
//
// Layout. Both products run transposed, with the cache as the 16-row operand A of mma.m16n8k16 and the query rows as
// its 8 columns: S^T = K Q^T (16 positions x 8 rows) and O^T += V^T P^T (16 values x 8 rows), so that 1..8 rows waste
// nothing more than their tile. The order of the contracted index is free, so a lane's share of an operand can be
// whole 16-byte pieces of cached rows:
//   K: lane (g, t) = (lane / 4, lane % 4) holds the values 32 c + 8 t .. + 7 of the positions g and g + 8: two k-steps
//      of A, whose k index 2 t + {0, 1} stands for value 32 c + 8 t + 4 s + {0, 1} and 2 t + 8 + {0, 1} for the two
//      behind them. Q's fragment in shared memory is laid out for the same order.
//   V: lane (g, t) holds the values 64 c + 8 g .. + 7 of the positions 2 t, 2 t + 1, 2 t + 8, 2 t + 9; byte permutes
//      pair neighbouring positions, and row g of the tile j of chunk c stands for value 64 c + 8 g + 2 j, row g + 8 for
//      the one behind it.
// P^T's operand is the transposed accumulator of S^T, turned by movmatrix. No tile passes through shared memory: the
// pieces of the next tile are loaded into the registers of the one before as soon as those are used, 8 KB (of
// 128-wide f16 heads) per warp in flight. (Pieces copied ahead into shared memory, 190 KB per SM in flight, were
// slower: 248 against 199 us for 983 MB. It is the warps' instructions per tile that count, not the bytes in
// flight.) For a few rows the rate of tcgen05 is not what is missing, and its tiles would have to pass through shared
// memory. Measured: 64 sequences of 4096, 32/8 heads of 128, bf16: 168 us, 6.4 TB/s (0.98 of measured); 64 ragged ones up to
// 16384: 161 us (0.94); one of 131072, f16: 88 us (0.94) and the join 8 us more.
//
// Split parts. The tensor cores take operands of the cache's type. q (scaled by a power of two to at most 2 per row) enters
// as PARTS values of that type whose sum holds its bits: one where it is no wider than the cache, two bf16 for f16, three
// bf16 for f32 (24 bits), two f16 for f32 (22 bits, of a row's largest value: f16's smallest step ends them 2^-25 below
// it). The weights p enter in as many, two at least (16 or 22 bits): in one part each weight would be rounded to the output's own
// width and the output be some 30% further off (f16: 2.5e-4 instead of 2.1e-4 of it, bf16: 2.1e-3 instead of 1.7e-3); the
// second costs 1 to 4% (bf16: 64 sequences of 4096 169 and 170 us, 16 with 8 new tokens on tcgen05 84 and 88 us). Products of the parts go to the same f32 accumulators.
#pragma once
#include "paged.cuh"
#include "tma.cuh"

namespace nrc {
namespace pattn {

constexpr int THREADS = 128, WARPS = 4;
constexpr int TILE = 16;             // positions per warp and step
constexpr int UNIT = TILE * WARPS;   // positions per block and step: the unit of the schedule
// Blocks per SM, by the registers.
constexpr int WEIGHTS_RESIDENT = 4;
constexpr int resident(int hd, int nt) { return nt > 1 ? 2 : hd <= 32 ? 4 : 3; }

// What one launch needs beside the arguments.
struct Plan {
  CUtensorMap k_map, v_map;        // tc: [page][KV head][position][value] of K and V
  PagedAttnArgs a;
  uint32_t gqa, rows, row_blocks;  // query rows per KV head (gqa * n_new), blocks of 8 * NT of them
  uint32_t blocks;                 // blocks of the attention kernel
  uint32_t weight_blocks;          // blocks of the weights' kernel
  uint32_t tc;                     // many rows: the kernel of paged_attn_tc.cuh
  uint32_t tc_rows, tc_tile;       // its copies' positions, and its tiles'
  uint32_t direct;                 // one (sequence, KV head, row block) per block: nothing is split
  uint32_t min_units;
  int4* cut;                       // [blocks]: the work that starts in this block and ends in a later one
  float* lse;                      // [n_seqs][n_heads * n_new] (row order), for the weights
  float2* part_nl;                 // [2 * blocks][8 * NT]: reference and sum
  float* part_o;                   // [2 * blocks][8 * NT][head_dim]
  uint32_t step_pages, step_off;   // UNIT positions in pages and the rest
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
// The tensor cores cut the low bits of their sums off, always towards zero (over 64000 positions that came to 5e-5 of the
// output), so sums over many tiles are formed outside of them.
NRC_DEV void add4(float (&to)[4], const float (&d)[4]) {
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    const float2 s = __fadd2_rn(make_float2(to[i], to[i + 1]), make_float2(d[i], d[i + 1]));
    to[i] = s.x;
    to[i + 1] = s.y;
  }
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
constexpr int weight_parts(int parts) { return parts < 2 ? 2 : parts; }
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

NRC_DEV uint4 ldg16(const void* p) {
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
NRC_DEV uint2 ldg8(const void* p) {
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
NRC_DEV uint32_t units_of(uint32_t len, uint32_t unit = UNIT) { return len ? (len + unit - 1) / unit : 1u; }
// What a (sequence, KV head, row block) costs its first block beside its units: the queries, the first tiles' latency, the
// join. Counted in units, so that a share of many short sequences is not longer than one of a long sequence's middle (64
// ragged sequences: 188 us uncounted, 158 us). On tcgen05, 24 sequences of 1000..9001, 5 new tokens, calls of us at 6, 14 and
// 20 units, then what the weights' pass adds at 3, 6 and 12: 40/8 heads of 64, f32 over f16 99, 92, 96 and 54, 45, 45; bf16 102, 101, 101
// and 49, 44, 52; 32/8 heads of 128, f16 133, 137, 137 and 75, 65, 72; f32 over bf16 146, 147, 147 and 79, 71, 73; 64 of 300..4000 with 4 new
// tokens, bf16 167, 173, 188 and 124, 89, 88. Wide heads' tiles cost more each, so they would do with fewer.
constexpr uint32_t SETUP = 2, TC_SETUP = 14, TC_WEIGHTS_SETUP = 6;
constexpr int TC_TILE = 128;         // rows of a tile of the tcgen05 kernel

// K pieces of a tile: [chunk of 32 values][position g or g + 8].
template <int HD>
struct KTile {
  uint4 w[HD / 32][2];
};
// V pieces of a tile: whole chunks of 64 values (16 bytes per position), a last chunk of 32 (8 bytes).
template <int HD>
struct VTile {
  uint4 w[HD / 64 > 0 ? HD / 64 : 1][4];
  uint2 h[4];
  // Operand A of value tile mt: rows g, g + 8 (two neighbouring values), k = positions.
  NRC_DEV void operand(uint32_t (&a)[4], int mt) const {
    uint32_t x[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      if (mt < HD / 64 * 4) {
        const uint4& q = w[mt / 4][i];
        x[i] = mt % 4 == 0 ? q.x : mt % 4 == 1 ? q.y : mt % 4 == 2 ? q.z : q.w;
      } else {
        x[i] = mt % 2 == 0 ? h[i].x : h[i].y;
      }
    }
    a[0] = __byte_perm(x[0], x[1], 0x5410);
    a[1] = __byte_perm(x[0], x[1], 0x7632);
    a[2] = __byte_perm(x[2], x[3], 0x5410);
    a[3] = __byte_perm(x[2], x[3], 0x7632);
  }
  // Whether an infinity or NaN stands among the pieces.
  template <bool BF>
  NRC_DEV bool odd() const {
    constexpr uint32_t EXP = BF ? 0x7f807f80u : 0x7c007c00u;
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; i++) {
#pragma unroll
      for (int c = 0; c < HD / 64; c++)
        any = any || __vcmpeq2(w[c][i].x & EXP, EXP) || __vcmpeq2(w[c][i].y & EXP, EXP) || __vcmpeq2(w[c][i].z & EXP, EXP) ||
              __vcmpeq2(w[c][i].w & EXP, EXP);
      if (HD % 64) any = any || __vcmpeq2(h[i].x & EXP, EXP) || __vcmpeq2(h[i].y & EXP, EXP);
    }
    return any;
  }
};

// A warp's way through its tiles, every WARPS-th from `tile` on below position `end`. Where pages are whole tiles
// (page_size % 16 == 0) one lookup, alike in all lanes, serves a tile; else each lane looks its position up.
struct Walk {
  const uint8_t *k, *v;    // the KV head's first row, this lane's pieces
  const int32_t* table;
  int64_t row;             // byte offset of the current tile's first row (or of this lane's)
  int64_t step;            // bytes between positions
  uint32_t end, pos;       // pos: of the tile looked up next (its first, or this lane's own)
  uint32_t pi, off;        // page index and offset of pos
  int32_t page;            // table[pi], read one tile ahead
  uint32_t ok;             // positions of the current tile that can be read, as bits
  bool in_page;
  bool bad;                // a page outside the pool was met: tiles have to be masked by cached()

  NRC_DEV void fetch() { page = pos < end ? table[pi] : 0; }
  NRC_DEV void begin(const Plan& p, uint32_t b, uint32_t h, uint32_t tile, uint32_t end_, int lane) {
    const int g = lane >> 2, t = lane & 3;
    step = p.a.kv.pos_stride * 2;
    in_page = p.a.kv.page_size % TILE == 0;
    k = static_cast<const uint8_t*>(p.a.kv.k) + (int64_t)h * p.a.kv.head_stride * 2 + 16 * t + (in_page ? g * step : 0);
    v = static_cast<const uint8_t*>(p.a.kv.v) + (int64_t)h * p.a.kv.head_stride * 2 + 16 * g + (in_page ? 2 * t * step : 0);
    table = p.a.kv.table + (size_t)b * p.a.kv.table_stride;
    end = end_;
    bad = false;
    pos = tile * TILE + (in_page ? 0 : lane & 15);
    pi = pos / p.a.kv.page_size;
    off = pos - pi * p.a.kv.page_size;
    fetch();
  }
  // Makes the tile at `pos` the current one and moves on.
  NRC_DEV void next(const Plan& p) {
    const bool live = pos < end, found = (uint32_t)page < p.a.kv.n_pages;
    row = ((int64_t)page * p.a.kv.page_stride + (int64_t)off * p.a.kv.pos_stride) * 2;
    if (in_page) {
      ok = !live || !found ? 0u : end - pos < TILE ? (1u << (end - pos)) - 1u : 0xffffu;
      if (live && !found) bad = true;
    } else {
      ok = __ballot_sync(0xffffffffu, live && found) & 0xffffu;
      if (__any_sync(0xffffffffu, live && !found)) bad = true;
    }
    if (live && !found) atomicOr(p.err, ERR_BAD_PAGE);
    pos += UNIT;
    pi += p.step_pages;
    off += p.step_off;
    if (off >= p.a.kv.page_size) {
      off -= p.a.kv.page_size;
      pi++;
    }
    fetch();
  }
  template <int HD>
  NRC_DEV void load_k(KTile<HD>& t, int lane) const {
    const int g = lane >> 2;
    const uint8_t *p0, *p1;
    if (in_page) {
      p0 = k + row;
      p1 = p0 + 8 * step;
    } else {
      p0 = k + __shfl_sync(0xffffffffu, row, g);
      p1 = k + __shfl_sync(0xffffffffu, row, g + 8);
    }
    if (ok == 0xffffu) {
#pragma unroll
      for (int c = 0; c < HD / 32; c++) t.w[c][0] = ldg16(p0 + 64 * c), t.w[c][1] = ldg16(p1 + 64 * c);
    } else {
#pragma unroll
      for (int i = 0; i < 2; i++)
#pragma unroll
        for (int c = 0; c < HD / 32; c++)
          t.w[c][i] = (ok >> (g + 8 * i)) & 1 ? ldg16((i ? p1 : p0) + 64 * c) : make_uint4(0, 0, 0, 0);
    }
  }
  template <int HD>
  NRC_DEV void load_v(VTile<HD>& t, int lane) const {
    const int g = lane >> 2, q = lane & 3;
    const uint8_t* pr[4];
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const int r = (i & 1) + 8 * (i >> 1);
      pr[i] = v + (in_page ? row + r * step : __shfl_sync(0xffffffffu, row, 2 * q + r));
    }
    if (ok == 0xffffu) {
#pragma unroll
      for (int i = 0; i < 4; i++) {
#pragma unroll
        for (int c = 0; c < HD / 64; c++) t.w[c][i] = ldg16(pr[i] + 128 * c);
        if (HD % 64) t.h[i] = ldg8(pr[i] + 2 * (HD - 32) - 8 * g);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const bool there = (ok >> (2 * q + (i & 1) + 8 * (i >> 1))) & 1;
#pragma unroll
        for (int c = 0; c < HD / 64; c++) t.w[c][i] = there ? ldg16(pr[i] + 128 * c) : make_uint4(0, 0, 0, 0);
        if (HD % 64) t.h[i] = there ? ldg8(pr[i] + 2 * (HD - 32) - 8 * g) : make_uint2(0, 0);
      }
    }
  }
  // Which positions of a tile are cached, where a bad page was met.
  NRC_DEV uint32_t cached(const Plan& p, uint32_t b, uint32_t p0, int lane) const {
    const uint32_t at = p0 + (lane & 15);
    return __ballot_sync(0xffffffffu, at < end && paged_row(p.a.kv, b, at) >= 0) & 0xffffu;
  }
};

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

// A score's exponential is taken as 2^(s + ref): ref is LIFT less the largest score seen when the row's reference was last
// set, and is set again (its sums rescaled) when an exponent passes LIFT + SLACK, so most tiles need no reduction over
// their positions. f16 weights: up to 2^15, and with bits down to 2^-24, 2^-32 of the row's sum. UNSET: nothing seen.
constexpr float SLACK = 7.0f, LIFT = 8.0f, UNSET = 3e38f;

// q . K_t in f32, value after value, of the query row that begins at element `at` and a cached row: the definition's way, for
// what the tensor cores' operands cannot hold. q as it was given.
template <bool BF, int HD>
NRC_DEV float dot_row(const Plan& p, int64_t at, const uint4* k) {
  float d = 0.0f;
#pragma unroll 4
  for (int c = 0; c < HD / 8; c++) {
    const uint4 w = k[c];
#pragma unroll
    for (int e = 0; e < 8; e++) d = fmaf(load_as_f32(p.a.q, at + 8 * c + e, p.a.dtype), load_as_f32(&w, e, BF ? NRC_BF16 : NRC_F16), d);
  }
  return d;
}
NRC_DEV int64_t query_row(const Plan& p, uint32_t b, uint32_t h, uint32_t r) {
  return (int64_t)b * p.a.q_seq + (int64_t)(r / p.gqa) * p.a.q_token + (int64_t)(h * p.gqa + r % p.gqa) * p.a.q_head;
}
NRC_DEV const uint4* cached_row(const void* rows, int64_t row, const Plan& p, uint32_t h) {
  return reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(rows) + row + (int64_t)h * p.a.kv.head_stride);
}

// What position t receives from the query rows [r0, r1), formed anew in f32 where the tensor cores' sum is no number: an
// infinite key times the zeros of a column that is no row is NaN there, and so is an infinite key times the parts of a split
// query. A row that is NaN itself leaves NaN.
template <bool BF, int HD>
__device__ __noinline__ float weight_again(const Plan& p, uint32_t b, uint32_t h, uint32_t r0, uint32_t r1, uint32_t len, uint32_t t) {
  const float* lse = p.lse + ((size_t)b * p.a.kv.n_kv_heads + h) * p.rows;
  const int64_t row = paged_row(p.a.kv, b, t);
  float sum = 0.0f;
  for (uint32_t r = r0; r < r1 && sum == sum; r++) {
    const float l = lse[r];
    if (t + (p.a.n_new - 1 - r / p.gqa) >= len || l == -INFINITY) continue;
    const float d = l == l ? dot_row<BF, HD>(p, query_row(p, b, h, r), cached_row(p.a.kv.k, row, p, h)) : l;
    sum += exp2_fast(fmaf(d, p.a.scale * 1.44269504088896340736f, -l));
  }
  return sum;
}

// A row of a piece of work, the positions [begin, end), formed anew in f32 by one warp where the tensor cores' sums are no
// numbers: there an infinite key or value meets the parts of a split operand (inf - inf), a weight that 16 bits round to 0,
// or the weight 0 of a row that does not see it. Here it counts by IEEE's rules: a score of -inf has weight 0, an infinite
// value of weight above 0 is the output's, a position that the row does not see is left out. Written where the piece's
// results go: to part_row of the partial results, or (part_row < 0) to the output. A lane takes a position for the scores, HD / 32
// values for the sums.
template <bool BF, int HD>
__device__ __noinline__ void row_again(const Plan& p, uint32_t b, uint32_t h, uint32_t r, uint32_t begin, uint32_t end,
                                       int64_t part_row) {
  constexpr int VALUES = HD / 32;
  const int lane = threadIdx.x & 31;
  const uint32_t len = seq_len(p, b), behind = p.a.n_new - 1 - r / p.gqa;
  end = min(end, len > behind ? len - behind : 0);
  auto score = [&](uint32_t t, int64_t& row) {
    row = t < end ? paged_row(p.a.kv, b, t) : -1;
    if (row < 0) return -INFINITY;
    return dot_row<BF, HD>(p, query_row(p, b, h, r), cached_row(p.a.kv.k, row, p, h)) * (p.a.scale * 1.44269504088896340736f);
  };
  float top = -INFINITY, sum = 0.0f, o[VALUES] = {};
  int64_t row;
  bool none = false;  // no number: a score of NaN or +inf
  for (uint32_t t0 = begin; t0 < end && !none; t0 += 32) {
    const float s = score(t0 + lane, row);
    top = fmaxf(top, s);
    none = __any_sync(0xffffffffu, !(s < INFINITY));
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, i));
  const float low = none || top == -INFINITY ? UNSET : -top;
  for (uint32_t t0 = begin; t0 < end && !none; t0 += 32) {
    const float s = score(t0 + lane, row), e = exp2_fast(s + low);
    sum += e;
    float part[VALUES] = {};
    for (uint32_t j = 0; j < min(32u, end - t0); j++) {
      const int64_t at = __shfl_sync(0xffffffffu, row, j);
      const float weight = __shfl_sync(0xffffffffu, e, j);
      if (at < 0) continue;
#pragma unroll
      for (int i = 0; i < VALUES; i++)
        part[i] = fmaf(weight, load_as_f32(cached_row(p.a.kv.v, at, p, h), lane + 32 * i, BF ? NRC_BF16 : NRC_F16), part[i]);
    }
#pragma unroll
    for (int i = 0; i < VALUES; i++) o[i] += part[i];
  }
#pragma unroll
  for (int i = 16; i > 0; i >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, i);
  if (none) sum = __int_as_float(0x7fffffff);
#pragma unroll
  for (int i = 0; i < VALUES; i++) {
    if (none) o[i] = sum;
    if (part_row < 0)
      store_from_f32(p.a.out,
                     (int64_t)b * p.a.o_seq + (int64_t)(r / p.gqa) * p.a.o_token + (int64_t)(h * p.gqa + r % p.gqa) * p.a.o_head + lane + 32 * i,
                     p.a.dtype, sum == 0.0f ? 0.0f : o[i] / sum);
    else
      p.part_o[part_row * HD + lane + 32 * i] = o[i];
  }
  if (lane) return;
  if (part_row >= 0)
    p.part_nl[part_row] = make_float2(low, sum);
  else if (p.lse)
    p.lse[((size_t)b * p.a.kv.n_kv_heads + h) * p.rows + r] = log2f(sum) - low;
}

// S^T of a tile. Few columns: two chains of products, so that one's latency hides the other's.
template <bool BF, int HD, int PARTS, int NT>
NRC_DEV void scores(float (&s)[NT][4], const KTile<HD>& k, const Queries<HD, PARTS, NT>& qs, int lane) {
  constexpr int CHAINS = NT == 1 ? 2 : 1;
  float x[CHAINS][NT][4];
#pragma unroll
  for (int u = 0; u < CHAINS; u++)
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 4; i++) x[u][n][i] = 0.0f;
#pragma unroll
  for (int c = 0; c < HD / 32; c++) {
    const uint4 k0 = k.w[c][0], k1 = k.w[c][1];
#pragma unroll
    for (int u = 0; u < 2; u++) {
      const uint32_t a[4] = {u ? k0.z : k0.x, u ? k1.z : k1.x, u ? k0.w : k0.y, u ? k1.w : k1.y};
#pragma unroll
      for (int j = 0; j < PARTS; j++)
#pragma unroll
        for (int n = 0; n < NT; n++) {
          const uint2 q = qs.frag[j][2 * c + u][n][lane];
          mma<BF>(x[u % CHAINS][n], a, q.x, q.y);
        }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; n++)
#pragma unroll
    for (int i = 0; i < 4; i++) s[n][i] = CHAINS == 2 ? x[0][n][i] + x[CHAINS - 1][n][i] : x[0][n][i];
}

// Where block `i` starts, and the units each block takes: sequences in order, in each the (KV head, row
// block) pairs in order (hbs of them), in each its units. Every block finds its start alone, from the lengths.
struct Start {
  uint32_t b, hb, unit;  // sequence, pair, first unit (SETUP units that are no work come first)
  uint64_t left;         // units of work of this block
  uint64_t share, total;
};
template <int T = THREADS>
NRC_DEV Start find_start(const Plan& p, uint32_t hbs, uint32_t unit, uint32_t setup, uint64_t* warp_sums, Start* found) {
  const uint32_t n = p.a.kv.n_seqs;
  const uint32_t per = (n + T - 1) / T, b0 = min(threadIdx.x * per, n), b1 = min(b0 + per, n);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint64_t sum = 0;
  for (uint32_t b = b0; b < b1; b++) sum += setup + units_of(seq_len(p, b), unit);
  uint64_t x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) warp_sums[warp] = x;
  __syncthreads();
  uint64_t before = x - sum, all = 0;
  for (int w = 0; w < T / 32; w++) {
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
    uint32_t b = b0, u = setup + units_of(seq_len(p, b), unit);
    while (at >= (uint64_t)u * hbs) {
      at -= (uint64_t)u * hbs;
      u = setup + units_of(seq_len(p, ++b), unit);
    }
    found->b = b;
    found->hb = (uint32_t)(at / u);
    found->unit = (uint32_t)(at % u);
    found->left = min(share, total - start);
  }
  __syncthreads();
  return *found;
}

// Exponentials of 8 columns' scores, added to the rows' sums, as operand B of O^T.
template <bool BF, int PARTS>
NRC_DEV void weights_operand(uint32_t (&pb)[PARTS][2], const float (&s)[4], const float (&ref)[2], float (&l)[2]) {
  float e[4];
#pragma unroll
  for (int i = 0; i < 4; i++) {
    e[i] = exp2_fast(s[i] + ref[i & 1]);
    l[i & 1] += e[i];
  }
  uint32_t lo[PARTS], hi[PARTS];
  split2<BF, PARTS>(e[0], e[1], lo);
  split2<BF, PARTS>(e[2], e[3], hi);
#pragma unroll
  for (int j = 0; j < PARTS; j++) {
    pb[j][0] = transpose8x8(lo[j]);
    pb[j][1] = transpose8x8(hi[j]);
  }
}

template <bool BF, int HD, int PARTS, int NT>
__global__ void __launch_bounds__(THREADS, resident(HD, NT)) k_attn(const __grid_constant__ Plan p) {
  constexpr int MT = HD / 16, COLS = 8 * NT, WP = weight_parts(PARTS);
  extern __shared__ __align__(16) uint8_t dyn_s[];  // the warps' sums, to be joined
  __shared__ Queries<HD, PARTS, NT> qs;
  __shared__ float n_s[WARPS][COLS], l_s[WARPS][COLS];
  __shared__ uint64_t warp_sums[WARPS];
  __shared__ Start start_s;
  __shared__ uint32_t odd_s;  // columns whose sums are no numbers
  float(*o_s)[COLS][HD + 2] = reinterpret_cast<float(*)[COLS][HD + 2]>(dyn_s);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t hbs = p.a.kv.n_kv_heads * p.row_blocks;
  if (threadIdx.x == 0) odd_s = 0;
  pdl_trigger();  // the join waits for this grid's end by itself
  Start st;
  if (p.direct) {
    st.b = blockIdx.x / hbs;
    st.hb = blockIdx.x % hbs;
    st.unit = 0;
    st.left = SETUP + units_of(seq_len(p, st.b));
    st.share = st.left;
  } else {
    st = find_start(p, hbs, UNIT, SETUP, warp_sums, &start_s);
    if (threadIdx.x == 0) p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  bool first = true;
  while (st.left) {
    const uint32_t b = st.b, h = st.hb / p.row_blocks, rb = st.hb % p.row_blocks;
    const uint32_t len = seq_len(p, b), units = units_of(len);
    const uint32_t v0 = st.unit, v1 = (uint32_t)min((uint64_t)(SETUP + units), v0 + st.left);
    const uint32_t u0 = v0 > SETUP ? v0 - SETUP : 0, u1 = v1 > SETUP ? v1 - SETUP : 0;
    if (u1 == 0) break;  // the share ends before the first unit: the next block's work
    __syncthreads();  // the queries and sums of the work before are read
    const uint32_t end = min(u1 * UNIT, len);
    Walk walk;
    walk.begin(p, b, h, u0 * WARPS + warp, end, lane);
    KTile<HD> k;
    VTile<HD> v;
    walk.next(p);
    walk.load_k<HD>(k, lane);
    walk.load_v<HD>(v, lane);
    load_queries<BF, HD, PARTS, NT>(p, b, h, rb, qs);
    __syncthreads();
    float acc[MT][NT][4], ref[NT][2], l[NT][2], fac[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int i = 0; i < 2; i++) {
        fac[n][i] = qs.factor[8 * n + 2 * t + i];
        ref[n][i] = UNSET;
        l[n][i] = 0.0f;
      }
#pragma unroll
    for (int j = 0; j < MT; j++)
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[j][n][i] = 0.0f;
    const uint32_t all_see = len > p.a.n_new - 1 ? len - (p.a.n_new - 1) : 0;  // every row sees these
    // Positions that column c of this lane's tiles sees.
    auto sees = [&](int c) -> uint32_t {
      const uint32_t r = rb * COLS + c, behind = r < p.rows ? p.a.n_new - 1 - r / p.gqa : 0;
      return len > behind ? len - behind : 0;
    };

    for (uint32_t p0 = (u0 * WARPS + warp) * TILE; p0 < end; p0 += UNIT) {
      float s[NT][4];
      scores<BF, HD, PARTS, NT>(s, k, qs, lane);
      walk.next(p);
      walk.load_k<HD>(k, lane);
      const bool all = p0 + TILE <= all_see;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[n][i] *= fac[n][i & 1];
      if (!all || walk.bad) {
        const uint32_t ok = walk.bad ? walk.cached(p, b, p0, lane) : 0xffffu;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const uint32_t r = g + 8 * (i >> 1);
            if (!((ok >> r) & 1) || p0 + r >= sees(8 * n + 2 * t + (i & 1))) s[n][i] = -INFINITY;
          }
      }
      float over = -INFINITY;
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) over = fmaxf(over, fmaxf(s[n][i], s[n][i + 2]) + ref[n][i]);
      if (__any_sync(0xffffffffu, over > LIFT + SLACK)) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
          float f[2];
#pragma unroll
          for (int i = 0; i < 2; i++) {
            float x = fmaxf(s[n][i], s[n][i + 2]);
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
            const float now = fminf(ref[n][i], LIFT - x);
            f[i] = exp2_fast(now - ref[n][i]);
            ref[n][i] = now;
            l[n][i] *= f[i];
          }
#pragma unroll
          for (int j = 0; j < MT; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) acc[j][n][i] *= f[i & 1];
        }
      }
      // Where only some of the new tokens see a position, 0 times an infinite value must not reach the others.
      const bool careful = !all && p.a.n_new > 1 && __any_sync(0xffffffffu, v.template odd<BF>());
      if (!careful) {
        uint32_t a[MT][4];
#pragma unroll
        for (int j = 0; j < MT; j++) v.operand(a[j], j);
#pragma unroll
        for (int n = 0; n < NT; n++) {
          uint32_t pb[WP][2];
          weights_operand<BF, WP>(pb, s[n], ref[n], l[n]);
#pragma unroll
          for (int j = 0; j < MT; j++) {
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < WP; i++) mma<BF>(d, a[j], pb[i][0], pb[i][1]);
            add4(acc[j][n], d);
          }
        }
      } else {
        // Each token's rows are taken from a product with the values behind it cleared.
        const uint32_t tok0 = rb * COLS / p.gqa, tok1 = min(p.a.n_new, (rb * COLS + COLS - 1) / p.gqa + 1);
#pragma unroll
        for (int n = 0; n < NT; n++) {
          uint32_t pb[WP][2];
          weights_operand<BF, WP>(pb, s[n], ref[n], l[n]);
          for (uint32_t tok = tok0; tok < tok1; tok++) {
            const uint32_t behind = p.a.n_new - 1 - tok, stop = len > behind ? len - behind : 0, at = p0 + 2 * t;
            const uint32_t mask0 = (at < stop ? 0xffffu : 0u) | (at + 1 < stop ? 0xffff0000u : 0u);
            const uint32_t mask1 = (at + 8 < stop ? 0xffffu : 0u) | (at + 9 < stop ? 0xffff0000u : 0u);
#pragma unroll
            for (int j = 0; j < MT; j++) {
              uint32_t a[4];
              v.operand(a, j);
              a[0] &= mask0, a[1] &= mask0, a[2] &= mask1, a[3] &= mask1;
              float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
              for (int i = 0; i < WP; i++) mma<BF>(d, a, pb[i][0], pb[i][1]);
#pragma unroll
              for (int i = 0; i < 4; i++)
                if ((rb * COLS + 8 * n + 2 * t + (i & 1)) / p.gqa == tok) acc[j][n][i] += d[i];
            }
          }
        }
      }
      walk.load_v<HD>(v, lane);
    }

    // Join the warps.
#pragma unroll
    for (int n = 0; n < NT; n++) {
#pragma unroll
      for (int i = 0; i < 2; i++) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], o);
        if (g == 0) {
          n_s[warp][8 * n + 2 * t + i] = ref[n][i];
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
    const uint32_t part = 2 * blockIdx.x + (first && u0 ? 0 : 1);
    for (uint32_t i = threadIdx.x; i < COLS * HD; i += THREADS) {
      const uint32_t col = i / HD, d = i % HD, r = rb * COLS + col;
      if (r >= p.rows) break;
      float low = n_s[0][col], o = 0.0f, sum = 0.0f;
#pragma unroll
      for (int w = 1; w < WARPS; w++) low = fminf(low, n_s[w][col]);
#pragma unroll
      for (int w = 0; w < WARPS; w++) {
        const float f = exp2_fast(low - n_s[w][col]);
        sum += f * l_s[w][col];
        o += f * o_s[w][col][d];
      }
      if (fmaf(o, 0.0f, sum) != sum || !(sum < INFINITY)) atomicOr(&odd_s, 1u << col);  // NaN or infinite
      if (complete) {
        const uint32_t tok = r / p.gqa, head = h * p.gqa + r % p.gqa;
        store_from_f32(p.a.out, (int64_t)b * p.a.o_seq + (int64_t)tok * p.a.o_token + (int64_t)head * p.a.o_head + d,
                       p.a.dtype, sum == 0.0f ? 0.0f : o / sum);
        if (d == 0 && p.lse) p.lse[((size_t)b * p.a.kv.n_kv_heads + h) * p.rows + r] = log2f(sum) - low;
      } else {
        p.part_o[((size_t)part * COLS + col) * HD + d] = o;
        if (d == 0) p.part_nl[(size_t)part * COLS + col] = make_float2(low, sum);
      }
    }
    __syncthreads();
    if (odd_s) {
      for (int c = warp; c < COLS; c += WARPS)
        if ((odd_s >> c) & 1)
          row_again<BF, HD>(p, b, h, rb * COLS + c, u0 * UNIT, u1 * UNIT, complete ? -1 : (int64_t)part * COLS + c);
      __syncthreads();
      if (threadIdx.x == 0) odd_s = 0;
    }
    // Work that starts here and goes on: the join kernel's item, with the number of blocks that hold its parts.
    if (u1 < units && !(first && u0) && threadIdx.x == 0) {
      const uint64_t rest = units - u1;
      p.cut[blockIdx.x] = make_int4((int)b, (int)st.hb, (int)(1 + (rest + st.share - 1) / st.share), 0);
    }
    first = false;
    st.left -= v1 - v0;
    st.unit = 0;
    if (++st.hb == hbs) {
      st.hb = 0;
      st.b++;
    }
  }
}

// One block per (attention block whose last work goes on, row): the parts' references and sums joined, the parts dealt
// to JOIN_THREADS / HD groups of threads.
constexpr int JOIN_THREADS = 384;
template <int HD>
__global__ void __launch_bounds__(JOIN_THREADS) k_join(const __grid_constant__ Plan p, int cols) {
  constexpr int GROUPS = JOIN_THREADS / HD;
  __shared__ float o_s[GROUPS][HD], l_s[GROUPS];
  pdl_trigger();
  pdl_wait();
  const int4 cut = p.cut[blockIdx.x];
  const uint32_t b = cut.x, h = cut.y / p.row_blocks, rb = cut.y % p.row_blocks, n = cut.z;
  const uint32_t col = blockIdx.y, r = rb * cols + col, d = threadIdx.x % HD, group = threadIdx.x / HD;
  if (n == 0 || r >= p.rows) return;
  // The first part is the last work of its block, the others the first of theirs.
  auto part = [&](uint32_t i) { return ((size_t)2 * (blockIdx.x + i) + (i == 0 ? 1 : 0)) * cols + col; };
  float low = UNSET;
  for (uint32_t i = threadIdx.x & 31; i < n; i += 32) low = fminf(low, p.part_nl[part(i)].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
  float o = 0.0f, sum = 0.0f;
#pragma unroll 8
  for (uint32_t i = group; i < n; i += GROUPS) {
    const float2 nl = p.part_nl[part(i)];
    const float f = exp2_fast(low - nl.x);
    sum += f * nl.y;
    o += f * p.part_o[part(i) * HD + d];
  }
  o_s[group][d] = o;
  if (d == 0) l_s[group] = sum;
  __syncthreads();
  if (group) return;
#pragma unroll
  for (int i = 1; i < GROUPS; i++) o += o_s[i][d], sum += l_s[i];
  const uint32_t tok = r / p.gqa, head = h * p.gqa + r % p.gqa;
  store_from_f32(p.a.out, (int64_t)b * p.a.o_seq + (int64_t)tok * p.a.o_token + (int64_t)head * p.a.o_head + d, p.a.dtype,
                 sum == 0.0f ? 0.0f : o / sum);
  if (d == 0 && p.lse) p.lse[((size_t)b * p.a.kv.n_kv_heads + h) * p.rows + r] = log2f(sum) - low;
}

// Weights: the scores again (the same products, the same bits), then 2^(s - lse) summed over the query rows in a fixed order and
// added. The attention's schedule, without row blocks. Bound by reading K again, 95 us beside the attention's 168 for 64
// sequences of 4096, 32/8 heads of 128, bf16. (Scores kept by the attention would be 8 bytes per row and position, written and
// read, where K is 2 per value: less below head_dim / 4 rows, more from there on. Not built; it takes a workspace of the
// positions' size.)
template <bool BF, int HD, int PARTS, int NT>
__global__ void __launch_bounds__(THREADS, WEIGHTS_RESIDENT) k_weights(const __grid_constant__ Plan p) {
  constexpr int COLS = 8 * NT;
  __shared__ Queries<HD, PARTS, NT> qs;
  __shared__ uint64_t warp_sums[WARPS];
  __shared__ Start start_s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const uint32_t hbs = p.a.kv.n_kv_heads;
  Start st = find_start(p, hbs, UNIT, SETUP, warp_sums, &start_s);
  bool waited = false;
  while (st.left) {
    const uint32_t b = st.b, h = st.hb, len = seq_len(p, b), units = units_of(len);
    const uint32_t v0 = st.unit, v1 = (uint32_t)min((uint64_t)(SETUP + units), v0 + st.left);
    const uint32_t u0 = v0 > SETUP ? v0 - SETUP : 0, u1 = v1 > SETUP ? v1 - SETUP : 0, end = min(u1 * UNIT, len);
    if (u1 == 0) break;
    float* w = p.a.weights + ((size_t)b * p.a.kv.n_kv_heads + h) * p.a.weights_len;
    const uint32_t all_see = len > p.a.n_new - 1 ? len - (p.a.n_new - 1) : 0;
    for (uint32_t rb = 0; rb < p.row_blocks; rb++) {
      __syncthreads();
      Walk walk;
      walk.begin(p, b, h, u0 * WARPS + warp, end, lane);
      KTile<HD> k;
      walk.next(p);
      walk.load_k<HD>(k, lane);
      load_queries<BF, HD, PARTS, NT>(p, b, h, rb, qs);
      __syncthreads();
      if (!waited) pdl_wait();  // the sums below are the kernels' before
      waited = true;
      float fac[NT][2], lse[NT][2];
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const uint32_t r = rb * COLS + 8 * n + 2 * t + i;
          fac[n][i] = qs.factor[8 * n + 2 * t + i];
          // A row that is none, or saw nothing, adds nothing.
          const float x = r < p.rows ? p.lse[((size_t)b * p.a.kv.n_kv_heads + h) * p.rows + r] : INFINITY;
          lse[n][i] = x == -INFINITY ? INFINITY : x;
        }
      for (uint32_t p0 = (u0 * WARPS + warp) * TILE; p0 < end; p0 += UNIT) {
        float s[NT][4], sum[2] = {0.0f, 0.0f}, before[2];  // before: what stands at its positions
#pragma unroll
        for (int i = 0; i < 2; i++) before[i] = t == 0 && p0 + g + 8 * i < end ? w[p0 + g + 8 * i] : 0.0f;
        scores<BF, HD, PARTS, NT>(s, k, qs, lane);
        walk.next(p);
        walk.load_k<HD>(k, lane);
        const bool whole = p0 + TILE <= all_see && !walk.bad;
        const uint32_t ok = walk.bad ? walk.cached(p, b, p0, lane) : 0xffffu;
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            float x = fmaf(s[n][i], fac[n][i & 1], -lse[n][i & 1]);
            if (!whole) {
              const uint32_t q = rb * COLS + 8 * n + 2 * t + (i & 1), r = g + 8 * (i >> 1);
              const uint32_t behind = q < p.rows ? p.a.n_new - 1 - q / p.gqa : 0;
              if (!((ok >> r) & 1) || p0 + r + behind >= len) x = -INFINITY;
            }
            sum[i >> 1] += exp2_fast(x);
          }
#pragma unroll
        for (int i = 0; i < 2; i++) {
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
          sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
          const uint32_t r = g + 8 * i;
          if (t == 0 && p0 + r < end && ((ok >> r) & 1)) {
            if (!(sum[i] < INFINITY)) sum[i] = weight_again<BF, HD>(p, b, h, rb * COLS, min(p.rows, (rb + 1) * COLS), len, p0 + r);
            w[p0 + r] = before[i] + sum[i];
          }
        }
      }
    }
    st.left -= v1 - v0;
    st.unit = 0;
    if (++st.hb == hbs) {
      st.hb = 0;
      st.b++;
    }
  }
  if (!waited) pdl_wait();
}

template <bool BF, int HD, int PARTS, bool WEIGHTS>
cudaError_t launch_tc(Plan& p, cudaStream_t s);

template <bool BF, int HD, int PARTS, int NT>
cudaError_t launch_rows(Plan& p, cudaStream_t s) {
  void* args[] = {&p};
  const void* attn = (const void*)k_attn<BF, HD, PARTS, NT>;
  constexpr int sums = WARPS * 8 * NT * (HD + 2) * 4;
  if (cudaError_t e = ensure_smem_attr(attn, sums)) return e;
  return launch_kernel(attn, dim3(p.blocks), dim3(THREADS), sums, s, false, args);
}

template <bool BF, int HD, int PARTS, int NT>
cudaError_t launch(Plan& p, cudaStream_t s) {
  void* args[] = {&p};
  cudaError_t err = cudaSuccess;
  if constexpr (NT == 4 && HD % 64 == 0) err = p.tc ? launch_tc<BF, HD, PARTS, false>(p, s) : launch_rows<BF, HD, PARTS, NT>(p, s);
  else err = launch_rows<BF, HD, PARTS, NT>(p, s);
  if (err) return err;
  if (!p.direct) {
    int cols = 8 * NT;
    void* jargs[] = {&p, &cols};
    const uint32_t rows = p.rows < (uint32_t)cols ? p.rows : (uint32_t)cols;
    if (cudaError_t e = launch_kernel((const void*)k_join<HD>, dim3(p.blocks, rows), dim3(JOIN_THREADS / HD * HD), 0, s, true, jargs))
      return e;
  }
  if (p.a.weights) {
    if constexpr (NT == 4 && HD % 64 == 0)
      if (p.tc) return launch_tc<BF, HD, PARTS, true>(p, s);
    return launch_kernel((const void*)k_weights<BF, HD, PARTS, NT>, dim3(p.weight_blocks), dim3(THREADS), 0, s, true, args);
  }
  return cudaSuccess;
}
template <bool BF, int HD, int PARTS>
cudaError_t launch_nt(Plan& p, int nt, cudaStream_t s) {
  return nt == 1 ? launch<BF, HD, PARTS, 1>(p, s) : nt == 2 ? launch<BF, HD, PARTS, 2>(p, s) : launch<BF, HD, PARTS, 4>(p, s);
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
