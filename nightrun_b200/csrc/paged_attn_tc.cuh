// Paged attention of many query rows per KV head (drafts to be checked, wide groups) on the 5th-generation tensor cores.
//
// The same mathematics, schedule and join as paged_attn.cuh, for 9 and more rows: there the warps' own instructions
// bound the kernel (mma.sync fragments, splits and exponentials for 16 positions at a time), here the products, their
// operands' addressing and the sums over positions leave them. Per tile of 128 positions and 32 query rows:
//   S^T [128 x 32] = K Q^T        A = K rows as they lie (K-major), B = Q
//   O^T [HD x 32] += V^T P^T      A = V rows as they lie (M-major: a row is one position's values), B = P (N-major)
// with both accumulators in TMEM. The parts of a split Q or P are further columns (N = 32 per part): a product costs what
// reading its A costs, some 60 cycles here whatever N is, and the columns' sums are taken where they are read. A softmax
// thread owns a position (a TMEM lane): it reads its scores, takes the exponentials, adds them to 32 sums of its own and
// writes its 64-byte row of P; nothing crosses lanes before the end of the work, but where references are set. Two groups
// of four softmax warps take turns at the tiles, each with its own scores, weights, references and accumulators (joined at
// the end), so that one computes while the other's products run.
//
// Measured, calls with the join, this kernel against mma.sync: 16 sequences of 4096, 12, 16, 24 and 32 rows: f16, 64 wide 37, 56,
// 60, 63 against 35, 58, 76, 80 us, 128 wide 49, 77, 82, 86 against 49, 78, 129, 136 us; f32 over f16, 128 wide 50, 78, 84, 88 against 52, 84,
// 158, 166 us; f32 over bf16 54, 84, 90, 94 against 57, 93, 178, 185 us. 24 sequences of 1000..9001, 40/8 heads of 64, 5 new tokens, f32
// over f16: 92 against 138 us, with weights 137 against 193 us. A piece of work costs some 14
// tiles beside its tiles (queries in, the pipeline filled and drained, the tail, the join), which is what bounds it now where
// sequences are short; the schedule counts them.
//
// Roles (10 warps): 0-7 softmax (two groups), 8 brings K and V rows in by TMA (a page piece of tc_rows rows per copy) into a
// ring of half stages in the order of their use (K0 K1 V0 K2 V1 ...), 9 issues the products. mbarriers hand the stages on;
// every wait is bounded. (Rows copied by cp.async reached 16 bytes per clock and SM, 23 are needed.)
//
// Layouts. K, V, Q: 128-byte swizzled rows of 64 values (a 128-wide head takes two blocks). P: 64-byte rows of 32 columns,
// 64-byte swizzle, one block per part. HD = 64: V^T has 64 rows; the other 64 of M = 128 repeat them (leading stride 0).
// A tile holds whole page pieces: tc_tile = 112..128 positions; its other rows stay zero. Rows of V behind the sequence's
// end (whatever the page holds there) and in pages outside the pool are cleared before they are multiplied by 0.
//
// Positions that only some of the new tokens see (the last n_new - 1) are not in the tiles: they are added in f32 at the
// end of a sequence, each row its own, so an infinite value there reaches none that does not see it.
#pragma once
#include "paged_attn.cuh"
#include "tcgen05.cuh"

namespace nrc {
namespace pattn {

// The tensor cores cut the low bits of their sums off, always towards zero: some 4e-8 of the sum per product. So an
// accumulator takes this many tiles (8 products each), then it is added to an f32 sum beside it and begun anew: every tile
// for f32 outputs, 16 for the 16-bit ones, whose own rounding is 2^-12 of the value and more. 5 new tokens, 40/8 heads of 64,
// f32, 16000 and 64000 positions: 6e-7 and 8e-7 off where one accumulator for all tiles was 8e-6 and 3e-5 off; it costs 3% (24
// sequences of 1000..9001: 75 against 73 us; sums in registers instead of TMEM: 78 us, they spill).
constexpr uint32_t tc_drain(bool bf, int parts) { return parts == (bf ? 3 : 2) ? 1 : 16; }
// Tiles whose masks are kept. The copying warp writes tile T's before it waits for T's ring slot: it knows then that the
// products of tile T - 1 - D are done (in the weights' pass, where only K goes through the ring of D), hence that the scores
// two tiles before that have been read, and the masks with them. T - 2 - D may still be waiting to be: D + 3 at least.
constexpr int TC_MASKS = 16;
constexpr float TC_UNSEEN = -3.40282347e38f;  // among the tail's scores: of a position that the row does not see
constexpr int TC_COLS = 32, TC_THREADS = 10 * 32, TC_SOFTMAX = 256;
constexpr int tc_half(int hd) { return TC_TILE * hd * 2; }  // bytes of a half stage: one tile of K or V
constexpr int tc_ring(int hd, int parts) { return hd == 64 ? 6 : parts < 3 ? 5 : 4; }
constexpr int tc_smem(int hd, int parts, bool weights) {
  return tc_ring(hd, parts) * tc_half(hd) + (weights ? 0 : 2 * weight_parts(parts) * TC_TILE * 64) + parts * TC_COLS * hd * 2 + 1024;
}

NRC_DEV void tc_mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accum) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accum)
      : "memory");
}
// D f32, A and B of the cache's type, M = 128; a_m / b_n: the operand's rows run along M / N instead of K.
NRC_DEV uint32_t idesc_f16(bool bf, int n, bool a_m, bool b_n) {
  return (1u << 4) | ((bf ? 1u : 0u) << 7) | ((bf ? 1u : 0u) << 10) | ((a_m ? 1u : 0u) << 15) | ((b_n ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | (8u << 24);
}
// Shared-memory descriptor: address, leading and stride byte offsets, version 1, swizzle (2: 128 bytes, 4: 64 bytes). Only
// the low word holds the address: one thread issues all products, so it adds to that instead of building each anew.
struct Desc {
  uint32_t lo, hi;
  NRC_DEV uint64_t at(uint32_t bytes) const { return (uint64_t)hi << 32 | (lo + (bytes >> 4)); }
};
NRC_DEV Desc swizzled_desc(uint32_t addr, uint32_t lead, uint32_t stride, uint32_t swizzle) {
  return Desc{(addr >> 4) | (lead >> 4) << 16, (stride >> 4) | 1u << 14 | swizzle << 29};
}
// A box of 64 values x tc_rows positions of one (head, page), 128-byte swizzled.
NRC_DEV void tma_rows(uint32_t dst, const CUtensorMap* map, int value, int pos, int head, int page, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
          dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(value), "r"(pos), "r"(head), "r"(page), "r"(smem_u32(bar))
      : "memory");
}
NRC_DEV void st_shared16(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Barrier `id` among n threads; whether any of them brings true.
NRC_DEV bool sync_any(int id, int n, bool x) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %3, 0;\n\tbarrier.red.or.pred q, %1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(id), "r"(n), "r"((uint32_t)x)
      : "memory");
  return r != 0;
}

// Reduces 32 columns over the lanes: every step halves the columns that a lane holds, so 31 exchanges do. Lane i gets
// column i.
template <class Op>
NRC_DEV float over_lanes(const float2 (&x)[TC_COLS / 2], int lane, Op op) {
  float v[TC_COLS];
#pragma unroll
  for (int c = 0; c < TC_COLS / 2; c++) v[2 * c] = x[c].x, v[2 * c + 1] = x[c].y;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
#pragma unroll
    for (int k = 0; k < o; k++) {
      const bool up = lane & o;
      v[k] = op(up ? v[k + o] : v[k], __shfl_xor_sync(0xffffffffu, up ? v[k] : v[k + o], o));
    }
  return v[0];
}

// The pieces of work of a block, the same for every role.
struct Work {
  uint32_t b, h, rb, len, units, u0, u1, seen;  // seen: positions that every new token sees
  uint32_t tiles;                               // tiles of this piece
};
// WEIGHTS: a piece is a KV head's, its row blocks one after the other.
template <bool WEIGHTS>
NRC_DEV bool next_work(const Plan& p, Start& st, uint32_t hbs, uint32_t setup, Work& w) {
  if (WEIGHTS && w.units && w.rb + 1 < p.row_blocks) {
    w.rb++;
    return true;
  }
  if (!st.left) return false;
  w.b = st.b;
  w.h = WEIGHTS ? st.hb : st.hb / p.row_blocks;
  w.rb = WEIGHTS ? 0 : st.hb % p.row_blocks;
  w.len = seq_len(p, st.b);
  w.units = units_of(w.len, p.tc_tile);
  const uint32_t v0 = st.unit, v1 = (uint32_t)min((uint64_t)(setup + w.units), v0 + st.left);
  w.u0 = v0 > setup ? v0 - setup : 0;
  w.u1 = v1 > setup ? v1 - setup : 0;
  w.seen = w.len > p.a.n_new - 1 ? w.len - (p.a.n_new - 1) : 0;
  const uint32_t end = min(w.u1, (w.seen + p.tc_tile - 1) / p.tc_tile);
  w.tiles = end > w.u0 ? end - w.u0 : 0;
  if (w.u1 == 0) {  // the share ends before the first unit
    st.left = 0;
    w.units = 0;
    return false;
  }
  st.left -= v1 - v0;
  st.unit = 0;
  if (++st.hb == hbs) {
    st.hb = 0;
    st.b++;
  }
  return true;
}

// WEIGHTS: the second pass of calls that add up the positions' weights: the scores again, as exponents above the rows' sums,
// added over the columns by the thread that owns the position.
template <bool BF, int HD, int PARTS, bool WEIGHTS>
__global__ void __launch_bounds__(TC_THREADS, 1) k_attn_tc(const __grid_constant__ Plan p) {
  constexpr int D = tc_ring(HD, PARTS), HALF = tc_half(HD), PB = TC_TILE * 64;
  constexpr int WP = weight_parts(PARTS), NP = TC_COLS * PARTS, NW = TC_COLS * WP;  // columns of S and of O: a part after the other
  constexpr uint32_t DRAIN = tc_drain(BF, PARTS), TMEM = WEIGHTS ? NP * 2 > 128 ? 256 : 128 : PARTS == 1 ? 256 : 512;
  static_assert(2 * NP + (WEIGHTS ? 0 : 2 * NW + 2 * TC_COLS) <= TMEM, "two groups' scores, accumulators and sums");
  extern __shared__ uint8_t dyn[];
  __shared__ __align__(8) uint64_t full[D], empty[D], s_full[2], s_empty[2], p_full[2], p_done[2], q_full, cut_full, drain;
  __shared__ uint32_t tmem_s, dead, odd_s;  // odd_s: columns whose sums are no numbers
  static_assert(TC_MASKS >= D + 3, "the copies would overwrite the mask of a tile that is still to be read");
  __shared__ uint32_t cached_s[TC_MASKS][4];          // which positions of a tile are cached, by tile number
  __shared__ __align__(16) float fac_s[TC_COLS], ref_s[2][TC_COLS];  // factor of each row, its reference per group
  __shared__ float f_s[2][TC_COLS], old_s[2][TC_COLS], top_s[2][4][TC_COLS], l_s[2][4][TC_COLS], tail_s[TC_COLS][17], sum_s[TC_COLS];
  __shared__ int64_t tail_off[16];
  __shared__ uint64_t warp_sums[TC_THREADS / 32];
  __shared__ Start start_s;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t hbs = p.a.kv.n_kv_heads * (WEIGHTS ? 1 : p.row_blocks), setup = WEIGHTS ? TC_WEIGHTS_SETUP : TC_SETUP;
  const uint32_t base = (smem_u32(dyn) + 1023) & ~1023u;
  const uint32_t ring = base, p_buf = ring + D * HALF, q_buf = p_buf + (WEIGHTS ? 0 : 2 * WP * PB);
  if (!WEIGHTS) pdl_trigger();
  if (threadIdx.x == 0) {
    for (int i = 0; i < D; i++) mbar_init(&full[i], 1), mbar_init(&empty[i], 1);
    for (int i = 0; i < 2; i++)
      mbar_init(&s_full[i], 1), mbar_init(&s_empty[i], 128), mbar_init(&p_full[i], 128), mbar_init(&p_done[i], 1);
    mbar_init(&q_full, TC_SOFTMAX);
    mbar_init(&cut_full, 1);
    mbar_init(&drain, 1);
    dead = 0;
    odd_s = 0;
    fence_barrier_init();
    if (!WEIGHTS) p.cut[blockIdx.x] = make_int4(0, 0, 0, 0);
  }
  for (uint32_t i = threadIdx.x * 16; i < D * HALF; i += TC_THREADS * 16) st_shared16(ring + i, 0, 0, 0, 0);
  fence_proxy_async_smem();  // the rows that no copy fills are zeros
  if (warp == 9) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_s)), "r"(TMEM) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  Start st = find_start<TC_THREADS>(p, hbs, p.tc_tile, setup, warp_sums, &start_s);  // its barriers publish the above
  tc_fence_after();
  const uint32_t tmem = tmem_s;
  // A wait that runs out ends the kernel's work: whoever sees it tells the others.
  auto wait = [&](uint64_t* bar, uint32_t parity) -> bool {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = globaltimer();
    while (!mbar_try_wait(bar, parity)) {
      if (*(volatile uint32_t*)&dead) return false;
      if (globaltimer() - t0 > 2000000000ull) {
        *(volatile uint32_t*)&dead = 1;
        atomicOr(p.err, ERR_WAIT_FULL);
        return false;
      }
    }
    return true;
  };
  Work w{};

  if (warp == 8) {
    // ---------------------------------------------------------------- copies
    const uint32_t rows = p.tc_rows, pieces = p.tc_tile / rows;
    uint32_t item = 0, tile = 0, cuts = 0;
    bool ok = true;
    // Piece `lane` of the tile: page and first position in it; `there`: lanes whose piece is to be copied. `clear`: the rows
    // that are not (a bit per row, lane q's word holds rows 32 q ..) are zeroed once the others have landed.
    auto copy = [&](const CUtensorMap* map, uint32_t h, int32_t page, uint32_t off, uint32_t there, bool cut, uint32_t valid) {
      const uint32_t slot = item % D, use = item / D, dst = ring + slot * HALF;
      if (use) ok = __all_sync(0xffffffffu, ok && wait(&empty[slot], (use - 1) & 1));
      item++;
      if (!ok) return;
      uint64_t* bar = cut ? &cut_full : &full[slot];
      if (lane == 0) mbar_arrive_expect_tx(bar, __popc(there) * rows * HD * 2);
      __syncwarp();
      if ((there >> lane) & 1)
#pragma unroll
        for (int c = 0; c < HD / 64; c++)
          tma_rows(dst + c * (TC_TILE * 128) + lane * rows * 128, map, 64 * c, (int)off, (int)h, page, bar);
      if (!cut) return;
      ok = __all_sync(0xffffffffu, wait(&cut_full, cuts++ & 1));
#pragma unroll
      for (int q = 0; q < 4; q++)
        if (!((__shfl_sync(0xffffffffu, valid, q) >> lane) & 1))
#pragma unroll
          for (int c = 0; c < HD / 8; c++)
            st_shared16(dst + (c / 8) * (TC_TILE * 128) + (32 * q + lane) * 128 + (c % 8) * 16, 0, 0, 0, 0);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&full[slot]);
    };
    const uint32_t all = (1u << pieces) - 1, batch = 32 / pieces;  // a tile's pieces; tiles whose pieces fill the lanes
    const auto rows_below = [&](uint32_t limit) {                    // lane q: the rows 32 q .. that lie below limit
      const uint32_t r = lane < 4 ? 32 * lane : TC_TILE;
      return limit <= r ? 0u : limit - r >= 32 ? 0xffffffffu : (1u << (limit - r)) - 1;
    };
    const uint32_t whole = rows_below(p.tc_tile);
    while (ok && next_work<WEIGHTS>(p, st, hbs, setup, w)) {
      const uint32_t begin = w.u0 * p.tc_tile, end = min(w.u1 * p.tc_tile, w.seen);
      const int32_t* table = p.a.kv.table + (size_t)w.b * p.a.kv.table_stride;
      // The pages of a batch of tiles, a piece per lane, read one batch ahead.
      uint32_t next_off = 0, cur_off = 0, found = 0, live = 0;
      int32_t next_page = 0, cur_page = 0;
      auto look_up = [&](uint32_t i0) {
        const uint32_t pos = begin + i0 * p.tc_tile + lane * rows, pi = pos / p.a.kv.page_size;
        next_off = pos - pi * p.a.kv.page_size;
        next_page = (uint32_t)lane < batch * pieces && pos < end ? table[pi] : 0;
      };
      look_up(0);
      int32_t v_page = 0;
      uint32_t v_off = 0, v_there = 0, v_valid = 0;
      bool v_cut = false;
      for (uint32_t i = 0, j = 0; i <= w.tiles && ok; i++) {
        int32_t page = 0;
        uint32_t off = 0, there = 0, valid = 0;
        bool cut = false;
        if (i < w.tiles) {
          if (j == 0) {
            cur_off = next_off;
            cur_page = next_page;
            const bool asked = (uint32_t)lane < batch * pieces && begin + i * p.tc_tile + lane * rows < end;
            const bool good = asked && (uint32_t)cur_page < p.a.kv.n_pages;
            if (asked && !good) atomicOr(p.err, ERR_BAD_PAGE);
            live = __ballot_sync(0xffffffffu, asked);
            found = __ballot_sync(0xffffffffu, good);
            look_up(i + batch);
          }
          page = __shfl_sync(0xffffffffu, cur_page, j * pieces + lane);
          off = __shfl_sync(0xffffffffu, cur_off, j * pieces + lane);
          there = (found >> (j * pieces)) & all;
          const uint32_t limit = min(end - begin - i * p.tc_tile, p.tc_tile);
          cut = limit < p.tc_tile || there != all;
          valid = whole;
          if (cut) {
            valid = rows_below(limit);
            if (there != ((live >> (j * pieces)) & all))  // a bad page: row by row
#pragma unroll
              for (int q = 0; q < 4; q++) {
                const uint32_t r = 32 * q + lane, word = __ballot_sync(0xffffffffu, r < limit && ((there >> (r / rows)) & 1));
                if (lane == q) valid = word;
              }
          }
          if (lane < 4) cached_s[tile % TC_MASKS][lane] = valid;
          tile++;
          if (++j == batch) j = 0;
          __syncwarp();
          copy(&p.k_map, w.h, page, off, there, false, 0);  // K's rows behind the end only make scores that are masked
        }
        if (!WEIGHTS && i > 0) copy(&p.v_map, w.h, v_page, v_off, v_there, v_cut, v_valid);
        v_page = page, v_off = off, v_there = there, v_valid = valid, v_cut = cut;
      }
    }
    // After a wait that ran out, what was copied has to land before the block may go.
    if (!ok)
      for (uint32_t it = item > D ? item - D : 0; it < item; it++) mbar_wait(&full[it % D], (it / D) & 1, 100000000ull);
  } else if (warp == 9) {
    // ---------------------------------------------------------------- products
    // The whole warp walks, so that addresses stay in uniform registers; one thread issues.
    uint32_t leader;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(leader));
    uint32_t item = 0, used[2] = {0, 0}, works = 0;
    bool ok = true;
    const uint32_t id_s = idesc_f16(BF, NP, false, false), id_o = idesc_f16(BF, NW, true, true);
    const Desc q_desc = swizzled_desc(q_buf, 16, 1024, 2), p_desc0 = swizzled_desc(p_buf, PB, 512, 4),
               p_desc1 = swizzled_desc(p_buf + WP * PB, PB, 512, 4);
    auto all_wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, wait(bar, parity)); };
    while (ok && next_work<WEIGHTS>(p, st, hbs, setup, w)) {
      if (w.tiles == 0) continue;  // nor do the softmax warps arrive
      ok = all_wait(&q_full, works++ & 1);
      for (uint32_t i = 0; i <= w.tiles && ok; i++) {
        if (i < w.tiles) {
          const uint32_t g = i & 1, k = g ? used[1] : used[0], slot = item % D;
          ok = all_wait(&full[slot], (item / D) & 1) && (k == 0 || all_wait(&s_empty[g], (k - 1) & 1));
          if (!ok) break;
          tc_fence_after();
          const Desc a = swizzled_desc(ring + slot * HALF, 16, 1024, 2);
          const uint32_t d = tmem + g * NP;
          if (leader) {
#pragma unroll
            for (int s = 0; s < HD / 16; s++)
              tc_mma_f16(d, a.at((s / 4) * (TC_TILE * 128) + (s % 4) * 32), q_desc.at((s / 4) * (NP * 128) + (s % 4) * 32), id_s,
                         s ? 1u : 0u);
            tc_commit(&s_full[g]);
            tc_commit(&empty[slot]);
          }
          __syncwarp();
          item++;
        }
        if (WEIGHTS && i < w.tiles) {  // no other products
          if (i & 1)
            used[1]++;
          else
            used[0]++;
        }
        if (!WEIGHTS && i > 0) {
          const uint32_t g = (i - 1) & 1, k = g ? used[1] : used[0], slot = item % D;
          ok = all_wait(&full[slot], (item / D) & 1) && all_wait(&p_full[g], k & 1);
          if (!ok) break;
          tc_fence_after();
          const Desc a = swizzled_desc(ring + slot * HALF, HD == 64 ? 0 : TC_TILE * 128, 1024, 2);
          const Desc b = g ? p_desc1 : p_desc0;
          const uint32_t d = tmem + 2 * NP + g * NW, onto = (i - 1) / 2 % DRAIN;
          if (leader) {
#pragma unroll
            for (int s = 0; s < TC_TILE / 16; s++) tc_mma_f16(d, a.at(s * 2048), b.at(s * 1024), id_o, s ? 1u : onto);
            tc_commit(&p_done[g]);
            tc_commit(&empty[slot]);
          }
          __syncwarp();
          item++;
          if (g)
            used[1]++;
          else
            used[0]++;
        }
      }
    }
    // Nothing of this block's is under way when its TMEM goes.
    if (leader) {
      tc_commit(&drain);
      if (!mbar_wait(&drain, 0)) atomicOr(p.err, ERR_DRAIN);
    }
    __syncwarp();
  } else {
    // ---------------------------------------------------------------- softmax
    const int g = warp >> 2, quarter = warp & 3, row = threadIdx.x & 127;
    const uint32_t lane_base = tmem + ((uint32_t)(quarter * 32) << 16);
    const uint32_t s_tm = lane_base + g * NP, o_tm = lane_base + 2 * NP, sum_tm = lane_base + 2 * NP + 2 * NW + g * TC_COLS;
    uint32_t used = 0, tile = 0;
    bool ok = true, first = true;
    if (WEIGHTS) pdl_wait();  // the sums below are the kernels' before
    while (next_work<WEIGHTS>(p, st, hbs, setup, w)) {
      // Queries: 8 threads per row, as in load_queries().
      {
        constexpr int VALUES = HD / 8;
        const int qr = threadIdx.x / 8, part = threadIdx.x % 8;
        const uint32_t r = w.rb * TC_COLS + qr;
        const bool real = r < p.rows;
        const uint32_t tok = real ? r / p.gqa : 0, head = w.h * p.gqa + (real ? r % p.gqa : 0);
        const int64_t at = (int64_t)w.b * p.a.q_seq + (int64_t)tok * p.a.q_token + (int64_t)head * p.a.q_head + part * VALUES;
        float x[VALUES], big = 0.0f;
#pragma unroll
        for (int i = 0; i < VALUES; i++) {
          x[i] = real ? load_as_f32(p.a.q, at + i, p.a.dtype) : 0.0f;
          big = fmaxf(big, fabsf(x[i]));
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
        const int e = big > 0.0f && big < INFINITY ? ilogbf(big) : 0;
#pragma unroll
        for (int i = 0; i < VALUES; i++) x[i] = ldexpf(x[i], -e);
#pragma unroll
        for (int c0 = 0; c0 < VALUES; c0 += 8) {
          uint32_t v[4][PARTS];
#pragma unroll
          for (int i = 0; i < 4; i++) split2<BF, PARTS>(x[c0 + 2 * i], x[c0 + 2 * i + 1], v[i]);
          const int d = part * VALUES + c0;
#pragma unroll
          for (int j = 0; j < PARTS; j++)
            st_shared16(q_buf + (d / 64) * (NP * 128) + (j * TC_COLS + qr) * 128 + ((((d / 8) % 8) ^ (qr & 7)) << 4), v[0][j],
                        v[1][j], v[2][j], v[3][j]);
        }
        if (part == 0) {
          const float f = ldexpf(p.a.scale * 1.44269504088896340736f, e);
          fac_s[qr] = f;
          float ref = UNSET;
          if (WEIGHTS) {  // a row that is none, or saw nothing, adds nothing
            const float lse = real ? p.lse[((size_t)w.b * p.a.kv.n_kv_heads + w.h) * p.rows + r] : -INFINITY;
            ref = lse == -INFINITY ? -INFINITY : -lse;
          }
          ref_s[0][qr] = ref_s[1][qr] = ref;
        }
        fence_proxy_async_smem();
        if (w.tiles) mbar_arrive(&q_full);
      }
      const bool last = w.u1 == w.units;
      const uint32_t tail = last ? w.len - w.seen : 0;  // positions that are in no tile
      if (threadIdx.x < tail) {
        const int64_t off = paged_row(p.a.kv, w.b, w.seen + threadIdx.x);
        if (off < 0) atomicOr(p.err, ERR_BAD_PAGE);
        tail_off[threadIdx.x] = off < 0 ? -1 : off + (int64_t)w.h * p.a.kv.head_stride;
      }
      named_sync(3, TC_SOFTMAX);  // factors, references, the tail's rows
      float2 l[TC_COLS / 2];
#pragma unroll
      for (int c = 0; c < TC_COLS / 2; c++) l[c] = make_float2(0.0f, 0.0f);
      const uint32_t used0 = used;
      // The accumulator's parts, added to what was drained before; its products are done.
      auto drained = [&](uint32_t to) {
        tc_fence_after();
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t sum[16], o[16];
          tc_ld16(sum_tm + 16 * h, sum);
          tc_wait_ld_regs<16>(sum);
#pragma unroll
          for (int c = 0; c < 16; c++) sum[c] = used - used0 > DRAIN ? sum[c] : 0u;  // the first time nothing stands there
#pragma unroll
          for (int j = 0; j < WP; j++) {
            tc_ld16(o_tm + g * NW + j * TC_COLS + 16 * h, o);
            tc_wait_ld_regs<16>(o);
#pragma unroll
            for (int c = 0; c < 16; c += 2) {
              const float2 x = __fadd2_rn(make_float2(__uint_as_float(sum[c]), __uint_as_float(sum[c + 1])),
                                          make_float2(__uint_as_float(o[c]), __uint_as_float(o[c + 1])));
              sum[c] = __float_as_uint(x.x);
              sum[c + 1] = __float_as_uint(x.y);
            }
          }
          tc_st16(to + 16 * h, sum);
        }
        tc_wait_st();
      };
      auto scaled = [&](uint32_t at) {  // 16 columns by their rows' factors
#pragma unroll
        for (int h = 0; h < 2; h++) {
          uint32_t o[16];
          tc_ld16(at + 16 * h, o);
          tc_wait_ld_regs<16>(o);
#pragma unroll
          for (int c = 0; c < 16; c++) o[c] = __float_as_uint(__uint_as_float(o[c]) * f_s[g][16 * h + c]);
          tc_st16(at + 16 * h, o);
        }
      };
      for (uint32_t i = g; i < w.tiles; i += 2) {
        float before = 0.0f;  // what stands at this thread's position: on its way while the scores are formed
        float* weight = nullptr;
        if constexpr (WEIGHTS) {
          const uint32_t pos = (w.u0 + i) * p.tc_tile + row;
          weight = p.a.weights + ((size_t)w.b * p.a.kv.n_kv_heads + w.h) * p.a.weights_len + pos;
          if ((uint32_t)row < p.tc_tile && pos < w.seen) before = *weight;
        }
        if (ok) ok = wait(&s_full[g], used & 1);
        if (sync_any(1 + g, 128, !ok)) {
          ok = false;
          break;
        }
        __syncwarp();
        tc_fence_after();
        const uint32_t there = cached_s[(tile + i) % TC_MASKS][quarter];
        const bool mine = (there >> lane) & 1;
        float2 x[TC_COLS / 2];  // exponents of neighbouring columns
        float over = -INFINITY;
        auto exponents = [&]() {
#pragma unroll
          for (int h = 0; h < 2; h++) {
            uint32_t v[PARTS][16];
#pragma unroll
            for (int j = 0; j < PARTS; j++) tc_ld16(s_tm + j * TC_COLS + 16 * h, v[j]);
#pragma unroll
            for (int j = 0; j < PARTS; j++) tc_wait_ld_regs<16>(v[j]);
#pragma unroll
            for (int c = 0; c < 16; c += 4) {
              const float4 f = *reinterpret_cast<const float4*>(&fac_s[16 * h + c]);
              const float4 r = *reinterpret_cast<const float4*>(&ref_s[g][16 * h + c]);
#pragma unroll
              for (int k = 0; k < 2; k++) {
                float2 t = make_float2(__uint_as_float(v[0][c + 2 * k]), __uint_as_float(v[0][c + 2 * k + 1]));
#pragma unroll
                for (int j = 1; j < PARTS; j++)
                  t = __fadd2_rn(t, make_float2(__uint_as_float(v[j][c + 2 * k]), __uint_as_float(v[j][c + 2 * k + 1])));
                t = __ffma2_rn(t, k ? make_float2(f.z, f.w) : make_float2(f.x, f.y), k ? make_float2(r.z, r.w) : make_float2(r.x, r.y));
                over = fmaxf(over, fmaxf(t.x, t.y));
                x[8 * h + c / 2 + k] = t;
              }
            }
          }
        };
        exponents();
        if constexpr (WEIGHTS) {
          tc_fence_before();
          mbar_arrive(&s_empty[g]);
          float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
          for (int c = 0; c < TC_COLS / 2; c++) sum = __fadd2_rn(sum, make_float2(exp2_fast(x[c].x), exp2_fast(x[c].y)));
          float add = sum.x + sum.y;
          if (mine && !(add < INFINITY))
            add = weight_again<BF, HD>(p, w.b, w.h, w.rb * TC_COLS, min(p.rows, (w.rb + 1) * TC_COLS), w.len, (w.u0 + i) * p.tc_tile + row);
          if (mine) *weight = before + add;
          used++;
          continue;
        }
        if (sync_any(1 + g, 128, mine && over > LIFT + SLACK)) {
          // New references: each column's largest exponent of the tile, over the lanes, then the warps. Where a row has no
          // reference yet the exponents say nothing: they are taken with reference 0.
          if (quarter == 0) old_s[g][lane] = ref_s[g][lane];
          named_sync(1 + g, 128);
          if (quarter == 0) ref_s[g][lane] = 0.0f;
          named_sync(1 + g, 128);
          __syncwarp();
          exponents();
          if (!mine) {
#pragma unroll
            for (int c = 0; c < TC_COLS / 2; c++) x[c] = make_float2(-INFINITY, -INFINITY);
          }
          top_s[g][quarter][lane] = over_lanes(x, lane, [](float a, float b) { return fmaxf(a, b); });
          named_sync(1 + g, 128);
          if (quarter == 0) {
            const float t = fmaxf(fmaxf(top_s[g][0][lane], top_s[g][1][lane]), fmaxf(top_s[g][2][lane], top_s[g][3][lane]));
            const float old = old_s[g][lane], now = fminf(old, LIFT - t);
            f_s[g][lane] = exp2_fast(now - old);
            ref_s[g][lane] = now;
          }
          named_sync(1 + g, 128);
          __syncwarp();
          exponents();
#pragma unroll
          for (int c = 0; c < TC_COLS / 2; c++) l[c] = make_float2(l[c].x * f_s[g][2 * c], l[c].y * f_s[g][2 * c + 1]);
          if (used != used0) {  // the accumulators too, once the products before are done
            ok = !sync_any(1 + g, 128, !wait(&p_done[g], (used - 1) & 1));
            __syncwarp();
            tc_fence_after();
            if (ok) {
#pragma unroll
              for (int j = 0; j < WP; j++) scaled(o_tm + g * NW + j * TC_COLS);
              if (used - used0 > DRAIN) scaled(sum_tm);
              tc_wait_st();
            }
          }
        }
        tc_fence_before();
        mbar_arrive(&s_empty[g]);
        if (there != 0xffffffffu && !mine) {
#pragma unroll
          for (int c = 0; c < TC_COLS / 2; c++) x[c] = make_float2(-INFINITY, -INFINITY);
        }
        if (used) ok = __all_sync(0xffffffffu, ok && wait(&p_done[g], (used - 1) & 1));  // the weights before are used up
        if (ok && used != used0 && (used - used0) % DRAIN == 0) drained(sum_tm);
        const uint32_t p_row = p_buf + g * WP * PB + row * 64;
#pragma unroll
        for (int c0 = 0; c0 < TC_COLS / 2; c0 += 4) {
          uint32_t v[4][WP];
#pragma unroll
          for (int c = 0; c < 4; c++) {
            const float2 e = make_float2(exp2_fast(x[c0 + c].x), exp2_fast(x[c0 + c].y));
            l[c0 + c] = __fadd2_rn(l[c0 + c], e);
            split2<BF, WP>(e.x, e.y, v[c]);
          }
#pragma unroll
          for (int j = 0; j < WP; j++)
            st_shared16(p_row + j * PB + (((c0 / 4) ^ ((row >> 1) & 3)) << 4), v[0][j], v[1][j], v[2][j], v[3][j]);
        }
        fence_proxy_async_smem();
        tc_fence_before();
        mbar_arrive(&p_full[g]);
        used++;
      }
      tile += w.tiles;
      if (!WEIGHTS && used != used0) {  // the whole sums to the accumulator's first columns, where both groups read them
        ok = __all_sync(0xffffffffu, ok && wait(&p_done[g], (used - 1) & 1));
        if (ok) drained(o_tm + g * NW);
      }
      tc_fence_before();
      // Sums over the positions: lanes, then (below) warps and groups.
      if (!WEIGHTS) l_s[g][quarter][lane] = over_lanes(l, lane, [](float a, float b) { return a + b; });
      // The last positions, seen by some of the new tokens only: one (row, position) pair per thread and step.
      if (tail) {
        for (uint32_t i = threadIdx.x; i < TC_COLS * tail; i += TC_SOFTMAX) {
          const uint32_t c = i / tail, j = i - c * tail, r = w.rb * TC_COLS + c, tok = r / p.gqa;
          float x = TC_UNSEEN;
          if (r < p.rows && w.seen + j + (p.a.n_new - 1 - tok) < w.len && tail_off[j] >= 0) {
            const uint4* kr = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.a.kv.k) + tail_off[j]);
            x = dot_row<BF, HD>(p, query_row(p, w.b, w.h, r), kr) * (p.a.scale * 1.44269504088896340736f);
          }
          tail_s[c][j] = x;
        }
      }
      if (sync_any(3, TC_SOFTMAX, !ok)) {  // sums, tail scores; both groups' products are done
        ok = false;
        break;
      }
      if constexpr (WEIGHTS) {
        if (threadIdx.x < tail) {  // rows in order
          float sum = 0.0f;
          for (int c = 0; c < TC_COLS; c++) {
            const float t = tail_s[c][threadIdx.x];
            if (t != TC_UNSEEN) sum += exp2_fast(t + ref_s[0][c]);
          }
          if (tail_off[threadIdx.x] >= 0)
            p.a.weights[((size_t)w.b * p.a.kv.n_kv_heads + w.h) * p.a.weights_len + w.seen + threadIdx.x] += sum;
        }
        named_sync(3, TC_SOFTMAX);
        continue;
      }
      // Per column: the common reference, the groups' factors, the whole sum; the tail's scores become weights.
      const bool complete = w.u0 == 0 && last, have1 = w.tiles > 1, have0 = w.tiles > 0;
      const uint32_t part = 2 * blockIdx.x + (first && w.u0 ? 0 : 1);
      if (warp == 0) {
        const uint32_t c = lane, r = w.rb * TC_COLS + c;
        const float ref0 = ref_s[0][c], ref1 = ref_s[1][c];
        float low = fminf(ref0, ref1);
        for (uint32_t j = 0; j < tail; j++) low = fminf(low, LIFT - tail_s[c][j]);
        const float f0 = exp2_fast(low - ref0), f1 = exp2_fast(low - ref1);
        float sum = f0 * (l_s[0][0][c] + l_s[0][1][c] + l_s[0][2][c] + l_s[0][3][c]) +
                    f1 * (l_s[1][0][c] + l_s[1][1][c] + l_s[1][2][c] + l_s[1][3][c]);
        for (uint32_t j = 0; j < tail; j++) {
          const float x = tail_s[c][j], e = exp2_fast(x + low);
          tail_s[c][j] = x == TC_UNSEEN ? -1.0f : e;  // not seen: not even 0 times what stands there
          if (x != TC_UNSEEN) sum += e;
        }
        f_s[0][c] = f0;
        f_s[1][c] = f1;
        sum_s[c] = complete ? sum == 0.0f ? 0.0f : 1.0f / sum : 1.0f;
        if (r < p.rows) {
          if (!(sum < INFINITY)) atomicOr(&odd_s, 1u << c);
          if (!complete)
            p.part_nl[(size_t)part * TC_COLS + c] = make_float2(low, sum);
          else if (p.lse)
            p.lse[((size_t)w.b * p.a.kv.n_kv_heads + w.h) * p.rows + r] = log2f(sum) - low;
        }
      }
      named_sync(3, TC_SOFTMAX);
      // Group g writes the columns 16 g .. 16 g + 15; a thread one value (TMEM lane) of each.
      __syncwarp();
      tc_fence_after();
      float o[16];
#pragma unroll
      for (int k = 0; k < 16; k++) o[k] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; h++) {  // the groups' sums
        if (h ? !have1 : !have0) continue;
        uint32_t v[16];
        tc_ld16(o_tm + h * NW + 16 * g, v);
        tc_wait_ld_regs<16>(v);
#pragma unroll
        for (int k = 0; k < 16; k++) o[k] = fmaf(f_s[h][16 * g + k], __uint_as_float(v[k]), o[k]);
      }
      tc_fence_before();
      if (row < HD) {
        for (uint32_t j0 = 0; j0 < tail; j0 += 4) {
          float v[4];
#pragma unroll
          for (int j = 0; j < 4; j++)
            v[j] = j0 + j < tail && tail_off[j0 + j] >= 0
                       ? load_as_f32(p.a.kv.v, tail_off[j0 + j] + row, BF ? NRC_BF16 : NRC_F16)
                       : 0.0f;
#pragma unroll
          for (int j = 0; j < 4; j++) {
            if (j0 + j >= tail) break;
#pragma unroll
            for (int k = 0; k < 16; k++) {
              const float e = tail_s[16 * g + k][j0 + j];
              if (!(e < 0.0f)) o[k] = fmaf(e, v[j], o[k]);
            }
          }
        }
        float zero = 0.0f;  // NaN where a sum is no number
#pragma unroll
        for (int k = 0; k < 16; k++) zero = fmaf(o[k], 0.0f, zero);
        if (zero != 0.0f)
#pragma unroll
          for (int k = 0; k < 16; k++)
            if (w.rb * TC_COLS + 16 * g + k < p.rows && !(fabsf(o[k]) < INFINITY)) atomicOr(&odd_s, 1u << (16 * g + k));
#pragma unroll
        for (int k = 0; k < 16; k++) {
          const uint32_t c = 16 * g + k, r = w.rb * TC_COLS + c;
          if (r < p.rows) {
            if (complete) {
              const uint32_t tok = r / p.gqa, head = w.h * p.gqa + r % p.gqa;
              store_from_f32(p.a.out, (int64_t)w.b * p.a.o_seq + (int64_t)tok * p.a.o_token + (int64_t)head * p.a.o_head + row,
                             p.a.dtype, o[k] * sum_s[c]);
            } else {
              p.part_o[((size_t)part * TC_COLS + c) * HD + row] = o[k];
            }
          }
        }
      }
      if (w.u1 < w.units && !(first && w.u0) && threadIdx.x == 0) {
        const uint64_t rest = w.units - w.u1;
        p.cut[blockIdx.x] = make_int4((int)w.b, (int)(w.h * p.row_blocks + w.rb), (int)(1 + (rest + st.share - 1) / st.share), 0);
      }
      first = false;
      named_sync(3, TC_SOFTMAX);  // everything shared is read before the next piece writes it
      if (odd_s) {
        const uint32_t begin = min(w.u0 * p.tc_tile, w.seen), end = last ? w.len : min(w.u1 * p.tc_tile, w.seen);
        for (int c = warp; c < TC_COLS; c += TC_SOFTMAX / 32)
          if ((odd_s >> c) & 1)
            row_again<BF, HD>(p, w.b, w.h, w.rb * TC_COLS + c, begin, end, complete ? -1 : (int64_t)part * TC_COLS + c);
        named_sync(3, TC_SOFTMAX);
        if (threadIdx.x == 0) odd_s = 0;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  __syncwarp();
  if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM) : "memory");
}

template <bool BF, int HD, int PARTS, bool WEIGHTS>
cudaError_t launch_tc(Plan& p, cudaStream_t s) {
  void* args[] = {&p};
  const void* fn = (const void*)k_attn_tc<BF, HD, PARTS, WEIGHTS>;
  constexpr int smem = tc_smem(HD, PARTS, WEIGHTS);
  if (cudaError_t e = ensure_smem_attr(fn, smem)) return e;
  return launch_kernel(fn, dim3(p.blocks), dim3(TC_THREADS), smem, s, WEIGHTS, args);
}

}  // namespace pattn
}  // namespace nrc
