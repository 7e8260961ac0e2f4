// Host side of the paged attention: the variant, the schedule and the workspace's layout.
#include <atomic>

#include "paged_attn.cuh"

namespace nrc {
namespace {

__device__ unsigned g_attn_err;

using pattn::Plan;

// SM count and error word of the current device, looked up once per device (no lock: each slot is written with the same
// values by whoever comes first).
struct Device {
  std::atomic<int> sms{0};
  std::atomic<unsigned*> err{nullptr};
};
constexpr int MAX_DEVICES = 64;
Device g_devices[MAX_DEVICES];

int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev >= MAX_DEVICES) return 148;  // only a size asked for without a device
  if ((n = g_devices[dev].sms.load(std::memory_order_relaxed))) return n;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  g_devices[dev].sms.store(n, std::memory_order_relaxed);
  return n;
}
cudaError_t error_word(unsigned** err) {
  int dev = 0;
  if (cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev < MAX_DEVICES && (*err = g_devices[dev].err.load(std::memory_order_relaxed))) return cudaSuccess;
  void* p = nullptr;
  if (cudaError_t e = cudaGetSymbolAddress(&p, g_attn_err)) return e;
  *err = static_cast<unsigned*>(p);
  if (dev < MAX_DEVICES) g_devices[dev].err.store(*err, std::memory_order_relaxed);
  return cudaSuccess;
}

// Parts of the cache's type that hold the bits of q's (and out's) type.
int parts_of(int cache, int dtype) {
  if (cache == NRC_F16) return dtype == NRC_F32 ? 2 : 1;
  return dtype == NRC_F32 ? 3 : dtype == NRC_F16 ? 2 : 1;
}

// Positions per copy: the largest piece of a page that fills a tile of 128 to 7 parts in 8, in whole groups of 8 rows (the
// swizzle's). 16 copies per tile at most.
bool tc_shape(uint32_t page, uint32_t* rows) {
  for (uint32_t r = pattn::TC_TILE; r >= 8; r -= 8)
    if (page % r == 0 && pattn::TC_TILE / r * r >= 112) {
      *rows = r;
      return true;
    }
  return false;
}

// The tensor maps of the tcgen05 kernel; false where the pages' strides cannot be told to the TMA unit.
bool make_maps(Plan& p) {
  const nrc_paged_kv& kv = p.a.kv;
  auto encode = tensor_map_encoder();
  if (!encode || kv.pos_stride <= 0 || kv.head_stride <= 0 || kv.page_stride <= 0) return false;
  const cuuint64_t dims[4] = {kv.head_dim, kv.page_size, kv.n_kv_heads, kv.n_pages};
  const cuuint64_t strides[3] = {(cuuint64_t)kv.pos_stride * 2, (cuuint64_t)kv.head_stride * 2, (cuuint64_t)kv.page_stride * 2};
  const cuuint32_t box[4] = {64, p.tc_rows, 1, 1}, step[4] = {1, 1, 1, 1};
  const auto type = kv.dtype == NRC_F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
  for (int i = 0; i < 2; i++)
    if (encode(i ? &p.v_map : &p.k_map, type, 4, i ? kv.v : kv.k, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
               CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
      return false;
  return true;
}

// Fills the plan and returns the workspace's bytes; `base` null: sizes only.
size_t make_plan(Plan& p, int* nt, uint8_t* base) {
  const nrc_paged_kv& kv = p.a.kv;
  p.gqa = p.a.n_heads / kv.n_kv_heads;
  p.rows = p.gqa * p.a.n_new;
  const uint32_t units = (p.a.max_len + pattn::UNIT - 1) / pattn::UNIT;
  // A share is 4 units at least, and a sequence of up to 4 is not split. In calls of us at 2, 4 and 8, f32 over f16, 32/8 heads of
  // 64: one sequence of 300 10.1, 13.3, 8.6 (unsplit), of 600 10.2, 12.6, 16.4, 16 of 500 14.6, 15.8, 14.9; bf16, 128 wide: one of 1024
  // 11.9, 15.0, 16.9, four of 1000 15.4, 17.3, 21.4. (Smaller shares gain on one short sequence: more partial results, for which
  // the workspace grows, and shorter ones.) Many or long sequences give every block more than that.
  p.min_units = 4;
  // 9 rows and more on the tcgen05 kernel, where its tiles fit: 64 or 128 wide heads, a tail of 15 positions at most, pages
  // that whole 8-row groups fill.
  p.tc = p.rows > 8 && p.a.n_new <= 16 && kv.head_dim % 64 == 0 && units > p.min_units && tc_shape(kv.page_size, &p.tc_rows);
  if (p.tc) p.tc_tile = pattn::TC_TILE / p.tc_rows * p.tc_rows;
  *nt = p.tc ? 4 : p.rows <= 8 ? 1 : p.rows <= 16 ? 2 : 4;
  const uint32_t cols = 8 * *nt;
  p.row_blocks = (p.rows + cols - 1) / cols;
  const uint64_t items = (uint64_t)kv.n_seqs * kv.n_kv_heads * p.row_blocks;
  p.step_pages = pattn::UNIT / kv.page_size;
  p.step_off = pattn::UNIT % kv.page_size;
  p.direct = units <= p.min_units && items <= 0x7fffffffu;
  const uint64_t w_units = (uint64_t)kv.n_seqs * kv.n_kv_heads * (units ? units : 1);
  const uint64_t w_resident = (uint64_t)sm_count() * pattn::WEIGHTS_RESIDENT;
  p.weight_blocks = (uint32_t)(w_units < w_resident ? w_units : w_resident);
  if (p.direct) {
    p.blocks = (uint32_t)items;
  } else {
    const uint64_t all = items * units, resident = (uint64_t)sm_count() * (p.tc ? 1 : pattn::resident(kv.head_dim, *nt));
    const uint64_t want = (all + p.min_units - 1) / p.min_units;
    p.blocks = (uint32_t)(want < resident ? want : resident);
  }
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) & ~(size_t)255;
    return base ? base + here : nullptr;
  };
  if (!p.direct) {
    p.cut = reinterpret_cast<int4*>(take(sizeof(int4) * p.blocks));
    p.part_nl = reinterpret_cast<float2*>(take(sizeof(float2) * 2 * p.blocks * cols));
    p.part_o = reinterpret_cast<float*>(take(sizeof(float) * 2 * p.blocks * cols * kv.head_dim));
  }
  p.lse = nullptr;
  if (p.a.weights) p.lse = reinterpret_cast<float*>(take(sizeof(float) * kv.n_seqs * kv.n_kv_heads * p.rows));
  return at;
}

}  // namespace

size_t paged_attn_workspace(const nrc_paged_kv& kv, uint32_t n_new, uint32_t n_heads, bool weights, uint32_t max_len) {
  Plan p{};
  p.a.kv = kv;
  p.a.n_new = n_new;
  p.a.n_heads = n_heads;
  p.a.max_len = max_len;
  p.a.weights = weights ? reinterpret_cast<float*>(1) : nullptr;
  int nt;
  return make_plan(p, &nt, nullptr);
}

cudaError_t paged_attn_run(const PagedAttnArgs& a, cudaStream_t s) {
  Plan p{};
  p.a = a;
  int nt;
  make_plan(p, &nt, static_cast<uint8_t*>(a.workspace));
  // Without tensor maps the other kernel runs on the same plan (32 rows at a time, the blocks of this one).
  if (p.tc && !make_maps(p)) p.tc = 0;
  if (cudaError_t e = error_word(&p.err)) return e;
  const int parts = parts_of(a.kv.dtype, a.dtype);
  if (a.kv.dtype == NRC_F16) return parts == 2 ? paged_attn_f16_2(p, nt, s) : paged_attn_f16_1(p, nt, s);
  return parts == 3 ? paged_attn_bf16_3(p, nt, s) : parts == 2 ? paged_attn_bf16_2(p, nt, s) : paged_attn_bf16_1(p, nt, s);
}

cudaError_t paged_attn_take_errors(unsigned* bits) {
  cudaError_t e = cudaMemcpyFromSymbol(bits, g_attn_err, sizeof(unsigned));
  const unsigned zero = 0;
  if (e == cudaSuccess && *bits) e = cudaMemcpyToSymbol(g_attn_err, &zero, sizeof zero);
  return e;
}

}  // namespace nrc
