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

// Fills the plan and returns the workspace's bytes; `base` null: sizes only.
size_t make_plan(Plan& p, int* nt, uint8_t* base) {
  const nrc_paged_kv& kv = p.a.kv;
  p.gqa = p.a.n_heads / kv.n_kv_heads;
  p.rows = p.gqa * p.a.n_new;
  *nt = p.rows <= 8 ? 1 : p.rows <= 16 ? 2 : 4;
  const uint32_t cols = 8 * *nt;
  p.row_blocks = (p.rows + cols - 1) / cols;
  const uint64_t items = (uint64_t)kv.n_seqs * kv.n_kv_heads * p.row_blocks;
  const uint32_t units = (p.a.max_len + pattn::UNIT - 1) / pattn::UNIT;
  p.step_pages = pattn::UNIT / kv.page_size;
  p.step_off = pattn::UNIT % kv.page_size;
  p.min_units = 4;
  p.direct = units <= p.min_units && items <= 0x7fffffffu;
  const uint64_t w_units = (uint64_t)kv.n_seqs * kv.n_kv_heads * (units ? units : 1);
  const uint64_t w_resident = (uint64_t)sm_count() * pattn::WEIGHTS_RESIDENT;
  p.weight_blocks = (uint32_t)(w_units < w_resident ? w_units : w_resident);
  if (p.direct) {
    p.blocks = (uint32_t)items;
  } else {
    const uint64_t all = items * units, resident = (uint64_t)sm_count() * pattn::resident(kv.head_dim, *nt);
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
