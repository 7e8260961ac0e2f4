// Paged KV cache: the device view and the launchers of the kernels over it
// (paged.cu: rotary append and eviction; paged_attn.cu: attention) and of the
// draft verification (verify.cu).
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "common.cuh"
#include "nrcuda.h"

namespace nrc {

enum : unsigned { ERR_BAD_PAGE = 8u, ERR_BAD_SLOT = 16u };

// cudaLaunchKernelExC with the programmatic-dependency attribute of the other kernels' launchers.
inline cudaError_t launch_kernel(const void* fn, dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool pdl,
                                 void** args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelExC(&cfg, fn, args);
}

// A value of one of the element types as f32 (exact), and back (one rounding, nearest even).
NRC_DEV float load_as_f32(const void* p, int64_t i, int dtype) {
  if (dtype == NRC_F32) return static_cast<const float*>(p)[i];
  if (dtype == NRC_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
NRC_DEV void store_from_f32(void* p, int64_t i, int dtype, float v) {
  if (dtype == NRC_F32)
    static_cast<float*>(p)[i] = v;
  else if (dtype == NRC_F16)
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Element offset of (sequence, slot, head 0), or -1 where the table leads outside the pool.
NRC_DEV int64_t paged_row(const nrc_paged_kv& kv, uint32_t seq, uint32_t slot) {
  const uint32_t pi = slot / kv.page_size, off = slot - pi * kv.page_size;
  const int32_t page = kv.table[(size_t)seq * kv.table_stride + pi];
  if (page < 0 || (uint64_t)page >= kv.n_pages) return -1;
  return (int64_t)page * kv.page_stride + (int64_t)off * kv.pos_stride;
}

cudaError_t rope_append_paged_run(const nrc_paged_kv& kv, const nrc_rope_args& r, cudaStream_t s);

struct EvictArgs {
  nrc_paged_kv kv;
  int32_t *kept, *new_lens;
  float* new_weights;
  const int32_t* lens;
  const float* weights;
  uint32_t weights_len, budget, recent, sinks;
};
cudaError_t kv_evict_run(const EvictArgs& a, cudaStream_t s);

struct PagedAttnArgs {
  nrc_paged_kv kv;
  void* out;
  const void* q;
  int64_t o_seq, o_token, o_head, q_seq, q_token, q_head;
  int dtype;
  uint32_t n_new, n_heads, max_len;
  const int32_t* lens;
  float scale;
  float* weights;
  uint32_t weights_len;
  void* workspace;
};
size_t paged_attn_workspace(const nrc_paged_kv& kv, uint32_t n_new, uint32_t n_heads, bool weights, uint32_t max_len);
cudaError_t paged_attn_run(const PagedAttnArgs& a, cudaStream_t s);

struct VerifyArgs {
  int32_t *tokens, *accepted;
  const void *p, *q;
  int64_t p_seq, p_token, q_seq, q_token;
  int dtype;
  uint32_t n_seqs, n_max, vocab;
  const int32_t* draft;
  const float* u;
  const int32_t* n_draft;
};
cudaError_t verify_draft_run(const VerifyArgs& a, cudaStream_t s);

// Error bits that the kernels of paged.cu / paged_attn.cu recorded on the current device, cleared
// by the read. The words are device variables: nothing is allocated, so the first call of an
// operator may already be part of a stream capture.
cudaError_t paged_take_errors(unsigned* bits);
cudaError_t paged_attn_take_errors(unsigned* bits);

}  // namespace nrc
