// C ABI of the operators over a paged KV cache (include/nrcuda.h): argument checks, then one launch
// each. Nothing is allocated and nothing waits.
#include <math.h>

#include "nrcuda.h"
#include "paged.cuh"

using namespace nrc;

int nrc_fail_api(int code, const char* fmt, ...);

namespace {

int cuda_rc(cudaError_t e, const char* what) {
  if (e == cudaSuccess) return NRC_OK;
  return nrc_fail_api(NRC_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned4(const void* a, const void* b = nullptr, const void* c = nullptr, const void* d = nullptr) {
  auto low = [](const void* p) { return reinterpret_cast<uintptr_t>(p) & 3; };
  return !(low(a) | low(b) | low(c) | low(d));
}
// A pointer that holds whole values of the type.
inline bool aligned(const void* p, int dtype) { return (reinterpret_cast<uintptr_t>(p) & (dtype == NRC_F32 ? 3 : 1)) == 0; }
inline bool float_type(int t) { return t == NRC_F32 || t == NRC_F16 || t == NRC_BF16; }

int check_kv(const nrc_paged_kv* kv) {
  if (!kv) return nrc_fail_api(NRC_ERR_INVALID, "null cache");
  if (kv->dtype != NRC_F16 && kv->dtype != NRC_BF16) return nrc_fail_api(NRC_ERR_INVALID, "cache type %d", kv->dtype);
  if (kv->head_dim < 32 || kv->head_dim > 128 || kv->head_dim % 32)
    return nrc_fail_api(NRC_ERR_INVALID, "head_dim %u (32, 64, 96 or 128)", kv->head_dim);
  if (kv->page_size == 0 || kv->n_kv_heads == 0 || kv->n_kv_heads > 16384)
    return nrc_fail_api(NRC_ERR_INVALID, "page size %u, %u KV heads", kv->page_size, kv->n_kv_heads);
  if (kv->n_seqs > 65535) return nrc_fail_api(NRC_ERR_INVALID, "%u sequences (65535 at most)", kv->n_seqs);
  if (kv->n_pages > 0x7fffffffull || (uint64_t)kv->max_pages * kv->page_size > 0x7fffffffull)
    return nrc_fail_api(NRC_ERR_INVALID, "more than 2^31-1 pages, or positions in a sequence's table");
  if (kv->table_stride < kv->max_pages) return nrc_fail_api(NRC_ERR_INVALID, "table rows overlap");
  if (kv->n_pages && (!kv->k || !kv->v)) return nrc_fail_api(NRC_ERR_INVALID, "null pages");
  if (kv->n_seqs && kv->max_pages && !kv->table) return nrc_fail_api(NRC_ERR_INVALID, "null table");
  if ((kv->n_pages > 1 && !kv->page_stride) || (kv->page_size > 1 && !kv->pos_stride) || (kv->n_kv_heads > 1 && !kv->head_stride))
    return nrc_fail_api(NRC_ERR_INVALID, "rows of the pages overlap");
  if (!aligned4(kv->table)) return nrc_fail_api(NRC_ERR_INVALID, "table is not 4-byte aligned");
  if (!aligned16(kv->k) || !aligned16(kv->v) || kv->page_stride % 8 || kv->pos_stride % 8 || kv->head_stride % 8)
    return nrc_fail_api(NRC_ERR_INVALID, "pages and their strides must be multiples of 16 bytes");
  return NRC_OK;
}

}  // namespace

extern "C" {

int nrc_rope_freqs_yarn(float* out, float* mscale, size_t rot_dim, float theta, float factor, float beta_fast,
                        float beta_slow, float orig) {
  if (!out || !mscale || rot_dim == 0 || rot_dim % 2 || !(theta > 1.0f) || !(factor > 0.0f) || !(beta_slow > 0.0f) ||
      !(beta_fast > beta_slow) || !(orig > 0.0f))
    return nrc_fail_api(NRC_ERR_INVALID, "bad rope_freqs_yarn arguments");
  const double TWO_PI = 6.283185307179586476925;
  // The (fractional) pair index whose angle makes `turns` turns within the original context.
  auto at = [&](double turns) { return (double)rot_dim * log(orig / (turns * TWO_PI)) / (2.0 * log((double)theta)); };
  const double low = fmax(0.0, floor(at(beta_fast))), high = fmin((double)rot_dim - 1.0, ceil(at(beta_slow)));
  const double width = fmax(high - low, 1e-3);
  for (size_t i = 0; i < rot_dim / 2; i++) {
    const double freq = pow((double)theta, -2.0 * (double)i / (double)rot_dim);
    const double stretch = fmin(1.0, fmax(0.0, ((double)i - low) / width));
    out[i] = (float)(freq * (1.0 - stretch) + freq / factor * stretch);
  }
  *mscale = factor <= 1.0f ? 1.0f : (float)(0.1 * log((double)factor) + 1.0);
  return NRC_OK;
}

int nrc_rope_append(const nrc_paged_kv* kv, const nrc_rope_args* r, void* stream) {
  if (int rc = check_kv(kv)) return rc;
  if (!r) return nrc_fail_api(NRC_ERR_INVALID, "null arguments");
  if (!float_type(r->dtype)) return nrc_fail_api(NRC_ERR_INVALID, "type %d", r->dtype);
  if (r->style != 0 && r->style != 1) return nrc_fail_api(NRC_ERR_INVALID, "style %d", r->style);
  if (r->rot_dim % 2 || r->rot_dim > kv->head_dim)
    return nrc_fail_api(NRC_ERR_INVALID, "rot_dim %llu", (unsigned long long)r->rot_dim);
  if (r->tokens > 0x7fffffff || r->n_heads > 16384) return nrc_fail_api(NRC_ERR_INVALID, "shape too large");
  if (r->tokens == 0) return NRC_OK;
  if ((r->n_heads && (!r->q_out || !r->q)) || !r->k || !r->v || !r->pos || !r->seq || !r->slot || (r->rot_dim && !r->freqs))
    return nrc_fail_api(NRC_ERR_INVALID, "null pointer");
  if ((r->tokens > 1 && r->n_heads && !r->qo_token) || (r->n_heads > 1 && !r->qo_head))
    return nrc_fail_api(NRC_ERR_INVALID, "rows of q_out overlap");
  if (!aligned(r->q, r->dtype) || !aligned(r->k, r->dtype) || !aligned(r->v, r->dtype) || !aligned(r->q_out, r->dtype) ||
      !aligned4(r->freqs, r->pos, r->seq, r->slot))
    return nrc_fail_api(NRC_ERR_INVALID, "a pointer is not aligned to its type");
  return cuda_rc(rope_append_paged_run(*kv, *r, static_cast<cudaStream_t>(stream)), "rope_append");
}

static int check_attn(const nrc_paged_kv* kv, size_t n_new, size_t n_heads, size_t* max_len) {
  if (int rc = check_kv(kv)) return rc;
  if (n_new == 0 || n_new > NRC_MAX_BATCH) return nrc_fail_api(NRC_ERR_INVALID, "%zu new tokens (1..64)", n_new);
  if (n_heads == 0 || n_heads % kv->n_kv_heads || n_heads > 16384)
    return nrc_fail_api(NRC_ERR_INVALID, "%zu query heads over %u KV heads", n_heads, kv->n_kv_heads);
  const size_t slots = (size_t)kv->max_pages * kv->page_size;
  if (*max_len == 0 || *max_len > slots) *max_len = slots;
  return NRC_OK;
}

int nrc_attn_paged_workspace(const nrc_paged_kv* kv, size_t n_new, size_t n_heads, int with_weights, size_t max_len,
                             size_t* out_bytes) {
  if (!out_bytes) return nrc_fail_api(NRC_ERR_INVALID, "null pointer");
  if (int rc = check_attn(kv, n_new, n_heads, &max_len)) return rc;
  *out_bytes = paged_attn_workspace(*kv, (uint32_t)n_new, (uint32_t)n_heads, with_weights != 0, (uint32_t)max_len);
  return NRC_OK;
}

int nrc_attn_paged(const nrc_paged_kv* kv, const nrc_attn_args* r, void* stream) {
  if (!r) return nrc_fail_api(NRC_ERR_INVALID, "null arguments");
  size_t max_len = r->max_len;
  if (int rc = check_attn(kv, r->n_new, r->n_heads, &max_len)) return rc;
  if (!float_type(r->dtype)) return nrc_fail_api(NRC_ERR_INVALID, "type %d", r->dtype);
  if (!isfinite(r->scale)) return nrc_fail_api(NRC_ERR_INVALID, "scale is not finite");
  if (r->weights && (r->weights_len == 0 || r->weights_len > 0x7fffffff))
    return nrc_fail_api(NRC_ERR_INVALID, "weights of length %llu", (unsigned long long)r->weights_len);
  if (kv->n_seqs == 0) return NRC_OK;
  if (!r->out || !r->q || !r->lens) return nrc_fail_api(NRC_ERR_INVALID, "null pointer");
  if ((kv->n_seqs > 1 && !r->o_seq) || (r->n_new > 1 && !r->o_token) || (r->n_heads > 1 && !r->o_head))
    return nrc_fail_api(NRC_ERR_INVALID, "rows of out overlap");
  if (!aligned(r->out, r->dtype) || !aligned(r->q, r->dtype) || !aligned4(r->lens, r->weights))
    return nrc_fail_api(NRC_ERR_INVALID, "a pointer is not aligned to its type");
  PagedAttnArgs a{};
  a.kv = *kv;
  a.out = r->out;
  a.q = r->q;
  a.o_seq = r->o_seq, a.o_token = r->o_token, a.o_head = r->o_head;
  a.q_seq = r->q_seq, a.q_token = r->q_token, a.q_head = r->q_head;
  a.dtype = r->dtype;
  a.n_new = (uint32_t)r->n_new, a.n_heads = (uint32_t)r->n_heads, a.max_len = (uint32_t)max_len;
  a.lens = r->lens;
  a.scale = r->scale;
  a.weights = r->weights;
  a.weights_len = (uint32_t)r->weights_len;
  a.workspace = r->workspace;
  const size_t need = paged_attn_workspace(*kv, a.n_new, a.n_heads, a.weights != nullptr, a.max_len);
  if (need && (!r->workspace || r->workspace_bytes < need || !aligned16(r->workspace)))
    return nrc_fail_api(NRC_ERR_INVALID, "workspace of %llu bytes, 16-byte aligned: %zu needed",
                        r->workspace ? (unsigned long long)r->workspace_bytes : 0ull, need);
  if (r->out == r->q) return nrc_fail_api(NRC_ERR_INVALID, "out and q overlap");  // q is read again for the weights
  return cuda_rc(paged_attn_run(a, static_cast<cudaStream_t>(stream)), "attn_paged");
}

int nrc_kv_evict(const nrc_paged_kv* kv, int32_t* kept, int32_t* new_lens, float* new_weights, const int32_t* lens,
                 const float* weights, size_t weights_len, size_t budget, size_t recent, size_t sinks, void* stream) {
  if (int rc = check_kv(kv)) return rc;
  if (weights_len > 0x7fffffff || budget > weights_len || budget > (size_t)kv->max_pages * kv->page_size)
    return nrc_fail_api(NRC_ERR_INVALID, "budget %zu over weights of length %zu and %u pages of %u", budget, weights_len,
                        kv->max_pages, kv->page_size);
  if (recent > budget || sinks > budget - recent)
    return nrc_fail_api(NRC_ERR_INVALID, "%zu first and %zu latest positions in a budget of %zu", sinks, recent, budget);
  if (kv->n_seqs == 0) return NRC_OK;
  if ((budget && !kept) || !new_lens || !lens || (weights_len && (!weights || !new_weights)))
    return nrc_fail_api(NRC_ERR_INVALID, "null pointer");
  if (!aligned4(kept, new_lens, new_weights) || !aligned4(lens, weights))
    return nrc_fail_api(NRC_ERR_INVALID, "a pointer is not 4-byte aligned");
  EvictArgs a{};
  a.kv = *kv;
  a.kept = kept, a.new_lens = new_lens, a.new_weights = new_weights;
  a.lens = lens, a.weights = weights;
  a.weights_len = (uint32_t)weights_len, a.budget = (uint32_t)budget, a.recent = (uint32_t)recent, a.sinks = (uint32_t)sinks;
  return cuda_rc(kv_evict_run(a, static_cast<cudaStream_t>(stream)), "kv_evict");
}

int nrc_verify_draft(int32_t* tokens, int32_t* accepted, const void* p, int64_t p_seq, int64_t p_token, const void* q,
                     int64_t q_seq, int64_t q_token, int dtype, size_t n_seqs, size_t n_max, size_t vocab,
                     const int32_t* draft, const float* u, const int32_t* n_draft, void* stream) {
  if (!float_type(dtype)) return nrc_fail_api(NRC_ERR_INVALID, "type %d", dtype);
  if (n_max > NRC_MAX_BATCH - 1) return nrc_fail_api(NRC_ERR_INVALID, "%zu drafted tokens (63 at most)", n_max);
  if (vocab == 0 || vocab > 0x7fffffff || n_seqs > 0xfffffff) return nrc_fail_api(NRC_ERR_INVALID, "bad shape");
  if (n_seqs == 0) return NRC_OK;
  if (!tokens || !accepted || !p || !u || (n_max && !draft)) return nrc_fail_api(NRC_ERR_INVALID, "null pointer");
  if (!aligned(p, dtype) || !aligned(q, dtype) || !aligned4(tokens, accepted, draft, u) || !aligned4(n_draft))
    return nrc_fail_api(NRC_ERR_INVALID, "a pointer is not aligned to its type");
  VerifyArgs a{};
  a.tokens = tokens, a.accepted = accepted;
  a.p = p, a.q = q;
  a.p_seq = p_seq, a.p_token = p_token, a.q_seq = q_seq, a.q_token = q_token;
  a.dtype = dtype;
  a.n_seqs = (uint32_t)n_seqs, a.n_max = (uint32_t)n_max, a.vocab = (uint32_t)vocab;
  a.draft = draft, a.u = u, a.n_draft = n_draft;
  return cuda_rc(verify_draft_run(a, static_cast<cudaStream_t>(stream)), "verify_draft");
}

}  // extern "C"
