// C ABI of the operators over a paged KV cache (include/nrcuda.h): argument checks, then one launch
// each. Nothing is allocated and nothing waits.
#include <math.h>

#include <algorithm>
#include <cstdlib>

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

// Rows of `width` bytes at `at` + sum of i_d * stride_d (bytes) for i_d < n_d: a strided tensor, its contiguous dimension apart.
struct Rows {
  struct Dim {
    int64_t stride, n;
  };
  const void* at;
  int64_t width;
  Dim dim[3];
};
Rows flat(const void* at, uint64_t bytes) { return Rows{at, (int64_t)bytes, {{0, 1}, {0, 1}, {0, 1}}}; }

// Whether sum of x_d * stride_d + delta, x_d in [lo_d, hi_d], can lie within (-below, above): dimensions in order of falling
// strides, each tried only as far as the ones behind it can make up for. A few steps where every stride spans all the
// smaller ones, as views of a tensor have it; a layout that takes more than `steps` counts as one that can.
struct Meet {
  struct Dim {
    int64_t stride, lo, hi;
  };
  Dim dim[6];
  int n = 0, steps = 1 << 14;
  bool other = false;  // x = 0 does not count
  int64_t below, above;
  void add(int64_t stride, int64_t lo, int64_t hi) {
    if (stride < 0) stride = -stride, std::swap(lo, hi), lo = -lo, hi = -hi;
    if (lo == 0 && hi == 0) return;
    for (int i = 0; i < n; i++)
      if (dim[i].stride == stride) {
        dim[i].lo += lo, dim[i].hi += hi;
        return;
      }
    dim[n++] = Dim{stride, lo, hi};
  }
  static int64_t floor_div(int64_t a, int64_t b) { return a / b - (a % b < 0); }
  bool from(int d, int64_t delta, bool zero) {
    if (steps-- <= 0) return true;
    if (d == n) return delta > -below && delta < above && !(other && zero);
    int64_t least = 0, most = 0;
    for (int i = d + 1; i < n; i++) least += dim[i].stride * dim[i].lo, most += dim[i].stride * dim[i].hi;
    const Dim& D = dim[d];
    int64_t x0 = D.lo, x1 = D.hi;
    if (D.stride) {  // -below < delta + x stride + [least, most] < above
      x0 = std::max(x0, floor_div(-below - delta - most, D.stride) + 1);
      x1 = std::min(x1, floor_div(above - 1 - delta - least, D.stride));
    }
    for (int64_t x = x0; x <= x1; x++)
      if (from(d + 1, delta + x * D.stride, zero && x == 0)) return true;
    return false;
  }
  bool find(int64_t delta) {
    std::sort(dim, dim + n, [](const Dim& a, const Dim& b) { return a.stride > b.stride; });
    return from(0, delta, true);
  }
};
bool rows_overlap(const Rows& a) {
  Meet m;
  m.below = m.above = a.width;
  m.other = true;
  for (const auto& d : a.dim)
    if (d.n > 1) {
      for (int i = 0; i < m.n; i++)
        if (m.dim[i].stride == std::abs(d.stride)) return true;
      if (d.stride == 0) return true;
      m.add(d.stride, -(d.n - 1), d.n - 1);
    }
  std::sort(m.dim, m.dim + m.n, [](const Meet::Dim& x, const Meet::Dim& y) { return x.stride < y.stride; });
  int64_t extent = a.width;  // most layouts: every stride spans all of the smaller ones
  bool nested = true;
  for (int i = 0; i < m.n; i++) {
    nested = nested && m.dim[i].stride >= extent;
    extent += m.dim[i].stride * m.dim[i].hi;
  }
  return !nested && m.find(0);
}
bool overlap(const Rows& a, const Rows& b) {
  auto span = [](const Rows& r, int64_t& lo, int64_t& hi) {
    lo = 0, hi = r.width;
    for (const auto& d : r.dim) {
      if (d.n <= 0) hi = lo - 1;
      const int64_t last = (d.n - 1) * d.stride;
      (last < 0 ? lo : hi) += last;
    }
  };
  if (!a.at || !b.at) return false;
  int64_t a0, a1, b0, b1;
  span(a, a0, a1), span(b, b0, b1);
  const int64_t delta = (int64_t)(reinterpret_cast<uintptr_t>(b.at) - reinterpret_cast<uintptr_t>(a.at));
  if (a0 >= a1 || b0 >= b1 || delta + b0 >= a1 || delta + b1 <= a0) return false;
  Meet m;  // rows of b that begin within a row of a, or before it by less than their width
  m.below = b.width, m.above = a.width;
  for (const auto& d : b.dim)
    if (d.stride) m.add(d.stride, 0, d.n - 1);
  for (const auto& d : a.dim)
    if (d.stride) m.add(d.stride, -(d.n - 1), 0);
  return m.find(delta);
}
int overlapping(const char* what) { return nrc_fail_api(NRC_ERR_INVALID, "%s overlap", what); }

Rows cache_rows(const nrc_paged_kv& kv, const void* at) {
  return Rows{at, (int64_t)kv.head_dim * 2, {{kv.page_stride * 2, (int64_t)kv.n_pages}, {kv.pos_stride * 2, kv.page_size},
                                             {kv.head_stride * 2, kv.n_kv_heads}}};
}
// For the calls that write them.
int check_k_and_v(const nrc_paged_kv& kv) {
  return kv.n_pages && overlap(cache_rows(kv, kv.k), cache_rows(kv, kv.v)) ? overlapping("K's and V's rows") : NRC_OK;
}

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
  if (rows_overlap(cache_rows(*kv, kv->k))) return overlapping("rows of the pages");
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
  if (int rc = check_k_and_v(*kv)) return rc;
  if ((r->n_heads && (!r->q_out || !r->q)) || !r->k || !r->v || !r->pos || !r->seq || !r->slot || (r->rot_dim && !r->freqs))
    return nrc_fail_api(NRC_ERR_INVALID, "null pointer");
  const int64_t size = r->dtype == NRC_F32 ? 4 : 2;
  auto rows = [&](const void* at, int64_t token, int64_t head, int64_t heads) {
    return Rows{at, (int64_t)kv->head_dim * size, {{token * size, (int64_t)r->tokens}, {head * size, heads}, {0, 1}}};
  };
  const int64_t hq = (int64_t)r->n_heads, hk = kv->n_kv_heads;
  if (hq) {
    const Rows out = rows(r->q_out, r->qo_token, r->qo_head, hq);
    if (rows_overlap(out)) return overlapping("rows of q_out");
    const bool in_place = r->q_out == r->q && (r->qo_token == r->q_token || r->tokens == 1) && (r->qo_head == r->q_head || hq == 1);
    if ((!in_place && overlap(out, rows(r->q, r->q_token, r->q_head, hq))) || overlap(out, rows(r->k, r->k_token, r->k_head, hk)) ||
        overlap(out, rows(r->v, r->v_token, r->v_head, hk)))
      return overlapping("q_out and (otherwise than in place) q, k or v");
  }
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
  const int64_t size = r->dtype == NRC_F32 ? 4 : 2;
  auto rows = [&](const void* at, int64_t seq, int64_t token, int64_t head) {
    return Rows{at, (int64_t)kv->head_dim * size, {{seq * size, kv->n_seqs}, {token * size, (int64_t)r->n_new}, {head * size, (int64_t)r->n_heads}}};
  };
  const Rows out = rows(r->out, r->o_seq, r->o_token, r->o_head);
  if (rows_overlap(out)) return overlapping("rows of out");
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
  const Rows q = rows(r->q, r->q_seq, r->q_token, r->q_head), lens = flat(r->lens, kv->n_seqs * 4ull),
             w = flat(r->weights, (uint64_t)kv->n_seqs * kv->n_kv_heads * r->weights_len * 4), ws = flat(need ? r->workspace : nullptr, need);
  if (overlap(out, q)) return overlapping("out and q");  // q is read again for the weights
  for (const Rows& x : {out, q, lens})
    if (overlap(w, x) || overlap(ws, x) || overlap(ws, w)) return overlapping("weights or workspace and the other tensors");
  if (overlap(out, lens)) return overlapping("out and lens");
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
  if (int rc = check_k_and_v(*kv)) return rc;
  if ((budget && !kept) || !new_lens || !lens || (weights_len && (!weights || !new_weights)))
    return nrc_fail_api(NRC_ERR_INVALID, "null pointer");
  if (!aligned4(kept, new_lens, new_weights) || !aligned4(lens, weights))
    return nrc_fail_api(NRC_ERR_INVALID, "a pointer is not 4-byte aligned");
  const uint64_t heads = (uint64_t)kv->n_seqs * kv->n_kv_heads;
  const Rows K = flat(kept, heads * budget * 4), L = flat(new_lens, kv->n_seqs * 4ull), W = flat(new_weights, heads * weights_len * 4),
             l = flat(lens, kv->n_seqs * 4ull), w = flat(weights, heads * weights_len * 4);
  if (overlap(K, L) || overlap(K, W) || overlap(L, W) || overlap(K, l) || overlap(K, w) || overlap(L, w) || overlap(W, l) ||
      (new_lens != lens && overlap(L, l)) || (new_weights != weights && overlap(W, w)))
    return overlapping("kept, new_lens, new_weights and (otherwise than in place) lens or weights");
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
  const int64_t size = dtype == NRC_F32 ? 4 : 2;
  auto rows = [&](const void* at, int64_t seq, int64_t token, size_t n) {
    return Rows{at, (int64_t)vocab * size, {{seq * size, (int64_t)n_seqs}, {token * size, (int64_t)n}, {0, 1}}};
  };
  const Rows T = flat(tokens, n_seqs * (n_max + 1) * 4), A = flat(accepted, n_seqs * 4), D = flat(draft, n_seqs * n_max * 4),
             U = flat(u, n_seqs * (n_max + 1) * 4), N = flat(n_draft, n_seqs * 4), P = rows(p, p_seq, p_token, n_max + 1),
             Q = rows(q, q_seq, q_token, n_max);
  // A sequence's block reads its drafts and their number before it writes: in place they may be.
  const bool drafts = tokens == draft && n_seqs == 1, number = accepted == n_draft;
  if (overlap(T, A) || (!drafts && overlap(T, D)) || overlap(T, U) || overlap(T, N) || overlap(T, P) || overlap(T, Q) ||
      overlap(A, D) || overlap(A, U) || (!number && overlap(A, N)) || overlap(A, P) || overlap(A, Q))
    return overlapping("tokens, accepted and the inputs");
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
