// Verification of drafted tokens against the target's probabilities.
#include "paged.cuh"

namespace nrc {
namespace {

constexpr int VD_THREADS = 1024;

// What is left of p at one token: max(p - q, 0) after a refusal, p itself otherwise; NaN and
// negative values count as nothing. The difference of two f32 values is formed in 64 bits.
NRC_DEV double left_of(float p, float q) {
  const double d = (double)p - (double)q;
  return d > 0.0 ? d : 0.0;
}

// One CTA per sequence. Thread i of the row sum owns the tokens [i * per, (i + 1) * per): its partial
// sum is taken in index order in 64 bits, the partial sums are scanned in index order, and the
// thread whose range holds the goal walks its tokens again.
__global__ void __launch_bounds__(VD_THREADS) k_verify_draft(const VerifyArgs a) {
  __shared__ double part[VD_THREADS];
  __shared__ uint32_t taken_s;
  __shared__ int last_s;
  const uint32_t b = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) {
    int nd = a.n_draft ? a.n_draft[b] : (int)a.n_max;
    nd = nd < 0 ? 0 : nd > (int)a.n_max ? (int)a.n_max : nd;
    int i = 0;
    for (; i < nd; i++) {
      const int32_t x = a.draft[(size_t)b * a.n_max + i];
      if (x < 0 || (uint32_t)x >= a.vocab) break;
      const float px = load_as_f32(a.p, (int64_t)b * a.p_seq + (int64_t)i * a.p_token + x, a.dtype);
      const float qx = a.q ? load_as_f32(a.q, (int64_t)b * a.q_seq + (int64_t)i * a.q_token + x, a.dtype) : 1.0f;
      if (!((double)a.u[(size_t)b * (a.n_max + 1) + i] * (double)qx < (double)px)) break;
    }
    taken_s = (uint32_t)i | (i < nd ? 0x80000000u : 0u);
    last_s = -1;
  }
  __syncthreads();
  const uint32_t taken = taken_s & 0x7fffffffu;
  bool refused = taken_s >> 31;
  const int64_t pr = (int64_t)b * a.p_seq + (int64_t)taken * a.p_token;
  const int64_t qr = (int64_t)b * a.q_seq + (int64_t)taken * a.q_token;
  const int32_t certain = refused && !a.q ? a.draft[(size_t)b * a.n_max + taken] : -1;
  const uint32_t per = (a.vocab + VD_THREADS - 1) / VD_THREADS;
  const uint32_t t0 = tid * per < a.vocab ? tid * per : a.vocab, t1 = t0 + per < a.vocab ? t0 + per : a.vocab;
  double total = 0.0;
  auto value = [&](uint32_t t) {
    const float p = load_as_f32(a.p, pr + t, a.dtype);
    const float q = !refused ? 0.0f : a.q ? load_as_f32(a.q, qr + t, a.dtype) : (int32_t)t == certain ? 1.0f : 0.0f;
    return left_of(p, q);
  };
  for (int round = 0; round < 2; round++) {  // the second only where the difference leaves nothing
    double sum = 0.0;
    int last = -1;
    for (uint32_t t = t0; t < t1; t++) {
      const double v = value(t);
      sum += v;
      if (v > 0.0) last = (int)t;
    }
    part[tid] = sum;
    if (last >= 0) atomicMax(&last_s, last);
    __syncthreads();
    if (tid == 0)
      for (int i = 1; i < VD_THREADS; i++) part[i] += part[i - 1];
    __syncthreads();
    total = part[VD_THREADS - 1];
    if (last_s >= 0 || !refused) break;
    refused = false;
  }
  const double goal = (double)a.u[(size_t)b * (a.n_max + 1) + a.n_max] * total;
  __shared__ int drawn;
  if (tid == 0) drawn = last_s < 0 ? 0 : last_s;
  __syncthreads();
  double run = tid ? part[tid - 1] : 0.0;
  if (part[tid] > goal && !(run > goal))
    for (uint32_t t = t0; t < t1; t++) {
      run += value(t);
      if (run > goal) {
        atomicMin(&drawn, (int)t);
        break;
      }
    }
  __syncthreads();
  if (tid <= a.n_max)
    a.tokens[(size_t)b * (a.n_max + 1) + tid] =
        tid < taken ? a.draft[(size_t)b * a.n_max + tid] : tid == taken ? drawn : -1;
  if (tid == 0) a.accepted[b] = (int32_t)taken;
}

}  // namespace

cudaError_t verify_draft_run(const VerifyArgs& a, cudaStream_t s) {
  k_verify_draft<<<a.n_seqs, VD_THREADS, 0, s>>>(a);
  return cudaGetLastError();
}

}  // namespace nrc
