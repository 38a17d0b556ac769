// Log probabilities of given tokens, the entropy of every row and its most likely
// alternatives, from logits (gfx950). With x the row's logits (capped: cap*tanh(x/cap)),
// m their maximum, l = sum exp(x - m) and s = sum exp(x - m) (x - m):
//
//   logprob = x[token] - m - log l,   entropy = log l - s / l
//   alternatives: the largest logits, ties to the lowest index, as log probabilities
//
// A logit of -infinity has the probability zero and adds nothing to the entropy; a NaN,
// +infinity or a row of -infinity makes the row's results NaN. A negative token gives 0
// (a place without one), a token past the vocabulary NaN. NaN logits come first among the
// alternatives.
//
// A workgroup a row.

#include "attend_common.hpp"

namespace fdi4 {

// A logit as a number whose order is the alternatives'.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = f2u(x + 0.f);       // (-0 is 0)
  if ((u & 0x7FFFFFFFu) > 0x7F800000u) return 0xFFFFFFFFu;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float logit_of(unsigned o) {
  if (o == 0xFFFFFFFFu) return __builtin_nanf("");
  return u2f(o & 0x80000000u ? o & 0x7FFFFFFFu : ~o);
}

// An alternative: larger is better, of equal logits the lower index.
__device__ __forceinline__ uint64_t candidate(float x, int i) {
  return (uint64_t)order_of(x) << 32 | (unsigned)~i;
}

__device__ __forceinline__ uint64_t max_u64(uint64_t x, uint64_t y) { return x > y ? x : y; }

__global__ __launch_bounds__(256) void token_logprobs_kernel(LogprobArgs a) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row = blockIdx.x;
  const int64_t x0 = row / a.inner * a.s_outer + row % a.inner * a.s_inner;
  const float inv_cap = 1.f / a.cap;
  auto at = [&](int i) {
    const float x = load_elem(a.x, x0 + i, a.dtype);
    return a.cap > 0.f ? soft_cap(x, a.cap, inv_cap) : x;
  };
  __shared__ float red[3][4];
  __shared__ uint64_t best_s[4];
  float m = -INFINITY;
  bool nan = false;
  for (int i = tid; i < a.vocab; i += 256) {
    const float x = at(i);
    nan |= x != x;
    m = fmaxf(m, x);
  }
  m = allreduce_max_f<1, 64>(nan ? INFINITY : m);
  if (lane == 0) red[0][w] = m;
  __syncthreads();
  m = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
  float l = 0.f, s = 0.f;
  for (int i = tid; i < a.vocab; i += 256) {
    const float d = at(i) - m, e = __builtin_amdgcn_exp2f(d * kLog2eF);
    l += e;
    if (d != -INFINITY) s = __builtin_fmaf(e, d, s);
  }
  l = allreduce_sum<1, 64>(l);
  s = allreduce_sum<1, 64>(s);
  if (lane == 0) {
    red[1][w] = l;
    red[2][w] = s;
  }
  __syncthreads();
  l = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
  s = (red[2][0] + red[2][1]) + (red[2][2] + red[2][3]);
  const float log_l = logf(l);
  if (tid == 0) {
    const int64_t tok = a.tokens[row];
    a.logprobs[row] = tok < 0 ? 0.f : tok >= a.vocab ? __builtin_nanf("")
                                                     : at((int)tok) - m - log_l;
    a.entropy[row] = log_l - s / l;
  }
  uint64_t last = ~0ull;
  for (int k = 0; k < a.top; ++k) {
    uint64_t best = 0;
    for (int i = tid; i < a.vocab; i += 256) {
      const uint64_t x = candidate(load_elem(a.x, x0 + i, a.dtype), i);
      if (x < last) best = max_u64(best, x);
    }
    for (int o = 1; o < 64; o *= 2) best = max_u64(best, __shfl_xor(best, o, 64));
    if (lane == 0) best_s[w] = best;
    __syncthreads();
    last = max_u64(max_u64(best_s[0], best_s[1]), max_u64(best_s[2], best_s[3]));
    __syncthreads();
    if (tid == 0) {
      float x = logit_of((unsigned)(last >> 32));
      if (a.cap > 0.f) x = soft_cap(x, a.cap, inv_cap);
      a.top_logprobs[row * a.top + k] = x - m - log_l;
      a.top_ids[row * a.top + k] = (int)~(unsigned)last;
    }
  }
}

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t st) {
  hipLaunchKernelGGL(token_logprobs_kernel, dim3((unsigned)a.rows), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace fdi4
