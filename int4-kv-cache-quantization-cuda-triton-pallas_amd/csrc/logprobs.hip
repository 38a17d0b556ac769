// Log probabilities of given tokens, the entropy of every row and its most likely
// alternatives, from logits (gfx950). With x the row's logits (capped: cap*tanh(x/cap)),
// m their maximum, l = sum exp(x - m) and s = sum exp(x - m) (x - m):
//
//   logprob = x[token] - m - log l,   entropy = log l - s / l
//   alternatives: the largest logits, ties to the lowest index, as log probabilities
//
// A logit of -infinity has the probability zero, also under a cap, and adds nothing to the
// entropy; a NaN, +infinity or a row of -infinity makes the row's results NaN. A negative token gives 0
// (a place without one), a token past the vocabulary NaN. NaN logits come first among the
// alternatives.
//
// A workgroup of NT threads takes a row in segments of 8 NT 16-byte vectors, a segment in
// registers: its maximum, then one exponential a logit. A thread keeps its own m, l and s,
// and they meet at the end. Bound: memory with 16-bit logits and no cap (2048 rows of 128000
// bfloat16 logits: 97 us, 5.4 TB/s); with a cap the vector units, which take some 20
// instructions a logit, two of them a quarter as fast (777 rows of 50021, 20 alternatives: 52 us).
//
// Alternatives: a thread also keeps the largest logit that it has met. The K-th largest of 64
// groups' such maxima is at most the K-th largest logit, so only logits from there on are
// candidates; every wave finds that bound by itself (18 of its bits, with ballots), and few
// vectors hold one. The candidates (some K a segment, fewer as the bound rises) are ranked
// once, by counting. Rows with more than kCandidates of them are read again for each
// alternative: those with thousands of ties, and those masked with a finite value where fewer
// than K of the groups hold another logit (4 rows of 32000 float32 logits, all but five at the
// lowest number: 13 us for 5 alternatives, 138 for 20, where usual rows take 11 and 10).

#include <algorithm>

#include "attend_common.hpp"

namespace fdi4 {

constexpr int kVectors = 8;              // 16-byte vectors of a thread in a segment
constexpr int kCandidates = 2048;
// Up to so many rows (one a CU) workgroups of 1024 threads: 4 rows of 32000 float32 logits with
// five alternatives 8.7 us, with 256 threads 15.7; 300 rows 20.6 and 20.1.
constexpr int kFewLogitRows = 256;

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

// Caps up to here take the short form, off by 2^-22 of the cap, 2^-16 at most: no more than four
// float32 steps of a logit of that size. (777 rows of 50021 float16 logits, 20 alternatives: 52
// us so, 66 by the long form.)
constexpr float kQuickCap = 64.f;

// A capped logit; infinite ones stay so (a product with the smallest number adds nothing to
// others). QUICK: caps up to kQuickCap.
template <bool QUICK>
__device__ __forceinline__ float cap_logit(float x, float cap) {
  return __builtin_fmaf(x, 1.4e-45f, QUICK ? quick_cap(x, cap, 2.f * kLog2eF / cap)
                                           : soft_cap(x, cap, 1.f / cap));
}

__device__ __forceinline__ uint64_t max_u64(uint64_t x, uint64_t y) { return x > y ? x : y; }

// Ranks `count` different candidates by counting and keeps the largest `top` in order.
template <int NT>
__device__ __forceinline__ void rank_candidates(const uint64_t* keys, int count, int top,
                                                uint64_t* sorted) {
  for (int i = threadIdx.x; i < count; i += NT) {
    const uint64_t x = keys[i];
    int rank = 0;
#pragma unroll 4
    for (int k = 0; k < count; ++k) rank += keys[k] > x;
    if (rank < top) sorted[rank] = x;
  }
}

struct LogSums {
  float m, l, s;                         // sum exp(x - m), sum exp(x - m) (x - m)
};

// How far a maximum lies below another one, as sums are rescaled by it: exp(-200) is zero, and
// where a row is masked with the type's lowest value the difference times a sum would be
// infinite, and zero times that NaN.
__device__ __forceinline__ float below(float m, float top) { return fmaxf(m - top, -200.f); }

__device__ __forceinline__ LogSums join(LogSums a, LogSums b) {
  LogSums r;
  r.m = fmaxf(a.m, b.m);
  const float da = below(a.m, r.m), db = below(b.m, r.m);
  const float ea = __builtin_amdgcn_exp2f(da * kLog2eF), eb = __builtin_amdgcn_exp2f(db * kLog2eF);
  r.l = __builtin_fmaf(a.l, ea, b.l * eb);
  r.s = __builtin_fmaf(__builtin_fmaf(a.l, da, a.s), ea, __builtin_fmaf(b.l, db, b.s) * eb);
  return r;
}

template <int MASK>
__device__ __forceinline__ LogSums join_lanes(LogSums a) {
  LogSums b;
  b.m = xchg<MASK>(a.m);
  b.l = xchg<MASK>(a.l);
  b.s = xchg<MASK>(a.s);
  return join(a, b);
}

template <int DT, bool TOP, int NT>
__global__ __launch_bounds__(NT, 4) void token_logprobs_kernel(LogprobArgs a) {
  constexpr int EV = DT == kEF32 ? 4 : 8;              // elements of a vector
  constexpr int EB = DT == kEF32 ? 4 : 2;
  constexpr int NW = NT / 64, GL = NT / 64;            // waves; lanes of a group
  // -infinity in both halves of a word (float32: in the word).
  constexpr unsigned kNone = DT == kEF32 ? 0xFF800000u : DT == kEF16 ? 0xFC00FC00u : 0xFF80FF80u;
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int64_t row = a.first + blockIdx.x;
  const int64_t x0 = row / a.inner * a.s_outer + row % a.inner * a.s_inner;
  const char* base = static_cast<const char*>(a.x) + x0 * EB;
  // Element 0 of vector 0 is at -skew: vectors lie on 16-byte boundaries.
  const int skew = (int)((uintptr_t)base % 16) / EB;
  const int vectors = (int)(((int64_t)a.vocab + skew + EV - 1) / EV);
  const int segments = (vectors + NT * kVectors - 1) / (NT * kVectors);
  // A logit as the softmax has it.
  auto capped = [&](float x) {
    return !(a.cap > 0.f) ? x : a.cap <= kQuickCap ? cap_logit<true>(x, a.cap)
                                                   : cap_logit<false>(x, a.cap);
  };

  __shared__ uint64_t list_s[TOP ? kCandidates : 1];
  __shared__ uint64_t sorted_s[TOP ? kMaxTop : 1];
  __shared__ unsigned group_s[2][64];
  __shared__ int count_s;
  __shared__ LogSums sums_s[NW];
  __shared__ uint64_t best_s[NW];
  unsigned largest = 0, low = 0;                       // of this thread; the bound
  if (TOP && tid == 0) count_s = 0;

  auto widen = [](U32x4 v, float* x) __attribute__((always_inline)) {
    widen_values<DT == kEF32 ? kVF32 : DT == kEF16 ? kVF16 : kVBF16>(v, x);
  };
  // Vector v of the row, -infinity for what lies before and behind it.
  auto load = [&](int v) __attribute__((always_inline)) -> U32x4 {
    const int64_t e0 = (int64_t)v * EV - skew;
    if (e0 >= 0 && e0 + EV <= a.vocab) return ld16(base + e0 * EB);
    unsigned y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (DT == kEF32) {
        y[j] = e0 + j >= 0 && e0 + j < a.vocab
                   ? reinterpret_cast<const unsigned*>(base)[e0 + j] : kNone;
      } else {
        const unsigned short* p = reinterpret_cast<const unsigned short*>(base);
        const int64_t e = e0 + 2 * j;
        y[j] = (e >= 0 && e < a.vocab ? p[e] : kNone & 0xFFFFu) |
               (e + 1 >= 0 && e + 1 < a.vocab ? (unsigned)p[e + 1] << 16 : kNone << 16);
      }
    }
    return U32x4{y[0], y[1], y[2], y[3]};
  };

  LogSums t = {kLeastF, 0.f, 0.f};
#pragma unroll 1
  for (int seg = 0; seg < segments; ++seg) {
    const int v0 = seg * NT * kVectors + tid;
    // Vectors a thread has here (uniform; the last may be behind the row).
    const int nk = min(kVectors, (vectors - seg * NT * kVectors + NT - 1) / NT);
    U32x4 raw[kVectors];
    if (seg + 1 < segments && (seg > 0 || skew == 0)) {
#pragma unroll
      for (int k = 0; k < kVectors; ++k)
        raw[k] = ld16(base + ((int64_t)(v0 + NT * k) * EV - skew) * EB);
    } else {
#pragma unroll
      for (int k = 0; k < kVectors; ++k)
        if (k < nk) raw[k] = load(v0 + NT * k);
    }
    float mv[kVectors], mx = -INFINITY;
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
      if (k < nk) {
        float x[EV];
        widen(raw[k], x);
        mv[k] = x[0];
#pragma unroll
        for (int j = 1; j < EV; ++j) mv[k] = fmaxf(mv[k], x[j]);
        mx = fmaxf(mx, mv[k]);
      }
    // (Of the logits as they are; a cap rises with them.)
    const float mn = fmaxf(t.m, capped(mx));
    const float dm = below(t.m, mn), g = __builtin_amdgcn_exp2f(dm * kLog2eF);
    t.s = __builtin_fmaf(t.l, dm, t.s) * g;
    t.l *= g;
    t.m = mn;
    float l2[2] = {0.f, 0.f}, s2[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kVectors; ++k)
      if (k < nk) {
        float x[EV];
        widen(raw[k], x);
        if (a.cap > 0.f) {
          if (a.cap <= kQuickCap) {
#pragma unroll
            for (int j = 0; j < EV; ++j) x[j] = cap_logit<true>(x[j], a.cap);
          } else {
#pragma unroll
            for (int j = 0; j < EV; ++j) x[j] = cap_logit<false>(x[j], a.cap);
          }
        }
#pragma unroll
        for (int j = 0; j < EV; ++j) {
          const float d = x[j] - mn, e = __builtin_amdgcn_exp2f(d * kLog2eF);
          l2[j & 1] += e;
          // (-infinity weighs nothing: 0 times a finite number.)
          s2[j & 1] = __builtin_fmaf(e, fmaxf(d, -1e30f), s2[j & 1]);
        }
      }
    const float lt = l2[0] + l2[1];
    t.l += lt;
    t.s += s2[0] + s2[1];

    if constexpr (TOP) {
      // A NaN among the thread's logits comes before all. Its sum is NaN then, but so is that
      // with +infinity alone.
      unsigned mine = order_of(mx);
      if (lt != lt) {
#pragma unroll
        for (int k = 0; k < kVectors; ++k)
          if (k < nk) {
            float x[EV];
            widen(raw[k], x);
#pragma unroll
            for (int j = 0; j < EV; ++j) mine = max(mine, order_of(x[j]));
          }
      }
      const bool nan = mine == 0xFFFFFFFFu;
      largest = max(largest, mine);
      unsigned gm = largest;
      if constexpr (GL >= 2) gm = max(gm, xchg_u32<1>(gm));
      if constexpr (GL >= 4) gm = max(gm, xchg_u32<2>(gm));
      if constexpr (GL >= 8) gm = max(gm, xchg_u32<4>(gm));
      if constexpr (GL >= 16) gm = max(gm, xchg_u32<8>(gm));
      if (tid % GL == 0) group_s[seg & 1][tid / GL] = gm;
      // (The other buffer may still be read by a wave that is a segment behind.)
      __syncthreads();
      if (__builtin_amdgcn_ballot_w64(mine >= low)) {
        const unsigned v = group_s[seg & 1][lane];
        unsigned bound = 0;
#pragma unroll
        for (int bit = 31; bit >= 14; --bit) {
          const unsigned more = bound | 1u << bit;
          if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(v >= more)) >= a.top) bound = more;
        }
        low = max(low, bound);
        if (mine >= low) {
#pragma unroll
          for (int k = 0; k < kVectors; ++k)
            if (k < nk && (nan || order_of(mv[k]) >= low)) {
              float x[EV];
              widen(raw[k], x);
              const int64_t e0 = (int64_t)(v0 + NT * k) * EV - skew;
#pragma unroll
              for (int j = 0; j < EV; ++j)
                if (e0 + j >= 0 && e0 + j < a.vocab && order_of(x[j]) >= low) {
                  const int at = atomicAdd(&count_s, 1);
                  if (at < kCandidates) list_s[at] = candidate(x[j], (int)(e0 + j));
                }
            }
        }
      }
    }
  }

  t = join_lanes<1>(t);
  t = join_lanes<2>(t);
  t = join_lanes<4>(t);
  t = join_lanes<8>(t);
  t = join_lanes<16>(t);
  t = join_lanes<32>(t);
  if (lane == 0) sums_s[w] = t;
  __syncthreads();
  t = sums_s[0];
#pragma unroll
  for (int k = 1; k < NW; ++k) t = join(t, sums_s[k]);
  const float log_l = logf(t.l);
  auto log_of = [&](float x) { return capped(x) - t.m - log_l; };
  if (tid == 0) {
    const int64_t tok = a.tokens[row];
    a.logprobs[row] = tok < 0 ? 0.f
                      : tok >= a.vocab ? __builtin_nanf("")
                                       : log_of(load_elem(a.x, x0 + tok, a.dtype));
    a.entropy[row] = log_l - t.s / t.l;
  }
  if constexpr (TOP) {
    if (count_s <= kCandidates) {
      rank_candidates<NT>(list_s, count_s, a.top, sorted_s);
    } else {
      // The best that is left, `top` times. (The first may be any: NaN at index 0 is ~0.)
      uint64_t last = ~0ull;
#pragma unroll 1
      for (int i = 0; i < a.top; ++i) {
        uint64_t best = 0;
#pragma unroll 1
        for (int v = tid; v < vectors; v += NT) {
          float x[EV];
          widen(load(v), x);
          const int64_t e0 = (int64_t)v * EV - skew;
#pragma unroll
          for (int j = 0; j < EV; ++j) {
            const uint64_t key = candidate(x[j], (int)(e0 + j));
            if (e0 + j >= 0 && e0 + j < a.vocab && (i == 0 || key < last))
              best = max_u64(best, key);
          }
        }
        for (int o = 1; o < 64; o *= 2) best = max_u64(best, __shfl_xor(best, o, 64));
        if (lane == 0) best_s[w] = best;
        __syncthreads();
        last = best_s[0];
        for (int k = 1; k < NW; ++k) last = max_u64(last, best_s[k]);
        if (tid == 0) sorted_s[i] = last;
        __syncthreads();
      }
    }
    __syncthreads();
    if (tid < a.top) {
      const uint64_t x = sorted_s[tid];
      a.top_logprobs[row * a.top + tid] = log_of(logit_of((unsigned)(x >> 32)));
      a.top_ids[row * a.top + tid] = (int)~(unsigned)x;
    }
  }
}

// Rows of a launch; more take another one.
constexpr int kMostRows = 1 << 22;

template <int DT, int NT>
void launch_logprobs(LogprobArgs a, hipStream_t st) {
  for (a.first = 0; a.first < a.rows; a.first += kMostRows) {
    const dim3 grid((unsigned)std::min<int64_t>(a.rows - a.first, kMostRows));
    if (a.top)
      hipLaunchKernelGGL((token_logprobs_kernel<DT, true, NT>), grid, dim3(NT), 0, st, a);
    else
      hipLaunchKernelGGL((token_logprobs_kernel<DT, false, NT>), grid, dim3(NT), 0, st, a);
  }
}

hipError_t launch_token_logprobs(const LogprobArgs& a, hipStream_t st) {
  const bool few = a.rows <= kFewLogitRows;
  if (a.dtype == kEF32) few ? launch_logprobs<kEF32, 1024>(a, st) : launch_logprobs<kEF32, 256>(a, st);
  if (a.dtype == kEF16) few ? launch_logprobs<kEF16, 1024>(a, st) : launch_logprobs<kEF16, 256>(a, st);
  if (a.dtype == kEBF16)
    few ? launch_logprobs<kEBF16, 1024>(a, st) : launch_logprobs<kEBF16, 256>(a, st);
  return hipGetLastError();
}

}  // namespace fdi4
