// Attention of the last tokens of every sequence over the paged INT4 cache that holds
// them (gfx950). Query i of sequence b, with n cached tokens and c queries, is at
// position p = n - c + i and sees the tokens
//
//   t < prefix,  t <= p with t < sinks or t > p - window;
//
//   x_t = cap * tanh(q . k_t / cap) - slope * |p - t|,  k_t = nib*scale - zp*scale,
//   out = sum_t p_t v_t / sum_t p_t,  p_t = exp(x_t - max).
//
// A row that sees nothing, and the queries i >= c, are zero.
//
// Here: what the two kernels share (up to 32 rows a kv-head: attend_few.hip; more:
// attend_chunk.hip), namely what a row sees, its logits, and the computation of a row by
// itself.
#pragma once

#include "decode_common.hpp"

namespace fdi4 {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef unsigned v4u __attribute__((ext_vector_type(4)));

constexpr int kKeyTile = 64;             // keys of a tile, within one scale group
constexpr float kLog2eF = 1.44269504088896f;
constexpr float kLeastF = -3.4028235e38f;

// The cached tokens that a row sees: t < head, and low <= t <= pos.
struct RowView {
  int head, low, pos;                    // pos: -1 or the row's own position, below n
};

__device__ __forceinline__ RowView row_view(const AttendArgs& a, int n, int cnt, int prefix,
                                            int i) {
  RowView v;
  const int p = n - cnt + i;
  const bool live = i < cnt;
  v.pos = live ? max(p, -1) : -1;
  v.low = a.window ? max(p - a.window + 1, 0) : 0;
  v.head = max(a.window ? min(a.sinks, p + 1) : 0, prefix);
  v.head = live ? max(min(v.head, n), 0) : 0;
  return v;
}

__device__ __forceinline__ bool sees(const RowView& v, int t) {
  return t < v.head || (t >= v.low && t <= v.pos);
}

__device__ __forceinline__ bool sees_any(const RowView& v) {
  return v.head > 0 || v.low <= v.pos;
}

// Queries of sequence b in use, and the tokens that all of them see.
__device__ __forceinline__ int count_of(const AttendArgs& a, int b) {
  return a.counts ? min(max(ld_ro(a.counts, b), 0), a.queries) : a.queries;
}

__device__ __forceinline__ int prefix_of(const AttendArgs& a, int b, int n) {
  return a.prefix ? min(max(ld_ro(a.prefix, b), 0), n) : 0;
}

// cap * tanh(x / cap) in float32, to 2^-20 of itself: with e = exp(-2|y|), y = x / cap, tanh|y| = (1 - e) / (1 +
// e). Its error is that of 1 - e, 2^-24, so below |y| = 0.35 the odd Taylor series takes
// over (to y^13: its next term is below 2^-28 of the sum).
__device__ __forceinline__ float soft_cap(float x, float cap, float inv_cap) {
  const float y = x * inv_cap, z = fabsf(y);
  const float e = __builtin_amdgcn_exp2f(z * (-2.f * kLog2eF));
  const float big = (1.f - e) * __builtin_amdgcn_rcpf(1.f + e);
  const float w = y * y;
  float s = 21844.f / 6081075.f;
  s = __builtin_fmaf(s, w, -1382.f / 155925.f);
  s = __builtin_fmaf(s, w, 62.f / 2835.f);
  s = __builtin_fmaf(s, w, -17.f / 315.f);
  s = __builtin_fmaf(s, w, 2.f / 15.f);
  s = __builtin_fmaf(s, w, -1.f / 3.f);
  const float small = __builtin_fmaf(z * w, s, z);
  const float t = z < 0.35f ? small : big;       // (NaN: big)
  return cap * __builtin_copysignf(t, y);
}

// The same to 2^-22 of the cap, in five instructions: cap - 2 cap / (1 + exp(2 y)). scale is 2
// log2(e) / cap. That error has the size of the cap, not of the score: 0.1 for a cap of 1e6. So
// the kernels take it up to a cap of their own (attend_wide, and the token log probabilities').
__device__ __forceinline__ float quick_cap(float x, float cap, float scale) {
  const float e = __builtin_amdgcn_exp2f(x * scale);
  return __builtin_fmaf(-2.f * cap, __builtin_amdgcn_rcpf(1.f + e), cap);
}

// The tiles of kKeyTile keys that a range of rows needs: those of [0, head) and, behind
// them, those of [low, pos].
struct TileList {
  int front, from, total;

  __device__ __forceinline__ int tile(int j) const { return j < front ? j : j - front + from; }
};

__device__ __forceinline__ TileList tile_list(int head, int low, int pos) {
  TileList l;
  l.front = (head + kKeyTile - 1) / kKeyTile;
  l.from = max(low / kKeyTile, l.front);
  l.total = l.front + max(pos / kKeyTile + (pos >= 0) - l.from, 0);
  return l;
}

// Whether a row sees a key of the tiles [j0, j1) of a list.
__device__ __forceinline__ bool sees_tiles(const RowView& v, const TileList& l, int j0, int j1) {
  auto in = [&](int t0, int t1) {
    return t0 < t1 && (t0 < v.head || max(t0, v.low) <= min(t1 - 1, v.pos));
  };
  const int f1 = min(j1, l.front), b0 = max(j0, l.front);
  return in(j0 * kKeyTile, f1 * kKeyTile) ||
         in((b0 - l.front + l.from) * kKeyTile, (j1 - l.front + l.from) * kKeyTile);
}

// ---- terms of 16 bits ---------------------------------------------------------

__device__ __forceinline__ unsigned pack_f16(float x, float y) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v2f{x, y}, v2h));
}

__device__ __forceinline__ unsigned pack_bf16(float x, float y) {
  return __builtin_bit_cast(unsigned, __builtin_convertvector(v2f{x, y}, v2bf));
}

// The upper halves of x and y: bfloat16 terms by truncation.
__device__ __forceinline__ unsigned pack_high(float x, float y) {
  return __builtin_amdgcn_perm(f2u(y), f2u(x), 0x07060302u);
}

__device__ __forceinline__ float less_high(float x) { return x - u2f(f2u(x) & 0xFFFF0000u); }

// Exponent e of |x| < 2^(e + 1) from the bits of |x| (0 and subnormals: -126).
__device__ __forceinline__ int exponent_of(unsigned bits) {
  return max((int)(bits >> 23), 1) - 127;
}

// ---- a row by itself ------------------------------------------------------------

// The kernel's arguments, read again from where they lie: what follows a kernel's loop
// uses this copy, so that its arguments hold no scalar registers in the loop.
__device__ __forceinline__ const AttendArgs& late_attend_args() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const AttendArgs*)p;
}

// Sums of one row over the tiles [j0, j1) of a list, by one wave: o[k] belongs to channel
// lane * (D / 64) + k. Keys that the row does not see take no part at all, so values and
// scales that are not finite come out as the formula has them. m = kLeastF and l = 0 if
// it sees nothing; m = -infinity and l = 0 if all logits are.
template <int D>
struct RowSums {
  float m, l, o[D / 64];
};

template <int D, int VDT>
__device__ __forceinline__ RowSums<D> plain_row(const AttendArgs& a, int b, int hk,
                                                          int R, int n, RowView view,
                                                          TileList list, int j0, int j1) {
  const DecodeArgs& c = a.c;
  constexpr int CH = D / 64;
  const int lane = threadIdx.x & 63;
  const int i = R / c.hq_per_kv, h = hk * c.hq_per_kv + R % c.hq_per_kv;
  const int64_t q0 = (int64_t)b * c.q_b + (int64_t)h * c.q_h + (int64_t)i * a.q_n;
  const float* sbase = c.k_scale + (int64_t)b * c.s_b + (int64_t)hk * c.s_h;
  const float* zbase = c.k_zp + (int64_t)b * c.s_b + (int64_t)hk * c.s_h;
  const int32_t* table = c.page_table ? c.page_table + (int64_t)b * c.pt_b : nullptr;
  const float slope = a.slopes ? a.slopes[h] : 0.f;
  const float inv_cap = 1.f / a.cap;
  RowSums<D> r;
  r.m = kLeastF;
  r.l = 0.f;
  for (int k = 0; k < CH; ++k) r.o[k] = 0.f;
#pragma unroll 1
  for (int j = j0; j < j1; ++j) {
    const int t0 = list.tile(j) * kKeyTile, t = t0 + lane;
    const bool mine = t < n && sees(view, t);
    const uint64_t who = __builtin_amdgcn_ballot_w64(mine);
    if (!who) continue;
    // Lane: a key's logit.
    const int tc = min(t, n - 1), lp = fdiv(tc, c.div_rows), tr = tc - lp * c.page_rows;
    const int64_t phys = min(max(table ? table[lp] : lp, 0), c.num_pages - 1);
    const uint8_t* kp =
        c.k_pages + phys * c.k_page + (int64_t)hk * c.k_head + (int64_t)tr * c.k_row;
    const int64_t g = (int64_t)fdiv(t0, a.div_group) * c.s_g;
    float x = 0.f;
#pragma unroll 1
    for (int d = 0; d < D; ++d) {
      const float s = sbase[g + d], z = zbase[g + d];
      const float k = (float)((kp[d >> 1] >> (4 * (d & 1))) & 15) * s - z * s;
      x = __builtin_fmaf(load_elem(c.q, q0 + d, c.q_dtype), k, x);
    }
    if (a.cap > 0.f) x = soft_cap(x, a.cap, inv_cap);
    if (a.slopes) x -= slope * (float)abs(view.pos - t);
    // (fmaxf drops a NaN; its probability below is NaN.)
    const float mt = allreduce_max_f<1, 64>(mine ? x : -INFINITY);
    const float mn = r.l > 0.f || r.m == -INFINITY ? fmaxf(r.m, mt) : mt;
    // A key with a logit of -infinity beside finite ones weighs nothing; where all are,
    // the caller makes the row NaN.
    const float p = !mine || (x == -INFINITY && mn == -INFINITY)
                        ? 0.f : __builtin_amdgcn_exp2f((x - mn) * kLog2eF);
    const float f = r.l > 0.f ? __builtin_amdgcn_exp2f((r.m - mn) * kLog2eF)
                              : (r.l == 0.f ? 0.f : r.l);
    r.m = mn;
    r.l = r.l * f + allreduce_sum<1, 64>(p);
    for (int k = 0; k < CH; ++k) r.o[k] *= f;
    // Lane: its channels of every value.
    const int64_t vrow = phys * c.v_page + (int64_t)hk * c.v_head + (int64_t)tr * c.v_row;
#pragma unroll 1
    for (int e = 0; e < kKeyTile; ++e) {
      if (!(who >> e & 1u)) continue;
      const float pe = __shfl(p, e, 64);
      const int64_t ve = __shfl(vrow, e, 64);
      for (int k = 0; k < CH; ++k)
        r.o[k] = __builtin_fmaf(pe, load_elem(c.v_pages, ve + lane * CH + k, VDT), r.o[k]);
    }
  }
  return r;
}

// A row's output, or its partial of a split: sums with weights exp2(log2e * logit - m2).
// `seen`: the row sees a key of the range.
template <int D>
__device__ __forceinline__ void store_plain_row(const AttendArgs& a, int b, int hk, int R,
                                                int split, const RowSums<D>& r, bool seen) {
  const DecodeArgs& c = a.c;
  constexpr int CH = D / 64;
  const int lane = threadIdx.x & 63;
  const int i = R / c.hq_per_kv, h = hk * c.hq_per_kv + R % c.hq_per_kv;
  const int64_t row = ((int64_t)b * c.num_q_heads + h) * a.queries + i;
  if (c.final_out) {
    const float inv = 1.f / r.l;
    for (int k = 0; k < CH; ++k)
      store_elem(c.out, row * D + lane * CH + k, c.out_dtype, seen ? r.o[k] * inv : 0.f);
    return;
  }
  const int64_t at = row * c.num_splits + split;
  for (int k = 0; k < CH; ++k) c.ws_acc[at * D + lane * CH + k] = r.o[k];
  if (lane == 0) {
    c.ws_ml[2 * at] = !seen ? -INFINITY : (r.l == 0.f ? kNoFinite : (double)r.m);
    c.ws_ml[2 * at + 1] = r.l;
  }
}

}  // namespace fdi4
