// Attention of several query rows per sequence over part of the paged INT4 cache
// and over drafted tokens (gfx950). For the row of node i and q-head h of sequence
// b, with n cached tokens and d_i drafts that node i sees,
//
//   out = sum_t p_t v_t / sum_t p_t,   p_t = exp(q . k_t - max)
//
// over the cached tokens t < n with t < sinks or t >= n + d_i - window (all of them
// without a window; d_i = 0 without drafts, the query being the last cached token),
// k_t = nib*scale - zp*scale, and over the drafts j with mask[i, j]. A row that sees
// nothing is zero.
//
// The plain form: one workgroup per row, a wave takes every fourth key.

#include "decode_common.hpp"

namespace fdi4 {

template <int D, int VDT>
__global__ __launch_bounds__(256) void decode_rows_kernel(RowsArgs a) {
  constexpr int CH = D / 64, W = 4;
  const DecodeArgs& c = a.c;
  const int row = blockIdx.x, b = blockIdx.y;
  const int hq = row / a.nodes, node = row % a.nodes;
  const int hk = hq / c.hq_per_kv;
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int n = seq_len_of(c, b);
  float q[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i)
    q[i] = load_elem(c.q, (int64_t)b * c.q_b + (int64_t)hq * c.q_h + (int64_t)node * a.q_n +
                              lane * CH + i, c.q_dtype);
  const uint8_t* mask =
      a.mask ? a.mask + (int64_t)b * a.mk_b + (int64_t)node * a.mk_i : nullptr;
  int mine = 0;
  if (mask)
    for (int j = 0; j < a.nodes; ++j) mine += mask[j] != 0;
  const int low = a.window ? min(max((int64_t)n + mine - a.window, (int64_t)0), (int64_t)n) : 0;
  const int sinks = min(a.sinks, low);
  const int cached = sinks + n - low;
  const int drafts = mask ? a.nodes : 0;
  float m = -INFINITY, l = 0.f, acc[CH] = {};
  for (int e = w; e < cached + drafts; e += W) {
    float k[CH], v[CH];
    if (e < cached) {
      const int t = e < sinks ? e : low + e - sinks;
      const int lp = t / c.page_rows, r = t % c.page_rows;
      const int pg = c.page_table ? c.page_table[(int64_t)b * c.pt_b + lp] : lp;
      const int64_t phys = min(max(pg, 0), c.num_pages - 1);
      const uint8_t* kp = c.k_pages + phys * c.k_page + (int64_t)hk * c.k_head +
                          (int64_t)r * c.k_row;
      const int64_t so = (int64_t)b * c.s_b + (int64_t)hk * c.s_h +
                         (int64_t)(lp / c.pages_per_group) * c.s_g;
      const int64_t vo = phys * c.v_page + (int64_t)hk * c.v_head + (int64_t)r * c.v_row;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const int d = lane * CH + i;
        const float s = c.k_scale[so + d], z = c.k_zp[so + d];
        k[i] = (float)((kp[d >> 1] >> (4 * (d & 1))) & 15) * s - z * s;
        v[i] = load_elem(c.v_pages, vo + d, VDT);
      }
    } else {
      const int j = e - cached;
      if (!mask[j]) continue;
      const float* kd = a.kd + (int64_t)b * a.kd_b + (int64_t)hk * a.kd_h + (int64_t)j * a.kd_n;
      const uint8_t* vd = a.vd + (int64_t)b * a.vd_b + (int64_t)hk * a.vd_h + (int64_t)j * a.vd_n;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        k[i] = kd[lane * CH + i];
        v[i] = load_elem(vd, lane * CH + i, VDT);
      }
    }
    float x = 0.f;
#pragma unroll
    for (int i = 0; i < CH; ++i) x = __builtin_fmaf(q[i], k[i], x);
    x = allreduce_sum<1, 64>(x);
    const float mn = fmaxf(m, x);
    const float f = exp2_of((double)m - (double)mn), p = exp2_of((double)x - (double)mn);
    m = mn;
    l = __builtin_fmaf(l, f, p);
#pragma unroll
    for (int i = 0; i < CH; ++i) acc[i] = __builtin_fmaf(acc[i], f, p * v[i]);
  }
  if (c.lens_out && blockIdx.x == 0 && threadIdx.x == 0) c.lens_out[b] = c.seq_lens[b];
  __shared__ float m_s[W], l_s[W], acc_s[W][D];
#pragma unroll
  for (int i = 0; i < CH; ++i) acc_s[w][lane * CH + i] = acc[i];
  if (lane == 0) {
    m_s[w] = m;
    l_s[w] = l;
  }
  __syncthreads();
  if (w) return;
  const float ms = fmaxf(fmaxf(m_s[0], m_s[1]), fmaxf(m_s[2], m_s[3]));
  float lt = 0.f, o[CH] = {};
  for (int i = 0; i < W; ++i) {
    if (m_s[i] == -INFINITY && l_s[i] == 0.f) continue;
    const float f = exp2_of((double)m_s[i] - (double)ms);
    lt = __builtin_fmaf(l_s[i], f, lt);
#pragma unroll
    for (int k = 0; k < CH; ++k) o[k] = __builtin_fmaf(acc_s[i][lane * CH + k], f, o[k]);
  }
#pragma unroll
  for (int k = 0; k < CH; ++k)
    store_elem(c.out, ((int64_t)b * gridDim.x + row) * D + lane * CH + k, c.out_dtype,
               lt == 0.f ? 0.f : o[k] / lt);
}

hipError_t launch_decode_rows(const RowsArgs& a, int D, int v_dtype, int batch, hipStream_t st) {
  dim3 grid(a.c.num_q_heads * a.nodes, batch);
#define FDI4_RW(DD, VV)                                                                     \
  if (D == DD && v_dtype == VV) {                                                           \
    hipLaunchKernelGGL((decode_rows_kernel<DD, VV>), grid, dim3(256), 0, st, a);            \
    return hipGetLastError();                                                               \
  }
  FDI4_RW(64, kVF32) FDI4_RW(64, kVF16) FDI4_RW(64, kVBF16)
  FDI4_RW(128, kVF32) FDI4_RW(128, kVF16) FDI4_RW(128, kVBF16)
  FDI4_RW(256, kVF32) FDI4_RW(256, kVF16) FDI4_RW(256, kVBF16)
#undef FDI4_RW
  return hipErrorInvalidValue;
}

}  // namespace fdi4
