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
// A wave a row, a lane a key for the logits and a lane a channel for the values.

#include "attend_common.hpp"

namespace fdi4 {

template <int D, int VDT>
__global__ __launch_bounds__(256) void attend_plain_kernel(AttendArgs a) {
  const DecodeArgs& c = a.c;
  const int rows = c.hq_per_kv * a.queries;
  const int tiles = (rows + 3) / 4;
  const int wj = (int)blockIdx.x / tiles, R = ((int)blockIdx.x - wj * tiles) * 4 +
                                              (int)(threadIdx.x >> 6);
  const int b = wj / a.kv_heads, hk = wj - b * a.kv_heads;
  if (R >= rows) return;
  const int n = seq_len_of(c, b), split = blockIdx.y;
  const RowView v = row_view(a, n, count_of(a, b), prefix_of(a, b, n), R / c.hq_per_kv);
  const TileList list = tile_list(v.head, v.low, v.pos);
  const int j0 = (int)((int64_t)split * list.total / c.num_splits);
  const int j1 = (int)((int64_t)(split + 1) * list.total / c.num_splits);
  const RowSums<D> r = plain_row<D, VDT>(a, b, hk, R, n, v, list, j0, j1);
  store_plain_row<D>(a, b, hk, R, split, r, r.m != kLeastF);
}

template <int D>
hipError_t launch_attend_d(const AttendArgs& a, int v_dtype, int batch, hipStream_t st) {
  const int64_t rows = (int64_t)a.c.hq_per_kv * a.queries;
  const dim3 grid((unsigned)((rows + 3) / 4 * batch * a.kv_heads), a.c.num_splits);
#define FDI4_ATT(VV)                                                                       \
  if (v_dtype == VV) {                                                                     \
    hipLaunchKernelGGL((attend_plain_kernel<D, VV>), grid, dim3(256), 0, st, a);           \
    return hipGetLastError();                                                              \
  }
  FDI4_ATT(kVF32) FDI4_ATT(kVF16) FDI4_ATT(kVBF16)
#undef FDI4_ATT
  return hipErrorInvalidValue;
}

hipError_t launch_attend(const AttendArgs& a, int D, int v_dtype, int batch, hipStream_t st) {
  if (a.chunk) return launch_attend_chunk(a, D, v_dtype, batch, st);
  if (D == 64) return launch_attend_d<64>(a, v_dtype, batch, st);
  if (D == 128) return launch_attend_d<128>(a, v_dtype, batch, st);
  if (D == 256) return launch_attend_d<256>(a, v_dtype, batch, st);
  return hipErrorInvalidValue;
}

}  // namespace fdi4
