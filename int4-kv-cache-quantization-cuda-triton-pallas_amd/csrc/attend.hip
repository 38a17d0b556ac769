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
// Up to 32 rows a kv-head: attend_few.hip; more: attend_chunk.hip.

#include "attend_common.hpp"

namespace fdi4 {

hipError_t launch_attend(const AttendArgs& a, int D, int v_dtype, int batch, hipStream_t st) {
  return a.chunk ? launch_attend_chunk(a, D, v_dtype, batch, st)
                 : launch_attend_few(a, D, v_dtype, batch, st);
}

}  // namespace fdi4
