// Norm of every query and key head and the position rotation, in one pass over a
// projection's output (gfx950). For a head x of D channels at position t:
//
//   y = x * rsqrt(mean(x^2) + eps) * w          (y = x without a weight)
//   (a, b) -> (a cos u - b sin u, b cos u + a sin u),   u = t * inv_freq_j,
//
// over the pairs j < R / 2, channels (j, j + R/2) or (2j, 2j + 1), times rotary_scale;
// channels from R on pass. Everything times the side's scale; queries are rounded once to
// their type, keys stay float32, as the cache takes them.
//
// The angle is formed in 64 bits as a number of turns, whose whole part is dropped before
// it is rounded to 32: a float32 product is off by 2^-24 of the angle, 0.006 at 100000.
//
// A wave a head.

#include "decode_common.hpp"

namespace fdi4 {

// Cosine and sine of position t times frequency f.
__device__ __forceinline__ void turn_of(int t, float f, float& cs, float& sn) {
  const double turns = (double)t * ((double)f * 0.15915494309189535);
  const float part = (float)(turns - rint(turns));
  sincospif(2.f * part, &sn, &cs);
}

__global__ __launch_bounds__(256) void norm_rotary_kernel(RotaryArgs a) {
  const int lane = threadIdx.x & 63, D = a.head_dim, half = a.rotary / 2;
  const int all = a.heads[0] + a.heads[1];
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.batch * a.tokens * all) return;
  const int64_t bt = row / all;
  const int hh = (int)(row - bt * all), b = (int)(bt / a.tokens), i = (int)(bt % a.tokens);
  const int side = hh >= a.heads[0], h = side ? hh - a.heads[0] : hh;
  const int64_t x0 = (int64_t)b * a.x_b[side] + (int64_t)h * a.x_h[side] + (int64_t)i * a.x_t[side];
  const int64_t o0 = (((int64_t)b * a.heads[side] + h) * a.tokens + i) * D;
  const int t = a.positions[(int64_t)b * a.p_b + (int64_t)i * a.p_t] + (a.p_t ? 0 : i);
  float norm = 1.f;
  if (a.weight[side]) {
    float s = 0.f;
    for (int d = lane; d < D; d += 64) {
      const float x = load_elem(a.x[side], x0 + d, a.dtype);
      s = __builtin_fmaf(x, x, s);
    }
    norm = 1.f / sqrtf(allreduce_sum<1, 64>(s) / (float)D + a.eps);
  }
  auto value = [&](int d) {
    const float x = load_elem(a.x[side], x0 + d, a.dtype);
    return a.weight[side] ? x * norm * load_elem(a.weight[side], d, a.weight_dtype) : x;
  };
  const int dt = side ? (int)kEF32 : a.dtype;
  for (int p = lane; p < D / 2; p += 64) {
    if (p < half) {
      const int d0 = a.interleaved ? 2 * p : p, d1 = a.interleaved ? 2 * p + 1 : p + half;
      float cs, sn;
      turn_of(t, a.inv_freq[p], cs, sn);
      cs *= a.rotary_scale;
      sn *= a.rotary_scale;
      const float y0 = value(d0), y1 = value(d1);
      store_elem(a.out[side], o0 + d0, dt, (y0 * cs - y1 * sn) * a.scale[side]);
      store_elem(a.out[side], o0 + d1, dt, (y1 * cs + y0 * sn) * a.scale[side]);
    } else {
      const int d = a.rotary + 2 * (p - half);
      store_elem(a.out[side], o0 + d, dt, value(d) * a.scale[side]);
      store_elem(a.out[side], o0 + d + 1, dt, value(d + 1) * a.scale[side]);
    }
  }
}

hipError_t launch_norm_rotary(const RotaryArgs& a, hipStream_t st) {
  const int64_t rows = (int64_t)a.batch * a.tokens * (a.heads[0] + a.heads[1]);
  hipLaunchKernelGGL(norm_rotary_kernel, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a);
  return hipGetLastError();
}

}  // namespace fdi4
