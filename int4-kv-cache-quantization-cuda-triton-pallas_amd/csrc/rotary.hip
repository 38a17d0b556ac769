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
// norm_rotary_kernel: a lane holds 16 channels of a head, eight pairs, so a pair never leaves
// its lane; D / 16 lanes are a head and a wave 1024 / D heads of one token. The token's cosines
// and sines are computed once a wave, one or two a lane, and go round through LDS. A wave
// takes several groups of heads of its token where there are waves enough without.
// Bound: memory. 8 sequences of 2048 tokens, 32 + 8 heads of 128 bfloat16 channels: 94 us, 3.9
// TB/s (element by element, a wave a head: 448 us).

#include <algorithm>

#include "decode_common.hpp"

namespace fdi4 {

// Cosine and sine of position t times frequency f.
__device__ __forceinline__ void turn_of(int64_t t, float f, float& cs, float& sn) {
  const double turns = (double)t * ((double)f * 0.15915494309189535);
  const float part = (float)(turns - rint(turns));
  sincospif(2.f * part, &sn, &cs);
}

// Eight elements of type DT from 16-byte loads, as float32.
template <int DT>
__device__ __forceinline__ void load8(const void* p, int64_t i, float* x) {
  if constexpr (DT == kEF32) {
    const float* f = static_cast<const float*>(p) + i;
    widen_values<kVF32>(ld16(f), x);
    widen_values<kVF32>(ld16(f + 4), x + 4);
  } else {
    widen_values<DT == kEF16 ? kVF16 : kVBF16>(ld16(static_cast<const unsigned short*>(p) + i), x);
  }
}

__device__ __forceinline__ unsigned pair_of(float x, float y, int dt) {
  if (dt == kEF16)
    return (unsigned)__builtin_bit_cast(unsigned short, (_Float16)x) |
           (unsigned)__builtin_bit_cast(unsigned short, (_Float16)y) << 16;
  return (unsigned)bf16_rne(x) | (unsigned)bf16_rne(y) << 16;
}

template <int DT>
__device__ __forceinline__ void store8(void* p, int64_t i, const float* x) {
  if constexpr (DT == kEF32) {
    float* f = static_cast<float*>(p) + i;
    st16(f, U32x4{f2u(x[0]), f2u(x[1]), f2u(x[2]), f2u(x[3])});
    st16(f + 4, U32x4{f2u(x[4]), f2u(x[5]), f2u(x[6]), f2u(x[7])});
  } else {
    st16(static_cast<unsigned short*>(p) + i,
         U32x4{pair_of(x[0], x[1], DT), pair_of(x[2], x[3], DT), pair_of(x[4], x[5], DT),
               pair_of(x[6], x[7], DT)});
  }
}

// Waves of a launch; more take another one.
constexpr int kMostWaves = 1 << 25;

// Item of a wave: (token, group of `chunk` rounds of heads).
template <int D, int DT>
__global__ __launch_bounds__(256) void norm_rotary_kernel(RotaryArgs a, int chunks, int rounds) {
  constexpr int LPR = D / 16, RPW = 64 / LPR;      // lanes a head, heads a round
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int j = lane % LPR, r = lane / LPR;
  const int item = a.first + (int)blockIdx.x * 4 + w;
  const int bt = item / chunks, chunk = item - bt * chunks;
  __shared__ float2 turn_s[4][D / 2];
  if (bt >= a.batch * a.tokens) return;
  const int b = bt / a.tokens, i = bt - b * a.tokens;
  const int half = a.rotary / 2, all = a.heads[0] + a.heads[1];

  // This lane's channels: eight from d0 and eight from d1.
  const bool turns = j < a.rotary / 16;
  const int d0 = turns && !a.interleaved ? 8 * j : 16 * j;
  const int d1 = turns && !a.interleaved ? half + 8 * j : 16 * j + 8;

  // The token's turns, pair 8 j + k of lane j's k-th.
  const int64_t t =
      (int64_t)a.positions[(int64_t)b * a.p_b + (int64_t)i * a.p_t] + (a.p_t ? 0 : i);
  float cs[8], sn[8];
#pragma unroll
  for (int k = 0; k < D / 2; k += 64) {
    const int p = k + lane;
    if (p < half) {
      float c, s;
      turn_of(t, a.inv_freq[p], c, s);
      turn_s[w][p] = make_float2(c * a.rotary_scale, s * a.rotary_scale);
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const float2 x = turns ? turn_s[w][8 * j + k] : make_float2(1.f, 0.f);
    cs[k] = x.x;
    sn[k] = x.y;
  }

  const int h1 = min((chunk + 1) * rounds * RPW, all);
  for (int h0 = chunk * rounds * RPW; h0 < h1; h0 += RPW) {
    const int hh = min(h0 + r, all - 1), side = hh >= a.heads[0];
    const int h = side ? hh - a.heads[0] : hh;
    const int64_t x0 =
        (int64_t)b * a.x_b[side] + (int64_t)h * a.x_h[side] + (int64_t)i * a.x_t[side];
    float x[16];
    load8<DT>(a.x[side], x0 + d0, x);
    load8<DT>(a.x[side], x0 + d1, x + 8);
    const void* wt = a.weight[side];
    if (wt) {
      float y[16];
      if (a.weight_dtype == kEF32) {
        load8<kEF32>(wt, d0, y);
        load8<kEF32>(wt, d1, y + 8);
      } else if (a.weight_dtype == kEF16) {
        load8<kEF16>(wt, d0, y);
        load8<kEF16>(wt, d1, y + 8);
      } else {
        load8<kEBF16>(wt, d0, y);
        load8<kEBF16>(wt, d1, y + 8);
      }
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        s[0] = __builtin_fmaf(x[k], x[k], s[0]);
        s[1] = __builtin_fmaf(x[8 + k], x[8 + k], s[1]);
      }
      const float sum = allreduce_sum<1, LPR>(s[0] + s[1]);
      const float norm = 1.f / sqrtf(sum * (1.f / D) + a.eps);
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = x[k] * norm * y[k];
    }
    const float scale = a.scale[side];
    if (turns) {
      if (a.interleaved) {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float u = x[2 * k], v = x[2 * k + 1];
          x[2 * k] = u * cs[k] - v * sn[k];
          x[2 * k + 1] = v * cs[k] + u * sn[k];
        }
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float u = x[k], v = x[8 + k];
          x[k] = u * cs[k] - v * sn[k];
          x[8 + k] = v * cs[k] + u * sn[k];
        }
      }
    }
#pragma unroll
    for (int k = 0; k < 16; ++k) x[k] *= scale;
    if (h0 + r < h1) {
      const int64_t o0 = (((int64_t)b * a.heads[side] + h) * a.tokens + i) * D;
      if (side) {
        store8<kEF32>(a.out[1], o0 + d0, x);
        store8<kEF32>(a.out[1], o0 + d1, x + 8);
      } else {
        store8<DT>(a.out[0], o0 + d0, x);
        store8<DT>(a.out[0], o0 + d1, x + 8);
      }
    }
  }
}

// Rows of any alignment and rotary dimensions: a wave a head, element by element.
__global__ __launch_bounds__(256) void norm_rotary_any_kernel(RotaryArgs a) {
  const int lane = threadIdx.x & 63, D = a.head_dim, half = a.rotary / 2;
  const int all = a.heads[0] + a.heads[1];
  const int64_t row = a.first + (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.batch * a.tokens * all) return;
  const int64_t bt = row / all;
  const int hh = (int)(row - bt * all), b = (int)(bt / a.tokens), i = (int)(bt % a.tokens);
  const int side = hh >= a.heads[0], h = side ? hh - a.heads[0] : hh;
  const int64_t x0 = (int64_t)b * a.x_b[side] + (int64_t)h * a.x_h[side] + (int64_t)i * a.x_t[side];
  const int64_t o0 = (((int64_t)b * a.heads[side] + h) * a.tokens + i) * D;
  const int64_t t =
      (int64_t)a.positions[(int64_t)b * a.p_b + (int64_t)i * a.p_t] + (a.p_t ? 0 : i);
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

template <int D>
hipError_t launch_rotary(RotaryArgs a, hipStream_t st) {
  const int all = a.heads[0] + a.heads[1], total = (all * D + 1023) / 1024;
  const int64_t tokens = (int64_t)a.batch * a.tokens;
  // Rounds of heads a wave: one while that leaves waves for fewer than 16 a SIMD.
  const int rounds = (int)std::min<int64_t>(std::max<int64_t>(tokens * total / 16384, 1), total);
  const int chunks = (total + rounds - 1) / rounds;
  for (int64_t i = 0; i < tokens * chunks; i += kMostWaves) {
    a.first = (int)i;
    const dim3 grid((unsigned)((std::min<int64_t>(tokens * chunks - i, kMostWaves) + 3) / 4));
    if (a.dtype == kEF32)
      hipLaunchKernelGGL((norm_rotary_kernel<D, kEF32>), grid, dim3(256), 0, st, a, chunks, rounds);
    else if (a.dtype == kEF16)
      hipLaunchKernelGGL((norm_rotary_kernel<D, kEF16>), grid, dim3(256), 0, st, a, chunks, rounds);
    else
      hipLaunchKernelGGL((norm_rotary_kernel<D, kEBF16>), grid, dim3(256), 0, st, a, chunks,
                         rounds);
  }
  return hipGetLastError();
}

hipError_t launch_norm_rotary(RotaryArgs a, hipStream_t st) {
  // Rows and weights by 16-byte loads, sixteen rotated channels a lane.
  if (a.vec && a.rotary % 16 == 0) {
    if (a.head_dim == 64) return launch_rotary<64>(a, st);
    if (a.head_dim == 128) return launch_rotary<128>(a, st);
    return launch_rotary<256>(a, st);
  }
  const int64_t rows = (int64_t)a.batch * a.tokens * (a.heads[0] + a.heads[1]);
  for (int64_t i = 0; i < rows; i += kMostWaves) {
    a.first = (int)i;
    const dim3 grid((unsigned)((std::min<int64_t>(rows - i, kMostWaves) + 3) / 4));
    hipLaunchKernelGGL(norm_rotary_any_kernel, grid, dim3(256), 0, st, a);
  }
  return hipGetLastError();
}

}  // namespace fdi4
