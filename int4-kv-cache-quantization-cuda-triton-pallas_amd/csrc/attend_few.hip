// Attention of a few cached tokens (gfx950): up to 16 rows a kv-head, one token of a decode
// step above all. Memory bound: what counts is that the cache is read once, in long runs.
//
// A workgroup of four waves takes the rows of one kv-head over a range of 64-key tiles,
// which go to the waves in turn. A wave loads 32 keys straight to registers and dequantizes
// them there (k = nib*s - zp*s as float16 in units of a power of two for the scale group's
// largest). The next keys are loaded as soon as these are multiplied, the next values as
// soon as these are. Waves meet at the end, in LDS, and splits in the merge kernel.
//
//   scores: v_mfma_f32_16x16x32_f16 of 16 keys (A) and 16 rows (B): lane (g, r) loads the
//      channels g * D/4 .. of key r and of row r, eight of them a product.
//   values: lane (g, r) holds the scores of row r with keys 4g .. 4g + 3 of both 16-key
//      halves, which is the B operand of a product of 32 keys, and loads the channels r *
//      D/16 .. of the same keys: byte permutes pair them.
//
// Terms as the kernel of many rows (attend_chunk.hip) has them, but two of keys also for
// 16-bit outputs: the vector units have time.

#include "attend_common.hpp"

namespace fdi4 {

typedef float v4f __attribute__((ext_vector_type(4)));

template <int D, int VDT, bool WIDE>
struct FewGeo {
  static constexpr int TQ = WIDE ? 2 : 1;
  static constexpr int TV = VDT == kVF32 ? (WIDE ? 3 : 2) : 1;
  static constexpr int TP = VDT == kVF16 ? (WIDE ? 2 : 1) : (WIDE ? 3 : 1);
  static constexpr int VEB = VDT == kVF32 ? 4 : 2;
  static constexpr int NK = D / 32;                    // products of a score; packed words a lane
  static constexpr int CH = D / 4;                     // key channels of a lane
  static constexpr int NA = D / 16;                    // value channels of a lane; output tiles
  static constexpr int VW = NA * VEB / 4;              // words of a value row a lane
  static constexpr int AS = D + 4;                     // floats of a row in LDS
};

__device__ __forceinline__ float over_quarters_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = fmaxf(u2f(r[0]), u2f(r[1]));
  auto s = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return fmaxf(u2f(s[0]), u2f(s[1]));
}

__device__ __forceinline__ float over_quarters_sum(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = u2f(r[0]) + u2f(r[1]);
  auto s = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return u2f(s[0]) + u2f(s[1]);
}

__device__ __forceinline__ unsigned over_quarters_umax(unsigned x) {
  auto r = __builtin_amdgcn_permlane16_swap(x, x, false, false);
  x = max((unsigned)r[0], (unsigned)r[1]);
  auto s = __builtin_amdgcn_permlane32_swap(x, x, false, false);
  return max((unsigned)s[0], (unsigned)s[1]);
}

template <int N>
struct Words {
  unsigned w[N];
};

template <int N>
__device__ __forceinline__ Words<N> load_stream(const uint8_t* p) {
  Words<N> r;
  if constexpr (N >= 4) {
#pragma unroll
    for (int k = 0; k < N; k += 4) {
      const KVec<4> x = load_k<4>(p + 4 * k);
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[k + j] = x.w[j];
    }
  } else {
    const KVec<N> x = load_k<N>(p);
#pragma unroll
    for (int j = 0; j < N; ++j) r.w[j] = x.w[j];
  }
  return r;
}

template <int D, int VDT, bool WIDE>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_few_kernel(AttendArgs a) {
  using G = FewGeo<D, VDT, WIDE>;
  constexpr int kWaves = 4;
  constexpr float kUp = VDT == kVF16 ? 6.f : 0.f, kSlack = 8.f;

  const DecodeArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wi = (int)blockIdx.x, wj = fdiv(wi, c.div_splits), split = wi - wj * c.num_splits;
  const int b = fdiv(wj, a.div_heads), hk = wj - b * a.kv_heads;
  const int rows = c.hq_per_kv * a.queries;
  const int n = seq_len_of(c, b), cnt = count_of(a, b), prefix = prefix_of(a, b, n);

  __shared__ __align__(16) float acc_s[kWaves][16][G::AS];
  __shared__ float m_s[kWaves][16], l_s[kWaves][16];

  // ---- this lane's row ----
  const int R = min(r16, rows - 1), qi = fdiv(R, c.div_hpk), qh = R - qi * c.hq_per_kv;
  const bool live = r16 < rows && qi < cnt;
  const RowView view = row_view(a, n, cnt, prefix, live ? qi : a.queries);
  const RowView v_lo = row_view(a, n, cnt, prefix, 0);
  const RowView v_hi = row_view(a, n, cnt, prefix, max(cnt - 1, 0));
  TileList list = tile_list(v_hi.head, v_lo.low, v_hi.pos);
  if (cnt == 0) list.total = 0;
  const int j0 = (int)((int64_t)split * list.total / c.num_splits);
  const int j1 = (int)((int64_t)(split + 1) * list.total / c.num_splits);
  bool wild = false;

  v4f acc[G::NA];
  float m = kLeastF, l = 0.f;
#pragma unroll
  for (int t = 0; t < G::NA; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};

  const float* sbase = c.k_scale + (int64_t)b * c.s_b + (int64_t)hk * c.s_h + g * G::CH;
  const float* zbase = c.k_zp + (int64_t)b * c.s_b + (int64_t)hk * c.s_h + g * G::CH;
  const uint8_t* kbase = c.k_pages + (int64_t)hk * c.k_head + g * (D / 8);
  const uint8_t* vbase = static_cast<const uint8_t*>(c.v_pages) +
                         ((int64_t)hk * c.v_head + r16 * G::NA) * G::VEB;
  const int32_t* table = c.page_table ? c.page_table + (int64_t)b * c.pt_b : nullptr;

  // Step u of this wave: 32 keys, two to a tile.
  const int mine = max(j1 - j0 - w + kWaves - 1, 0) / kWaves, steps = 2 * mine;
  auto key0_of = [&](int u) { return list.tile(j0 + w + kWaves * (u >> 1)) * kKeyTile + 32 * (u & 1); };

  Words<G::NK> kf[2];
  Words<G::VW> vf[2][4];
  // This lane's key of both halves of a step: page and row within it; the entries of the
  // table a step ahead.
  int entry[2], phys[2], prow[2];
  auto load_entries = [&](int u) __attribute__((always_inline)) {
    const int t0 = key0_of(min(u, steps - 1));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int lp = fdiv(min(t0 + 16 * h + r16, n - 1), c.div_rows);
      entry[h] = table ? table[lp] : lp;
    }
  };
  auto load_keys = [&](int u) __attribute__((always_inline)) {
    const int t0 = key0_of(min(u, steps - 1));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = min(t0 + 16 * h + r16, n - 1);
      prow[h] = t - fdiv(t, c.div_rows) * c.page_rows;
      phys[h] = min(max(entry[h], 0), c.num_pages - 1);
      kf[h] = load_stream<G::NK>(kbase + (int64_t)phys[h] * c.k_page + (int64_t)prow[h] * c.k_row);
    }
  };
  auto load_values = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pv = __shfl(phys[h], 4 * g + i, 16), rv = __shfl(prow[h], 4 * g + i, 16);
        vf[h][i] = load_stream<G::VW>(
            vbase + ((int64_t)pv * c.v_page + (int64_t)rv * c.v_row) * G::VEB);
      }
  };
  float sc[G::CH], zs[G::CH];
  int unit = 0;
  auto load_scales = [&](int u) __attribute__((always_inline)) {
    const int64_t at = (int64_t)fdiv(key0_of(min(u, steps - 1)), a.div_group) * c.s_g;
#pragma unroll
    for (int k = 0; k < G::CH; k += 4) {
      widen_values<kVF32>(ld16(sbase + at + k), sc + k);
      widen_values<kVF32>(ld16(zbase + at + k), zs + k);
    }
  };

  if (steps > 0) {
    load_entries(0);
    load_keys(0);
    load_values();
    load_scales(0);
    load_entries(1);

    // ---- the queries, B operands in units of a power of two for the row's largest ----
    v8h qop[G::TQ][G::NK];
    int q_unit;
    {
      const int64_t q0 = (int64_t)b * c.q_b + (int64_t)(hk * c.hq_per_kv + qh) * c.q_h +
                         (int64_t)qi * a.q_n + g * G::CH;
      float x[G::CH];
#pragma unroll
      for (int s = 0; s < G::CH; s += 8) {
        if (!a.q_vec) {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[s + k] = load_elem(c.q, q0 + s + k, c.q_dtype);
        } else if (c.q_dtype == kEF32) {
          const float* p = static_cast<const float*>(c.q) + q0 + s;
          widen_values<kVF32>(ld16(p), x + s);
          widen_values<kVF32>(ld16(p + 4), x + s + 4);
        } else {
          const U32x4 v = ld16(static_cast<const unsigned short*>(c.q) + q0 + s);
          if (c.q_dtype == kEF16) widen_values<kVF16>(v, x + s);
          else widen_values<kVBF16>(v, x + s);
        }
      }
      unsigned big = 0;
#pragma unroll
      for (int k = 0; k < G::CH; ++k) {
        x[k] = live ? x[k] : 0.f;
        big = max(big, f2u(x[k]) & 0x7FFFFFFFu);
      }
      big = over_quarters_umax(big);
      wild |= big >= 0x7F800000u;
      q_unit = exponent_of(min(big, 0x7F7FFFFFu)) - 7;
#pragma unroll
      for (int s = 0; s < G::NK; ++s) {
        v4u t[2];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float y0 = ldexpf(x[8 * s + 2 * k], -q_unit);
          const float y1 = ldexpf(x[8 * s + 2 * k + 1], -q_unit);
          t[0][k] = pack_f16(y0, y1);
          const v2h h = __builtin_bit_cast(v2h, (unsigned)t[0][k]);
          t[1][k] = pack_f16(y0 - (float)h[0], y1 - (float)h[1]);
        }
#pragma unroll
        for (int k = 0; k < G::TQ; ++k) qop[k][s] = __builtin_bit_cast(v8h, t[k]);
      }
    }
    const float slope = a.slopes ? a.slopes[hk * c.hq_per_kv + qh] * kLog2eF : 0.f;
    const float inv_cap = 1.f / a.cap, cap_scale = 2.f * kLog2eF / a.cap;

#pragma unroll 1
    for (int u = 0; u < steps; ++u) {
      const int t0 = key0_of(u);
      if ((u & 1) == 0) {
        unsigned big = 0;
#pragma unroll
        for (int k = 0; k < G::CH; ++k) {
          zs[k] *= sc[k];
          big = max(big, max(f2u(zs[k]) & 0x7FFFFFFFu,
                             f2u(__builtin_fmaf(15.f, sc[k], -zs[k])) & 0x7FFFFFFFu));
        }
        big = over_quarters_umax(big);
        wild |= big >= 0x7F800000u;
        unit = __builtin_amdgcn_readfirstlane(exponent_of(min(big, 0x7F7FFFFFu)) - 7);
#pragma unroll
        for (int k = 0; k < G::CH; ++k) {
          sc[k] = ldexpf(sc[k], -unit);
          zs[k] = ldexpf(zs[k], -unit);
        }
      }
      // ---- scores ----
      v4f sv[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) sv[h] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < G::NK; ++s)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned lo = kf[h].w[s] & 0x0F0F0F0Fu, hi = (kf[h].w[s] >> 4) & 0x0F0F0F0Fu;
          v4u t[2];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int ch = 8 * s + 2 * j;
            const float y0 = __builtin_fmaf((float)((lo >> (8 * j)) & 0xFFu), sc[ch], -zs[ch]);
            const float y1 =
                __builtin_fmaf((float)((hi >> (8 * j)) & 0xFFu), sc[ch + 1], -zs[ch + 1]);
            t[0][j] = pack_f16(y0, y1);
            const v2h x = __builtin_bit_cast(v2h, (unsigned)t[0][j]);
            t[1][j] = pack_f16(y0 - (float)x[0], y1 - (float)x[1]);
          }
          const v8h k0 = __builtin_bit_cast(v8h, t[0]), k1 = __builtin_bit_cast(v8h, t[1]);
          sv[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qop[0][s], sv[h], 0, 0, 0);
          if constexpr (WIDE)
            sv[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qop[1][s], sv[h], 0, 0, 0);
          sv[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qop[0][s], sv[h], 0, 0, 0);
        }
      if (u + 1 < steps) {
        load_keys(u + 1);
        load_entries(u + 2);
      }
      // (Of this tile the scales are used: the next one's are loaded under the rest.)
      const int key_unit = unit;
      if ((u & 1) && u + 1 < steps) load_scales(u + 1);

      v4u p[G::TP];
      const float f = ldexpf(1.f, min(max(q_unit + key_unit, -120), 120));
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = sv[i / 4][i % 4];
        if (a.cap > 0.f)
          x[i] = (WIDE ? soft_cap(y * f, a.cap, inv_cap) : quick_cap(y * f, a.cap, cap_scale)) *
                 kLog2eF;
        else
          x[i] = y * (f * kLog2eF);
        const int t = t0 + 16 * (i / 4) + 4 * g + i % 4;
        if (a.slopes) x[i] = __builtin_fmaf(-slope, fabsf((float)(view.pos - t)), x[i]);
        x[i] = sees(view, t) ? x[i] : -INFINITY;
      }
      float top = x[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) top = fmaxf(top, x[i]);
      top = over_quarters_max(top) - kUp;
      if (__builtin_amdgcn_ballot_w64(top > m + kSlack)) {
        const float mn = fmaxf(m, top);
        const float s = __builtin_amdgcn_exp2f(m - mn);
        m = mn;
        l *= s;
#pragma unroll
        for (int t = 0; t < G::NA; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) acc[t][i] *= s;
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float y0 = __builtin_amdgcn_exp2f(x[2 * k] - m);
        float y1 = __builtin_amdgcn_exp2f(x[2 * k + 1] - m);
        if constexpr (WIDE) l += y0 + y1;
        if constexpr (VDT == kVF16) {
          p[0][k] = pack_f16(y0, y1);
          const v2h h = __builtin_bit_cast(v2h, (unsigned)p[0][k]);
          if constexpr (WIDE) p[1][k] = pack_f16(y0 - (float)h[0], y1 - (float)h[1]);
          else l += (float)h[0] + (float)h[1];
        } else if constexpr (WIDE) {
#pragma unroll
          for (int q = 0; q < 3; ++q) {
            p[q][k] = pack_high(y0, y1);
            y0 = less_high(y0);
            y1 = less_high(y1);
          }
        } else {
          p[0][k] = pack_bf16(y0, y1);
          l += u2f(p[0][k] << 16) + u2f(p[0][k] & 0xFFFF0000u);
        }
      }
      // Values behind the sequence's end may be anything: zeros.
      if (t0 + 32 > n) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const unsigned keep = t0 + 16 * h + 4 * g + i < n ? ~0u : 0u;
#pragma unroll
            for (int k = 0; k < G::VW; ++k) vf[h][i].w[k] &= keep;
          }
      }
      // ---- values ----
#pragma unroll
      for (int t = 0; t < G::NA; ++t) {
        if constexpr (VDT == kVF32) {
          float x[2][4];
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[h][i] = u2f(vf[h][i].w[t]);
#pragma unroll
          for (int q = 0; q < G::TV; ++q) {
            const v4u av = {pack_high(x[0][0], x[0][1]), pack_high(x[0][2], x[0][3]),
                            pack_high(x[1][0], x[1][1]), pack_high(x[1][2], x[1][3])};
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int i = 0; i < 4; ++i) x[h][i] = less_high(x[h][i]);
#pragma unroll
            for (int z = 0; z < G::TP; ++z)
              if (z + q < 3) {
                acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(v8bf, av), __builtin_bit_cast(v8bf, p[z]), acc[t], 0, 0, 0);
              }
          }
        } else {
          const unsigned sel = t & 1 ? 0x07060302u : 0x05040100u;
          v4u av;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              av[2 * h + i] = __builtin_amdgcn_perm(vf[h][2 * i + 1].w[t / 2],
                                                    vf[h][2 * i].w[t / 2], sel);
#pragma unroll
          for (int z = 0; z < G::TP; ++z) {
            if constexpr (VDT == kVF16)
              acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                  __builtin_bit_cast(v8h, av), __builtin_bit_cast(v8h, p[z]), acc[t], 0, 0, 0);
            else
              acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                  __builtin_bit_cast(v8bf, av), __builtin_bit_cast(v8bf, p[z]), acc[t], 0, 0, 0);
          }
        }
      }
      if (u + 1 < steps) load_values();
    }
  }

  // ---- the waves meet ----
  l = over_quarters_sum(l);
  float probe = l;
#pragma unroll
  for (int t = 0; t < G::NA; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) probe = __builtin_fmaf(acc[t][i], 0.f, probe);
  const bool bad = wild || (live && !(probe >= 0.f && probe < INFINITY));
  if (g == 0) {
    m_s[w][r16] = m;
    l_s[w][r16] = l;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int t = 0; t < G::NA; t += 4)
      *reinterpret_cast<float4*>(&acc_s[w][r16][(4 * g + i) * G::NA + t]) =
          make_float4(acc[t][i], acc[t + 1][i], acc[t + 2][i], acc[t + 3][i]);
  __syncthreads();
  // Sixteen threads a row.
  const int row = tid >> 4, part = tid & 15;
  float weight[kWaves], total = 0.f, top = kLeastF;
#pragma unroll
  for (int k = 0; k < kWaves; ++k) top = fmaxf(top, m_s[k][row]);
#pragma unroll
  for (int k = 0; k < kWaves; ++k) {
    weight[k] = __builtin_amdgcn_exp2f(m_s[k][row] - top);
    total = __builtin_fmaf(weight[k], l_s[k][row], total);
  }
  const int oi = fdiv(min(row, rows - 1), c.div_hpk), oh = min(row, rows - 1) - oi * c.hq_per_kv;
  const bool seen = row < rows && sees_tiles(row_view(a, n, cnt, prefix, oi), list, j0, j1);
  if (__syncthreads_or(bad || (seen && !(total > 0.f)))) {
    const AttendArgs& a = late_attend_args();
    const DecodeArgs& c = a.c;
#pragma unroll 1
    for (int r = w; r < rows; r += kWaves) {
      const RowView v = row_view(a, n, cnt, prefix, r / c.hq_per_kv);
      const RowSums<D> x = plain_row<D, VDT>(a, b, hk, r, n, v, list, j0, j1);
      store_plain_row<D>(a, b, hk, r, split, x, x.m != kLeastF);
    }
    return;
  }
  if (row >= rows) return;
  const int64_t out_row = ((int64_t)b * c.num_q_heads + hk * c.hq_per_kv + oh) * a.queries + oi;
  const int64_t at = out_row * c.num_splits + split;
  const float inv = seen ? 1.f / total : 0.f;
#pragma unroll
  for (int k = 0; k < D / 64; ++k) {
    const int d = 64 * k + 4 * part;
    float y[4] = {};
#pragma unroll
    for (int x = 0; x < kWaves; ++x) {
      const float4 v = *reinterpret_cast<const float4*>(&acc_s[x][row][d]);
      y[0] = __builtin_fmaf(weight[x], v.x, y[0]);
      y[1] = __builtin_fmaf(weight[x], v.y, y[1]);
      y[2] = __builtin_fmaf(weight[x], v.z, y[2]);
      y[3] = __builtin_fmaf(weight[x], v.w, y[3]);
    }
    if (c.final_out) {
#pragma unroll
      for (int z = 0; z < 4; ++z)
        store_elem(c.out, out_row * D + d + z, c.out_dtype, seen ? y[z] * inv : 0.f);
    } else {
      *reinterpret_cast<float4*>(c.ws_acc + at * D + d) = make_float4(y[0], y[1], y[2], y[3]);
    }
  }
  if (!c.final_out && part == 0) {
    c.ws_ml[2 * at] = seen ? (double)top * 0.6931471805599453 : -INFINITY;
    c.ws_ml[2 * at + 1] = seen ? (double)total : 0.0;
  }
}

template <int D, int VDT>
hipError_t launch_few(const AttendArgs& a, int batch, hipStream_t st) {
  const dim3 grid((unsigned)(a.c.num_splits * batch * a.kv_heads));
  if (a.c.out_dtype == kEF32)
    hipLaunchKernelGGL((attend_few_kernel<D, VDT, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attend_few_kernel<D, VDT, false>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_attend_few(const AttendArgs& a, int D, int v_dtype, int batch, hipStream_t st) {
#define FDI4_FEW(DD, VV) \
  if (D == DD && v_dtype == VV) return launch_few<DD, VV>(a, batch, st);
  FDI4_FEW(64, kVF32) FDI4_FEW(64, kVF16) FDI4_FEW(64, kVBF16)
  FDI4_FEW(128, kVF32) FDI4_FEW(128, kVF16) FDI4_FEW(128, kVBF16)
  FDI4_FEW(256, kVF32) FDI4_FEW(256, kVF16) FDI4_FEW(256, kVBF16)
#undef FDI4_FEW
  return hipErrorInvalidValue;
}

}  // namespace fdi4
