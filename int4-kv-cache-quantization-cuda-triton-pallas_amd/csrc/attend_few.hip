// Attention of a few cached tokens (gfx950): up to 32 rows a kv-head, one token of a decode
// step above all. Memory bound: what counts is that the cache is read once, in long runs.
//
// A workgroup of four waves takes 16 rows of one kv-head over a range of 64-key tiles,
// which go to the waves in pairs. A wave loads 32 keys straight to registers; the next keys
// are loaded as soon as these are multiplied, the next values as soon as these are. Waves
// meet at the end, in LDS, and splits in the merge kernel.
//
//   terms: q . k_t = sum_d v_d (nib_td - zp_d), v = q*s. Per scale group and row, v is made
//      into two float16 terms (22 bits, in units of a power of two for the largest), once for
//      the group's keys, and multiplied by the nibbles as they are stored: a nibble at bits 6
//      to 9 of a float16 is the number nib * 2^-18. The constant sum_d v_d zp_d, in
//      float32, goes in with the exponent's FMA. Dequantized keys, in two terms as well, took
//      900 instructions of the vector units for 32 keys in place of 350, and 155 us in
//      place of 113 for 16 sequences of 16384 bfloat16 tokens and 8 kv-heads.
//   scores: v_mfma_f32_16x16x32_f16 of 16 keys (A) and 16 rows (B): lane (g, r) loads the
//      channels g * D/4 .. of key r and of row r, eight of them a product.
//   values: lane (g, r) holds the scores of row r with keys 4g .. 4g + 3 of both 16-key
//      halves, which is the B operand of a product of 32 keys, and loads the channels r *
//      D/16 .. of the same keys: byte permutes pair them.
//
// 16 sequences of 16384 tokens, 8 kv-heads, 32 q-heads, 128 bfloat16 channels, capped: 113 us,
// 6.1 TB/s, 109 in the kernel and the rest in the merge; the vector units are busy for 39 %.
//
// Probabilities: two terms of the values' type for 16-bit outputs (16 bits of them with bfloat16
// and float32 values, the latter in two bfloat16 terms themselves; 22 with float16 ones). One
// was 0 to 4 % faster (149.9 us in place of 151.8 for 24 sequences of 6000 float16 tokens, 16
// heads of 128) and rounded a quarter of the outputs to a neighbour, where two do so with 0.5
// %. WIDE, for what attend_chunk.hip says: two float16 or three bfloat16 terms, float32 values
// in three. PAGED: pages hold whole runs of 16 rows, so that a run's address is the same for
// all lanes.

#include "attend_common.hpp"

namespace fdi4 {

typedef float v4f __attribute__((ext_vector_type(4)));

template <int D, int VDT, bool WIDE>
struct FewGeo {
  static constexpr int TV = VDT == kVF32 ? (WIDE ? 3 : 2) : 1;
  static constexpr int TP = VDT == kVF16 || !WIDE ? 2 : 3;
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

template <int D, int VDT, bool WIDE, bool PAGED>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void attend_few_kernel(AttendArgs a) {
  using G = FewGeo<D, VDT, WIDE>;
  constexpr int kWaves = 4;
  constexpr float kUp = VDT == kVF16 ? 6.f : 0.f, kSlack = 8.f;

  const DecodeArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, r16 = lane & 15, g = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  // The groups of 16 rows of one (sequence, kv-head, split) run on one XCD.
  const int L = a.tiles > 1 ? (int)xcd_run_item(blockIdx.x, gridDim.x, (unsigned)a.tiles)
                            : (int)blockIdx.x;
  const int wi = a.tiles > 1 ? L / a.tiles : L, row0 = 16 * (L - wi * a.tiles);
  const int wj = fdiv(wi, c.div_splits), split = wi - wj * c.num_splits;
  const int b = fdiv(wj, a.div_heads), hk = wj - b * a.kv_heads;
  const int all_rows = c.hq_per_kv * a.queries, rows = min(all_rows - row0, 16);
  const int n = seq_len_of(c, b), cnt = count_of(a, b), prefix = prefix_of(a, b, n);

  __shared__ __align__(16) float acc_s[kWaves][16][G::AS];
  __shared__ float m_s[kWaves][16], l_s[kWaves][16];
  __shared__ __align__(16) float q_s[16][G::AS];       // the rows' queries
  __shared__ __align__(16) float sz_s[kWaves][2][D];   // a wave's scales and zero-points

  // ---- this lane's row ----
  const int R = row0 + min(r16, rows - 1), qi = fdiv(R, c.div_hpk), qh = R - qi * c.hq_per_kv;
  const bool live = r16 < rows && qi < cnt;
  const RowView view = row_view(a, n, cnt, prefix, live ? qi : a.queries);
  const int i_lo = fdiv(row0, c.div_hpk), i_hi = min(fdiv(row0 + rows - 1, c.div_hpk), cnt - 1);
  const RowView v_lo = row_view(a, n, cnt, prefix, i_lo);
  const RowView v_hi = row_view(a, n, cnt, prefix, max(i_hi, 0));
  TileList list = tile_list(v_hi.head, v_lo.low, v_hi.pos);
  if (i_hi < i_lo) list.total = 0;
  // Pairs of tiles, which mostly lie in one scale group, to splits and waves; single ones
  // where a wave would be without.
  const int pairs = (list.total + 1) >> 1;
  const int j0 = 2 * (int)((int64_t)split * pairs / c.num_splits);
  const int j1 = min(2 * (int)((int64_t)(split + 1) * pairs / c.num_splits), list.total);
  const int item = j1 - j0 > kWaves ? 2 : 1;
  bool wild = false;

  v4f acc[G::NA];
  float m = kLeastF, l = 0.f;
#pragma unroll
  for (int t = 0; t < G::NA; ++t) acc[t] = v4f{0.f, 0.f, 0.f, 0.f};

  const float* sbase = c.k_scale + (int64_t)b * c.s_b + (int64_t)hk * c.s_h;
  const float* zbase = c.k_zp + (int64_t)b * c.s_b + (int64_t)hk * c.s_h;
  const uint8_t* kbase = c.k_pages + (int64_t)hk * c.k_head;
  const uint8_t* vbase = static_cast<const uint8_t*>(c.v_pages) + (int64_t)hk * c.v_head * G::VEB;
  const int k_lane = g * (D / 8), v_lane = r16 * G::NA * G::VEB;
  const int32_t* table = c.page_table ? c.page_table + (int64_t)b * c.pt_b : nullptr;

  // Step u of this wave: 32 keys, two to a tile.
  const int rounds = max(j1 - j0 - w * item + kWaves * item - 1, 0) / (kWaves * item);
  const int last = j0 + (w + kWaves * (rounds - 1)) * item;   // its last item's first tile
  const int steps =
      rounds > 0 ? 2 * (item * (rounds - 1) + min(item, j1 - last)) : 0;
  auto key0_of = [&](int u) {
    const int k = u >> 1, round = item == 2 ? k >> 1 : k;
    const int j = j0 + (w + kWaves * round) * item + (item == 2 ? k & 1 : 0);
    return list.tile(j) * kKeyTile + 32 * (u & 1);
  };

  Words<G::NK> kf[2];
  Words<G::VW> vf[2][4];
  // PAGED: a run's place, the same for all lanes. Otherwise this lane's key of both halves
  // of a step, its page and row; the entries of the table a step ahead.
  int entry[2], phys[2], prow[2];
  auto key_at = [&](int u, int h) {
    const int t = key0_of(min(u, steps - 1)) + 16 * h;
    return PAGED ? min(t, (n - 1) & ~15) : min(t + r16, n - 1);
  };
  auto load_entries = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int lp = fdiv(key_at(u, h), c.div_rows);
      if constexpr (PAGED) entry[h] = table ? ld_ro(table, lp) : lp;
      else entry[h] = table ? table[lp] : lp;
    }
  };
  auto load_keys = [&](int u) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int t = key_at(u, h);
      prow[h] = t - fdiv(t, c.div_rows) * c.page_rows;
      phys[h] = min(max(entry[h], 0), c.num_pages - 1);
      const uint8_t* at = kbase + ((int64_t)phys[h] * c.k_page + (int64_t)prow[h] * c.k_row);
      kf[h] = load_stream<G::NK>(at + (PAGED ? k_lane + r16 * (int)c.k_row : k_lane));
    }
  };
  auto load_values = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint8_t* at =
          vbase + ((int64_t)phys[h] * c.v_page + (int64_t)prow[h] * c.v_row) * G::VEB;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (PAGED) {
          vf[h][i] = load_stream<G::VW>(at + (v_lane + (4 * g + i) * (int)(c.v_row * G::VEB)));
        } else {
          const int pv = __shfl(phys[h], 4 * g + i, 16), rv = __shfl(prow[h], 4 * g + i, 16);
          vf[h][i] = load_stream<G::VW>(
              vbase + (((int64_t)pv * c.v_page + (int64_t)rv * c.v_row) * G::VEB + v_lane));
        }
      }
    }
  };
  // Scales and zero-points of a group, D / 64 channels a lane (they go through LDS).
  constexpr int SL = D / 64;
  float sc[SL], zp[SL];
  auto group_at = [&](int u) { return fdiv(key0_of(min(u, steps - 1)), a.div_group); };
  auto load_scales = [&](int group) __attribute__((always_inline)) {
    const int64_t at = (int64_t)group * c.s_g + SL * lane;
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      sc[k] = sbase[at + k];
      zp[k] = zbase[at + k];
    }
  };

  if (steps > 0) {
    load_entries(0);
    load_keys(0);
    load_values();
    load_scales(group_at(0));
    load_entries(1);
  }

  // ---- the queries to LDS: sixteen threads a row; zeros for rows that are not there ----
  {
    const int row = tid >> 4, rr = row0 + min(row, rows - 1), i = fdiv(rr, c.div_hpk);
    const int d0 = (tid & 15) * G::NA;
    const int64_t q0 = (int64_t)b * c.q_b +
                       (int64_t)(hk * c.hq_per_kv + rr - i * c.hq_per_kv) * c.q_h +
                       (int64_t)i * a.q_n + d0;
    const bool there = row < rows && i < cnt;
#pragma unroll
    for (int k = 0; k < G::NA; k += 4) {
      float x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        x[j] = there ? load_elem(c.q, q0 + k + j, c.q_dtype) : 0.f;
        wild |= (f2u(x[j]) & 0x7FFFFFFFu) >= 0x7F800000u;
      }
      *reinterpret_cast<float4*>(&q_s[row][d0 + k]) = make_float4(x[0], x[1], x[2], x[3]);
    }
  }
  __syncthreads();

  if (steps > 0) {

    // Terms of a group: eight channels a product, in the order in which a shift brings
    // nibbles to bits 6 to 9 and 22 to 25 of a word. A score is S * unit - shift.
    v8h term[2][G::NK];
    float unit = 0.f, shift = 0.f;
    auto make_terms = [&]() __attribute__((always_inline)) {
#pragma unroll
      for (int k = 0; k < SL; ++k) {
        sz_s[w][0][SL * lane + k] = sc[k];
        sz_s[w][1][SL * lane + k] = zp[k];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      unsigned big = 0;
      float sum[4] = {0.f, 0.f, 0.f, 0.f}, v[G::CH];
#pragma unroll
      for (int k = 0; k < G::CH; k += 4) {
        const float4 qx = *reinterpret_cast<const float4*>(&q_s[r16][g * G::CH + k]);
        const float4 sx = *reinterpret_cast<const float4*>(&sz_s[w][0][g * G::CH + k]);
        const float4 zx = *reinterpret_cast<const float4*>(&sz_s[w][1][g * G::CH + k]);
        const float q4[4] = {qx.x, qx.y, qx.z, qx.w}, s4[4] = {sx.x, sx.y, sx.z, sx.w};
        const float z4[4] = {zx.x, zx.y, zx.z, zx.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[k + j] = q4[j] * s4[j];
          big = max(big, f2u(v[k + j]) & 0x7FFFFFFFu);
          sum[j] = __builtin_fmaf(v[k + j], z4[j], sum[j]);
        }
      }
      big = over_quarters_umax(big);
      shift = over_quarters_sum((sum[0] + sum[1]) + (sum[2] + sum[3]));
      // (Also from 2^117 on, where the unit would pass 2^120: row by row.)
      wild |= big >= (117u + 127u) << 23 || (f2u(shift) & 0x7FFFFFFFu) >= 0x7F800000u;
      const int e = exponent_of(min(big, 0x7F7FFFFFu)) - 14;
      // (Scores below 2^-100 are as good as 0, and their unit may be larger than it is.)
      unit = ldexpf(1.f, min(max(e + 18, -120), 120));
#pragma unroll
      for (int s = 0; s < G::NK; ++s) {
        v4u t[2];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float y0 = ldexpf(v[8 * s + k], -e), y1 = ldexpf(v[8 * s + k + 4], -e);
          t[0][k] = pack_f16(y0, y1);
          const v2h h = __builtin_bit_cast(v2h, (unsigned)t[0][k]);
          t[1][k] = pack_f16(y0 - (float)h[0], y1 - (float)h[1]);
        }
        term[0][s] = __builtin_bit_cast(v8h, t[0]);
        term[1][s] = __builtin_bit_cast(v8h, t[1]);
      }
    };
    int group = -1, held = group_at(0);   // of the terms; of sc and zp
    const float slope = a.slopes ? a.slopes[hk * c.hq_per_kv + qh] * kLog2eF : 0.f;
    const float inv_cap = 1.f / a.cap, cap_scale = 2.f * kLog2eF / a.cap;

#pragma unroll 1
    for (int u = 0; u < steps; ++u) {
      const int t0 = key0_of(u);
      if ((u & 1) == 0) {
        const int now = group_at(u);
        if (now != group) {
          make_terms();
          group = now;
        }
        // (The next group's scales come under this one's products: those of the next tile,
        // or of the one behind it, where the next one is in this group.)
        int v = u + 2;
        if (item == 2 && v < steps && group_at(v) == now) v += 2;
        const int next = v < steps ? group_at(v) : now;
        if (next != now && next != held) {
          load_scales(next);
          held = next;
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
          const unsigned x = kf[h].w[s];
          const v4u nib = {x << 6 & 0x03C003C0u, x << 2 & 0x03C003C0u, x >> 2 & 0x03C003C0u,
                           x >> 6 & 0x03C003C0u};
          const v8h k0 = __builtin_bit_cast(v8h, nib);
          sv[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, term[1][s], sv[h], 0, 0, 0);
          sv[h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, term[0][s], sv[h], 0, 0, 0);
        }
      if (u + 1 < steps) {
        load_keys(u + 1);
        load_entries(u + 2);
      }

      v4u p[G::TP];
      // Scores in units of log2.
      float x[8];
      if (a.cap > 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float y = __builtin_fmaf(sv[i / 4][i % 4], unit, -shift);
          x[i] = (WIDE ? soft_cap(y, a.cap, inv_cap) : quick_cap(y, a.cap, cap_scale)) * kLog2eF;
        }
      } else {
        const float f2 = unit * kLog2eF, s2 = shift * kLog2eF;
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_fmaf(sv[i / 4][i % 4], f2, -s2);
      }
      // (Element i is key 16 (i / 4) + 4 g + i % 4.)
      if (a.slopes) {
        const float d0 = (float)(view.pos - t0 - 4 * g);
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = __builtin_fmaf(-slope, fabsf(d0 - (float)(16 * (i / 4) + i % 4)), x[i]);
      }
      if (!(t0 + 32 <= v_lo.head || (t0 + 31 <= v_lo.pos && t0 >= v_hi.low))) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          x[i] = sees(view, t0 + 16 * (i / 4) + 4 * g + i % 4) ? x[i] : -INFINITY;
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
        l += y0 + y1;
        if constexpr (VDT == kVF16) {
          p[0][k] = pack_f16(y0, y1);
          const v2h h = __builtin_bit_cast(v2h, (unsigned)p[0][k]);
          p[1][k] = pack_f16(y0 - (float)h[0], y1 - (float)h[1]);
        } else {
#pragma unroll
          for (int q = 0; q + 1 < G::TP; ++q) {
            p[q][k] = pack_high(y0, y1);
            y0 = less_high(y0);
            y1 = less_high(y1);
          }
          p[G::TP - 1][k] = WIDE ? pack_high(y0, y1) : pack_bf16(y0, y1);
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
  const int oR = row0 + min(row, rows - 1), oi = fdiv(oR, c.div_hpk), oh = oR - oi * c.hq_per_kv;
  const bool seen = row < rows && sees_tiles(row_view(a, n, cnt, prefix, oi), list, j0, j1);
  if (__syncthreads_or(bad || (seen && !(total > 0.f)))) {
    const AttendArgs& a = late_attend_args();
    const DecodeArgs& c = a.c;
#pragma unroll 1
    for (int r = row0 + w; r < row0 + rows; r += kWaves) {
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

template <int D, int VDT, bool WIDE>
hipError_t launch_few(AttendArgs a, int batch, hipStream_t st) {
  a.tiles = (a.c.hq_per_kv * a.queries + 15) / 16;
  const int64_t wgs = (int64_t)a.tiles * a.c.num_splits * batch * a.kv_heads;
  if (!grid_fits(wgs, 256)) return hipErrorInvalidValue;
  const dim3 grid((unsigned)wgs);
  if (a.c.page_rows % 16 == 0)
    hipLaunchKernelGGL((attend_few_kernel<D, VDT, WIDE, true>), grid, dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((attend_few_kernel<D, VDT, WIDE, false>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_attend_few(const AttendArgs& a, int D, int v_dtype, int batch, hipStream_t st) {
#define FDI4_FEW(DD, VV) \
  if (D == DD && v_dtype == VV)                                   \
    return attend_wide(a.c.out_dtype, v_dtype, a.cap) ? launch_few<DD, VV, true>(a, batch, st) \
                                               : launch_few<DD, VV, false>(a, batch, st);
  FDI4_FEW(64, kVF32) FDI4_FEW(64, kVF16) FDI4_FEW(64, kVBF16)
  FDI4_FEW(128, kVF32) FDI4_FEW(128, kVF16) FDI4_FEW(128, kVBF16)
  FDI4_FEW(256, kVF32) FDI4_FEW(256, kVF16) FDI4_FEW(256, kVBF16)
#undef FDI4_FEW
  return hipErrorInvalidValue;
}

}  // namespace fdi4
