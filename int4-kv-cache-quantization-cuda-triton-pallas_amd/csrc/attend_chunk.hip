// Attention of a chunk of cached tokens on the matrix cores (gfx950): many rows a kv-head.
//
// Row R of a kv-head is query R / G of q-head R % G of its group (G q-heads share it).
// A workgroup takes 32 rows a wave, and keys in tiles that the whole workgroup stages into
// LDS: keys dequantized once for all rows (k = nib*s - zp*s as float16 in units of a power
// of two for the scale group's largest), values as they are. The next tile is loaded to
// registers while the present one is computed, two LDS buffers, one barrier a tile. Half of
// the waves stage the next tile before they compute, half behind it, so that the two waves
// of a SIMD are in different parts of a step (1295 us, 1203 to 1266 so on several cards, for 8
// sequences, 8 kv-heads and 32 q-heads of 128 bfloat16 channels, 1024 queries over 8192 tokens;
// 813 to 856 TFLOP/s).
//
//   scores: S^T = K Q^T by v_mfma_f32_32x32x16_f16, keys as A from LDS, queries as B in
//      registers for the whole call (in units of a power of two for the row's largest):
//      a lane holds 16 scores of 32 keys of one row, lane ^ 32 the others.
//   softmax: in units of log2, the shift of a row moves only when a score passes it by
//      kSlack, so the accumulators are rescaled rarely.
//   values: O^T = V^T P^T. The scores' lanes are already those of the B operand, in a
//      fixed order of keys, and the transposing LDS reads (ds_read_b64_tr_b16) bring V^T
//      in the same order: probabilities never leave their registers.
//
// Terms. bfloat16 outputs: one float16 term of keys (2^-11 of a product at most; a float16
// holds 3 bits more than the bfloat16 of a dequantizing cache) and of queries (16-bit ones
// fit exactly), one term of probabilities in the values' type (their sum takes them
// rounded), float32 values in two bfloat16 terms: 0.0021 in the 2-norm in place of the 0.0017
// of the output's own rounding. float16 values: two terms of keys (with one 5.1e-4, with two
// 2.3e-4, of which 2.1e-4 are the output's). Two terms of probabilities would leave the output's
// rounding alone and take 1575 us in place of 1236 at the size above, 1953 in place of 1641 with
// float16 values. WIDE, for float32 outputs, for float16 ones
// of other values, and under caps beyond 512: two terms of both, without the product of the
// second ones, probabilities in two float16 or three bfloat16 terms, float32 values in three.
//
// What bounds it: at that size the matrix cores are busy for 39 % of the time, the vector
// units for 59 and LDS for 25 (no bank conflicts): the two mostly work in turns. A step has all
// its scores before its weights, and the registers of accumulators, queries and scores leave two
// waves a SIMD (one with 256 channels).
//
// A workgroup that ends with a NaN, or meets a query or a scale that is not finite, takes its
// rows one by one: a value that a row does not see would otherwise reach it as 0 * inf. (One NaN
// among the values above: 151 ms.)

#include "attend_common.hpp"

namespace fdi4 {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

template <int D, int VDT, bool WIDE>
struct ChunkGeo {
  static constexpr int WAVES = WIDE || D == 256 ? 4 : 8;
  static constexpr int NT = WAVES * 64;
  static constexpr int M = WAVES * 32;                 // rows of a workgroup
  // Keys of a staged tile. Of float32 outputs 64 keys pay at 128 channels (8 sequences, 512
  // queries over 2048 tokens, bfloat16 values: 475 us, 547 with 32), while at 64 channels 32
  // leave registers for a second workgroup on a CU (229 us, 305 with 64); at 256 the buffers
  // and registers hold 64 with bfloat16 values and 16-bit outputs only.
  static constexpr int KT = WIDE ? (D == 128 ? 64 : 32) : (D == 256 && VDT != kVBF16 ? 32 : 64);
  static constexpr int NBUF = WIDE ? 1 : 2;
  static constexpr int TK = WIDE || VDT == kVF16 ? 2 : 1;   // terms of keys
  static constexpr int TQ = WIDE ? 2 : 1;              // and of queries
  static constexpr int TV = VDT == kVF32 ? (WIDE ? 3 : 2) : 1;
  static constexpr int TP = !WIDE ? 1 : VDT == kVF16 ? 2 : 3;
  static constexpr int VEB = VDT == kVF32 ? 4 : 2;
  static constexpr int PKB = D == 256 ? 8 : 4;         // packed key bytes of a thread's row
  static constexpr int CPT = 2 * PKB;                  // its channels
  static constexpr int SEG = D / CPT;                  // threads a row
  static constexpr int RPT = KT * SEG / NT;            // rows a thread
  static constexpr int VW = CPT * VEB / 4;             // words of its part of a value row
  // LDS rows. Keys 16 bytes longer than a power of two: lanes of consecutive keys read 16
  // bytes each. Values 64: the eight rows of a transposing read lie on other banks.
  static constexpr int KS = D * 2 + 16;
  static constexpr int VS = D * 2 + 64;
  static constexpr int kKeys = TK * KT * KS;
  static constexpr int kBuf = kKeys + TV * KT * VS;
  static constexpr int NA = D / 32;                    // 32-channel output tiles
  static constexpr int NK = D / 16;                    // channel steps of a score
  static_assert(KT * SEG % NT == 0 && SEG <= 16, "threads");
};

// The largest of three (the instruction quiets operands itself).
__device__ __forceinline__ float max3(float x, float y, float z) {
  float r;
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "v"(y), "v"(z));
  return r;
}

__device__ __forceinline__ float over_halves_max(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return fmaxf(u2f(r[0]), u2f(r[1]));
}

__device__ __forceinline__ float over_halves_sum(float x) {
  auto r = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return u2f(r[0]) + u2f(r[1]);
}

template <int D, int VDT, bool WIDE>
__global__ __launch_bounds__((ChunkGeo<D, VDT, WIDE>::NT), (ChunkGeo<D, VDT, WIDE>::WAVES / 4))
void attend_chunk_kernel(AttendArgs a) {
  using G = ChunkGeo<D, VDT, WIDE>;
  constexpr int M = G::M, KT = G::KT, NS = KT / 32;
  // Probabilities are 2^kUp at most when the shift moves, and 2^(kUp + kSlack) at any time:
  // float16 terms (up to 2^16) are normal down to 2^-20 of the largest.
  constexpr float kUp = VDT == kVF16 ? 6.f : 0.f, kSlack = 8.f;
  constexpr float kLn2 = 0.6931471805599453f;

  const DecodeArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63, r32 = lane & 31, half = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

  // The tiles of one (sequence, kv-head, split) run on one XCD, the longest first.
  const int L = (int)xcd_run_item(blockIdx.x, gridDim.x, (unsigned)a.tiles);
  const int wi = L / a.tiles, tile = a.tiles - 1 - (L - wi * a.tiles);
  const int wj = fdiv(wi, c.div_splits), split = wi - wj * c.num_splits;
  const int b = fdiv(wj, a.div_heads), hk = wj - b * a.kv_heads;
  const int rows = c.hq_per_kv * a.queries;
  const int row0 = tile * M, row1 = min(row0 + M, rows);
  const int n = seq_len_of(c, b), cnt = count_of(a, b), prefix = prefix_of(a, b, n);

  __shared__ __align__(16) uint8_t smem[G::NBUF * G::kBuf];
  __shared__ int unit_s[2];                            // exponent of a buffer's keys
  __shared__ int wild_s;

  // This lane's row.
  const int R = row0 + 32 * w + r32;
  const int qi = fdiv(min(R, rows - 1), c.div_hpk), qh = min(R, rows - 1) - qi * c.hq_per_kv;
  const bool live = R < rows && qi < cnt;
  const RowView view = row_view(a, n, cnt, prefix, live ? qi : a.queries);
  const int64_t out_row =
      ((int64_t)b * c.num_q_heads + hk * c.hq_per_kv + qh) * a.queries + qi;

  // What the workgroup sees, and this wave: limits grow with the query.
  const int i_lo = fdiv(row0, c.div_hpk), i_hi = min(fdiv(row1 - 1, c.div_hpk), cnt - 1);
  const RowView v_lo = row_view(a, n, cnt, prefix, i_lo);
  const RowView v_hi = row_view(a, n, cnt, prefix, max(i_hi, 0));
  TileList list = tile_list(v_hi.head, v_lo.low, v_hi.pos);
  if (i_hi < i_lo) list.total = 0;
  const int j0 = (int)((int64_t)split * list.total / c.num_splits);
  const int j1 = (int)((int64_t)(split + 1) * list.total / c.num_splits);
  const int wr0 = min(row0 + 32 * w, rows - 1), wr1 = min(row0 + 32 * w + 31, rows - 1);
  const int wi_lo = fdiv(wr0, c.div_hpk), wi_hi = min(fdiv(wr1, c.div_hpk), cnt - 1);
  const bool idle = row0 + 32 * w >= rows || wi_lo >= cnt;
  const RowView w_lo = row_view(a, n, cnt, prefix, min(wi_lo, cnt - 1));
  const RowView w_hi = row_view(a, n, cnt, prefix, max(wi_hi, 0));

  if (tid == 0) wild_s = 0;
  __syncthreads();

  // ---- the queries: B operands, channels 16 s + 8 half .. of the row ----
  v8h qop[G::TQ][G::NK];
  int q_unit = 0;
  if (j0 < j1) {
    const int64_t q0 = (int64_t)b * c.q_b + (int64_t)(hk * c.hq_per_kv + qh) * c.q_h +
                       (int64_t)qi * a.q_n + 8 * half;
    unsigned big = 0;
#pragma unroll
    for (int pass = 0; pass < 2; ++pass) {
      if (pass == 1) {
        auto x = __builtin_amdgcn_permlane32_swap(big, big, false, false);
        big = max((unsigned)x[0], (unsigned)x[1]);
        if (big >= 0x7F800000u) wild_s = 1;
        q_unit = exponent_of(min(big, 0x7F7FFFFFu)) - 7;
      }
#pragma unroll
      for (int s = 0; s < G::NK; ++s) {
        float x[8];
        if (!a.q_vec) {
#pragma unroll
          for (int k = 0; k < 8; ++k) x[k] = load_elem(c.q, q0 + 16 * s + k, c.q_dtype);
        } else if (c.q_dtype == kEF32) {
          const float* p = static_cast<const float*>(c.q) + q0 + 16 * s;
          widen_values<kVF32>(ld16(p), x);
          widen_values<kVF32>(ld16(p + 4), x + 4);
        } else {
          const U32x4 v = ld16(static_cast<const unsigned short*>(c.q) + q0 + 16 * s);
          if (c.q_dtype == kEF16) widen_values<kVF16>(v, x);
          else widen_values<kVBF16>(v, x);
        }
        if (pass == 0) {
#pragma unroll
          for (int k = 0; k < 8; ++k) big = live ? max(big, f2u(x[k]) & 0x7FFFFFFFu) : 0u;
        } else {
          v4u t[2];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float y0 = live ? ldexpf(x[2 * k], -q_unit) : 0.f;
            const float y1 = live ? ldexpf(x[2 * k + 1], -q_unit) : 0.f;
            t[0][k] = pack_f16(y0, y1);
            if constexpr (WIDE) {
              const v2h h = __builtin_bit_cast(v2h, (unsigned)t[0][k]);
              t[1][k] = pack_f16(y0 - (float)h[0], y1 - (float)h[1]);
            }
          }
#pragma unroll
          for (int k = 0; k < G::TQ; ++k) qop[k][s] = __builtin_bit_cast(v8h, t[k]);
        }
      }
    }
  }

  // ---- staging: this thread's rows of a tile and its channels ----
  const int seg = tid % G::SEG, srow = tid / G::SEG;
  constexpr int RSTEP = G::NT / G::SEG;
  const float* sbase = c.k_scale + (int64_t)b * c.s_b + (int64_t)hk * c.s_h + seg * G::CPT;
  const float* zbase = c.k_zp + (int64_t)b * c.s_b + (int64_t)hk * c.s_h + seg * G::CPT;
  const uint8_t* kbase = c.k_pages + (int64_t)hk * c.k_head + seg * G::PKB;
  const uint8_t* vbase = static_cast<const uint8_t*>(c.v_pages) +
                         ((int64_t)hk * c.v_head + seg * G::CPT) * G::VEB;
  const int32_t* table = c.page_table ? c.page_table + (int64_t)b * c.pt_b : nullptr;

  // Steps of KT keys: tile j has kKeyTile / KT of them.
  constexpr int PER = kKeyTile / KT;
  const int s0 = j0 * PER, s1 = j1 * PER;
  auto key0_of = [&](int s) { return list.tile(s / PER) * kKeyTile + s % PER * KT; };

  int entry[G::RPT];
  unsigned kw[G::RPT][G::PKB / 4];
  unsigned vw[G::RPT][G::VW];
  float sc[G::CPT], zs[G::CPT];
  int unit = 0, group = -1;
  auto load_entries = [&](int s) __attribute__((always_inline)) {
    const int t0 = key0_of(min(s, s1 - 1));
#pragma unroll
    for (int i = 0; i < G::RPT; ++i) {
      const int lp = fdiv(min(t0 + srow + i * RSTEP, n - 1), c.div_rows);
      entry[i] = table ? table[lp] : lp;
    }
  };
  auto load_tile = [&](int s) __attribute__((always_inline)) {
    const int t0 = key0_of(min(s, s1 - 1));
#pragma unroll
    for (int i = 0; i < G::RPT; ++i) {
      const int t = min(t0 + srow + i * RSTEP, n - 1);
      const int tr = t - fdiv(t, c.div_rows) * c.page_rows;
      const int64_t phys = min(max(entry[i], 0), c.num_pages - 1);
      const uint8_t* kp = kbase + phys * c.k_page + (int64_t)tr * c.k_row;
      const uint8_t* vp = vbase + (phys * c.v_page + (int64_t)tr * c.v_row) * G::VEB;
#pragma unroll
      for (int k = 0; k < G::PKB / 4; ++k) kw[i][k] = reinterpret_cast<const unsigned*>(kp)[k];
#pragma unroll
      for (int k = 0; k < G::VW / 4; ++k) {
        const U32x4 x = ld16(vp + 16 * k);
        vw[i][4 * k] = x.x;
        vw[i][4 * k + 1] = x.y;
        vw[i][4 * k + 2] = x.z;
        vw[i][4 * k + 3] = x.w;
      }
    }
    const int g = fdiv(t0, a.div_group);
    if (g != group) {
      group = g;
      const float* sp = sbase + (int64_t)g * c.s_g;
      const float* zp = zbase + (int64_t)g * c.s_g;
#pragma unroll
      for (int k = 0; k < G::CPT; k += 4) {
        widen_values<kVF32>(ld16(sp + k), sc + k);
        widen_values<kVF32>(ld16(zp + k), zs + k);
      }
      unit = 1 << 20;                                  // not in units yet
    }
  };
  auto write_tile = [&](int s, int buf) __attribute__((always_inline)) {
    if (unit == 1 << 20) {
      // Units of a power of two: the largest key that the group can hold is below 2^8.
      unsigned big = 0;
#pragma unroll
      for (int k = 0; k < G::CPT; ++k) {
        zs[k] *= sc[k];
        big = max(big, max(f2u(zs[k]) & 0x7FFFFFFFu,
                           f2u(__builtin_fmaf(15.f, sc[k], -zs[k])) & 0x7FFFFFFFu));
      }
      big = max(big, xchg_u32<1>(big));
      big = max(big, xchg_u32<2>(big));
      big = max(big, xchg_u32<4>(big));
      if constexpr (G::SEG > 8) big = max(big, xchg_u32<8>(big));
      if (big >= 0x7F800000u) wild_s = 1;
      unit = exponent_of(min(big, 0x7F7FFFFFu)) - 7;
#pragma unroll
      for (int k = 0; k < G::CPT; ++k) {
        sc[k] = ldexpf(sc[k], -unit);
        zs[k] = ldexpf(zs[k], -unit);
      }
    }
    uint8_t* base = smem + buf * G::kBuf;
    const int t0 = key0_of(s);
    if (tid == 0) unit_s[buf] = unit;
#pragma unroll
    for (int i = 0; i < G::RPT; ++i) {
      const int row = srow + i * RSTEP;
#pragma unroll
      for (int k = 0; k < G::PKB / 4; ++k) {
        const unsigned lo = kw[i][k] & 0x0F0F0F0Fu, hi = (kw[i][k] >> 4) & 0x0F0F0F0Fu;
        v4u t[2];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int ch = 8 * k + 2 * j;
          const float y0 = __builtin_fmaf((float)((lo >> (8 * j)) & 0xFFu), sc[ch], -zs[ch]);
          const float y1 =
              __builtin_fmaf((float)((hi >> (8 * j)) & 0xFFu), sc[ch + 1], -zs[ch + 1]);
          t[0][j] = pack_f16(y0, y1);
          if constexpr (G::TK == 2) {
            const v2h h = __builtin_bit_cast(v2h, (unsigned)t[0][j]);
            t[1][j] = pack_f16(y0 - (float)h[0], y1 - (float)h[1]);
          }
        }
#pragma unroll
        for (int x = 0; x < G::TK; ++x)
          *reinterpret_cast<v4u*>(base + (x * KT + row) * G::KS + seg * G::CPT * 2 + 16 * k) =
              t[x];
      }
      // Values behind the sequence's end may be anything: zeros.
      const unsigned keep = t0 + row < n ? ~0u : 0u;
      uint8_t* vdst = base + G::kKeys + row * G::VS + seg * G::CPT * 2;
      if constexpr (VDT != kVF32) {
#pragma unroll
        for (int k = 0; k < G::VW; k += 4)
          *reinterpret_cast<v4u*>(vdst + 4 * k) =
              v4u{vw[i][k] & keep, vw[i][k + 1] & keep, vw[i][k + 2] & keep, vw[i][k + 3] & keep};
      } else {
        float x[G::VW];
#pragma unroll
        for (int k = 0; k < G::VW; ++k) x[k] = u2f(vw[i][k] & keep);
#pragma unroll
        for (int q = 0; q < G::TV; ++q) {
#pragma unroll
          for (int k = 0; k < G::VW; k += 8)
            *reinterpret_cast<v4u*>(vdst + q * KT * G::VS + 2 * k) =
                v4u{pack_high(x[k], x[k + 1]), pack_high(x[k + 2], x[k + 3]),
                    pack_high(x[k + 4], x[k + 5]), pack_high(x[k + 6], x[k + 7])};
#pragma unroll
          for (int k = 0; k < G::VW; ++k) x[k] = less_high(x[k]);
        }
      }
    }
  };

  v16f acc[G::NA];
#pragma unroll
  for (int t = 0; t < G::NA; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[t][i] = 0.f;
  float m = kLeastF, l = 0.f;
  const float slope = a.slopes ? a.slopes[hk * c.hq_per_kv + qh] : 0.f;
  const float inv_cap = 1.f / a.cap, cap_scale = 2.f * kLog2eF / a.cap;

  // ---- one step: KT keys, blocks of 32 ----
  // Scores of block e of a buffer: 16 of a row's 32 (element i is key 8 (i / 4) + 4 half + i % 4).
  auto scores = [&](int buf, int e, v16f& sv) __attribute__((always_inline)) {
    const uint8_t* kl = smem + buf * G::kBuf + (32 * e + r32) * G::KS + half * 16;
#pragma unroll
    for (int i = 0; i < 16; ++i) sv[i] = 0.f;
#pragma unroll
    for (int k = 0; k < G::NK; ++k) {
      const v8h k0 = *reinterpret_cast<const v8h*>(kl + 32 * k);
      if constexpr (G::TK == 2) {
        const v8h k1 = *reinterpret_cast<const v8h*>(kl + KT * G::KS + 32 * k);
        sv = __builtin_amdgcn_mfma_f32_32x32x16_f16(k1, qop[0][k], sv, 0, 0, 0);
      }
      if constexpr (G::TQ == 2)
        sv = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qop[1][k], sv, 0, 0, 0);
      sv = __builtin_amdgcn_mfma_f32_32x32x16_f16(k0, qop[0][k], sv, 0, 0, 0);
    }
  };
  auto largest = [&](const v16f& x, float top) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 16; i += 2) top = max3(top, x[i], x[i + 1]);
    return top;
  };
  // The shift follows the rows' largest score, and the sums it.
  auto raise = [&](float top) __attribute__((always_inline)) {
    if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > m + kSlack) != 0, 0)) {
      const float mn = fmaxf(m, top);
      const float g = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= g;
#pragma unroll
      for (int t = 0; t < G::NA; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] *= g;
    }
  };
  // Probabilities of a block, B operands of its two products of 16 keys; their sum.
  struct Prob {
    v4u p[2][G::TP];
  };
  auto weigh = [&](const v16f& x, float f2, Prob& r) __attribute__((always_inline)) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        float y0 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * ks + 2 * k], f2, -m));
        float y1 = __builtin_amdgcn_exp2f(__builtin_fmaf(x[8 * ks + 2 * k + 1], f2, -m));
        if constexpr (WIDE) l += y0 + y1;
        if constexpr (VDT == kVF16) {
          r.p[ks][0][k] = pack_f16(y0, y1);
          if constexpr (WIDE) {
            const v2h h = __builtin_bit_cast(v2h, (unsigned)r.p[ks][0][k]);
            r.p[ks][1][k] = pack_f16(y0 - (float)h[0], y1 - (float)h[1]);
          } else {
            l = __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, (unsigned)r.p[ks][0][k]),
                                       v2h{(_Float16)1.f, (_Float16)1.f}, l, false);
          }
        } else if constexpr (WIDE) {
#pragma unroll
          for (int q = 0; q < 3; ++q) {
            r.p[ks][q][k] = pack_high(y0, y1);
            y0 = less_high(y0);
            y1 = less_high(y1);
          }
        } else {
          r.p[ks][0][k] = pack_bf16(y0, y1);
          l = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2bf, (unsigned)r.p[ks][0][k]),
                                              v2bf{(__bf16)1.f, (__bf16)1.f}, l, false);
        }
      }
  };
  const int l16 = lane & 15;
  const int v_lane = (4 * half + (l16 >> 2)) * G::VS + ((lane & 16) + 4 * (l16 & 3)) * 2;
  auto values = [&](int buf, int e, const Prob& r) __attribute__((always_inline)) {
    const uint8_t* vl = smem + buf * G::kBuf + G::kKeys + v_lane;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int t = 0; t < G::NA; ++t)
#pragma unroll
        for (int q = 0; q < G::TV; ++q) {
          const uint8_t* at = vl + (q * KT + 32 * e + 16 * ks) * G::VS + 64 * t;
          typedef __attribute__((address_space(3))) v4s lds_v4s;
          const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_v4s*)(__attribute__((address_space(3))) void*)at);
          const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (lds_v4s*)(__attribute__((address_space(3))) void*)(at + 8 * G::VS));
          typedef short v8s __attribute__((ext_vector_type(8)));
          const v8s av = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
          // (Of the float32 values' terms q and the probabilities' z those with q + z < 3.)
#pragma unroll
          for (int z = 0; z < G::TP; ++z)
            if (z + q < 3) {
              if constexpr (VDT == kVF16)
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    __builtin_bit_cast(v8h, av), __builtin_bit_cast(v8h, r.p[ks][z]), acc[t], 0, 0,
                    0);
              else
                acc[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                    __builtin_bit_cast(v8bf, av), __builtin_bit_cast(v8bf, r.p[ks][z]), acc[t], 0,
                    0, 0);
            }
        }
  };
  // Whether a step counts for this wave, and needs no mask.
  auto skipped = [&](int t0) {
    return idle || !(t0 < w_hi.head || (t0 <= w_hi.pos && t0 + KT > w_lo.low));
  };
  auto whole_at = [&](int t0) {
    return t0 + KT <= w_lo.head || (t0 + KT - 1 <= w_lo.pos && t0 >= w_hi.low);
  };
  const bool scored = a.cap > 0.f || a.slopes;
  auto factor = [&](int buf) {
    const int e2 = min(max(q_unit + __builtin_amdgcn_readfirstlane(unit_s[buf]), -120), 120);
    return ldexpf(1.f, e2);
  };

  // A step. The second block's weights go with the first one's values.
  auto compute = [&](int s, int buf) __attribute__((always_inline)) {
    const int t0 = key0_of(s);
    if (skipped(t0)) return;
    v16f x[NS];
#pragma unroll
    for (int e = 0; e < NS; ++e) scores(buf, e, x[e]);
    const float f = factor(buf);
    float f2 = f * kLog2eF;                            // to units of log2
    if (scored || !whole_at(t0)) {
      if (a.cap > 0.f) {
#pragma unroll
        for (int e = 0; e < NS; ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            x[e][i] = WIDE ? soft_cap(x[e][i] * f, a.cap, inv_cap)
                           : quick_cap(x[e][i], a.cap, cap_scale * f);
        f2 = kLog2eF;
      }
      if (a.slopes) {
        const float d0 = (float)(view.pos - t0 - 4 * half), s2 = slope * kLog2eF;
#pragma unroll
        for (int e = 0; e < NS; ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            x[e][i] = __builtin_fmaf(-s2, fabsf(d0 - (float)(32 * e + 8 * (i / 4) + i % 4)),
                                     x[e][i] * f2);
        f2 = 1.f;
      }
      if (!whole_at(t0)) {
#pragma unroll
        for (int e = 0; e < NS; ++e)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int t = t0 + 4 * half + 32 * e + 8 * (i / 4) + i % 4;
            x[e][i] = sees(view, t) ? x[e][i] : -INFINITY;
          }
      }
    }
    float top = -INFINITY;
#pragma unroll
    for (int e = 0; e < NS; ++e) top = largest(x[e], top);
    raise(over_halves_max(top) * f2 - kUp);
    Prob p[NS];
    weigh(x[0], f2, p[0]);
#pragma unroll
    for (int e = 0; e < NS; ++e) {
      if (e + 1 < NS) weigh(x[e + 1], f2, p[e + 1]);
      values(buf, e, p[e]);
    }
  };

  if (s0 < s1) {
    load_entries(s0);
    load_tile(s0);
    load_entries(s0 + 1);
    if constexpr (G::NBUF == 2) {
      write_tile(s0, 0);
      load_tile(s0 + 1);
      load_entries(s0 + 2);
      __syncthreads();
      for (int s = s0; s < s1; ++s) {
        const int buf = (s - s0) & 1;
        // Half the waves stage the next step before they compute, half behind it: the waves
        // of a SIMD are not in the same part of a step.
        auto stage = [&]() __attribute__((always_inline)) {
          if (s + 1 < s1) {
            write_tile(s + 1, buf ^ 1);
            load_tile(s + 2);
            load_entries(s + 3);
          }
        };
        if (w >= G::WAVES / 2) stage();
        compute(s, buf);
        if (w < G::WAVES / 2) stage();
        __syncthreads();
      }
    } else {
      for (int s = s0; s < s1; ++s) {
        write_tile(s, 0);
        if (s + 1 < s1) {
          load_tile(s + 1);
          load_entries(s + 2);
        }
        __syncthreads();
        compute(s, 0);
        __syncthreads();
      }
    }
  }

  // ---- the end ----
  l = over_halves_sum(l);
  const bool seen = live && sees_tiles(view, list, j0, j1);
  const float inv = seen ? 1.f / l : 0.f;
  float probe = l;
#pragma unroll
  for (int t = 0; t < G::NA; ++t)
#pragma unroll
    for (int i = 0; i < 16; ++i) probe = __builtin_fmaf(acc[t][i], 0.f, probe);
  // (Infinite sums count too: of rows that a value's infinity reaches they are right, but
  // their workgroup holds rows that it does not.)
  const bool bad = seen && !(probe > 0.f && probe < INFINITY);
  if (__syncthreads_or(bad || (j0 < j1 && wild_s))) {
    const AttendArgs& a = late_attend_args();
    const DecodeArgs& c = a.c;
#pragma unroll 1
    for (int r = row0 + w; r < row1; r += G::WAVES) {
      const int i = r / c.hq_per_kv;
      const RowView v = row_view(a, n, cnt, prefix, i);
      const RowSums<D> x = plain_row<D, VDT>(a, b, hk, r, n, v, list, j0, j1);
      store_plain_row<D>(a, b, hk, r, split, x, x.m != kLeastF);
    }
    return;
  }
  if (R >= rows) return;
  if (c.final_out) {
#pragma unroll
    for (int t = 0; t < G::NA; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4) {
        const int64_t at = out_row * D + 32 * t + 2 * i + 4 * half;
        float y[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] = seen ? acc[t][i + k] * inv : 0.f;
        if (c.out_dtype == kEF32)
          *reinterpret_cast<float4*>(static_cast<float*>(c.out) + at) =
              make_float4(y[0], y[1], y[2], y[3]);
        else
          *reinterpret_cast<uint2*>(static_cast<unsigned short*>(c.out) + at) =
              c.out_dtype == kEF16
                  ? make_uint2(pack_f16(y[0], y[1]), pack_f16(y[2], y[3]))
                  : make_uint2((unsigned)bf16_rne(y[0]) | (unsigned)bf16_rne(y[1]) << 16,
                               (unsigned)bf16_rne(y[2]) | (unsigned)bf16_rne(y[3]) << 16);
      }
    return;
  }
  const int64_t at = out_row * c.num_splits + split;
  if (seen) {
#pragma unroll
    for (int t = 0; t < G::NA; ++t)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<float4*>(c.ws_acc + at * D + 32 * t + 2 * i + 4 * half) =
            make_float4(acc[t][i], acc[t][i + 1], acc[t][i + 2], acc[t][i + 3]);
  }
  if (half == 0) {
    c.ws_ml[2 * at] = seen ? (double)m * (double)kLn2 : -INFINITY;
    c.ws_ml[2 * at + 1] = seen ? (double)l : 0.0;
  }
}

template <int D, int VDT, bool WIDE>
hipError_t launch_chunk(AttendArgs a, int batch, hipStream_t st) {
  using G = ChunkGeo<D, VDT, WIDE>;
  const int rows = a.c.hq_per_kv * a.queries;
  a.tiles = (rows + G::M - 1) / G::M;
  const int64_t wgs = (int64_t)a.tiles * a.c.num_splits * batch * a.kv_heads;
  if (!grid_fits(wgs, G::NT)) return hipErrorInvalidValue;
  hipLaunchKernelGGL((attend_chunk_kernel<D, VDT, WIDE>), dim3((unsigned)wgs), dim3(G::NT), 0, st,
                     a);
  return hipGetLastError();
}

hipError_t launch_attend_chunk(const AttendArgs& a, int D, int v_dtype, int batch,
                               hipStream_t st) {
  const bool wide = attend_wide(a.c.out_dtype, v_dtype, a.cap);
#define FDI4_CHUNK(DD, VV)                                                        \
  if (D == DD && v_dtype == VV)                                                   \
    return wide ? launch_chunk<DD, VV, true>(a, batch, st) : launch_chunk<DD, VV, false>(a, batch, st);
  FDI4_CHUNK(64, kVF32) FDI4_CHUNK(64, kVF16) FDI4_CHUNK(64, kVBF16)
  FDI4_CHUNK(128, kVF32) FDI4_CHUNK(128, kVF16) FDI4_CHUNK(128, kVBF16)
  FDI4_CHUNK(256, kVF32) FDI4_CHUNK(256, kVF16) FDI4_CHUNK(256, kVBF16)
#undef FDI4_CHUNK
  return hipErrorInvalidValue;
}

}  // namespace fdi4
