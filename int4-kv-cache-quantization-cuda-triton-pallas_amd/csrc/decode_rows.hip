// Attention of several query rows per (sequence, kv-head) over part of the paged INT4
// cache and over drafted tokens, on the matrix cores (gfx950). For the row of node i
// and q-head h of sequence b, with n cached tokens and d_i drafts that node i sees,
//
//   out = sum_t p_t v_t / sum_t p_t,   p_t = exp(q . k_t - max)
//
// over the cached tokens t < n with t < sinks or t >= n + d_i - window (all of them
// without a window; d_i = 0 without drafts, the query being the last cached token),
// k_t = nib*scale - zp*scale, and over the drafts j with mask[i, j]. A row that sees
// nothing is zero.
//
// A workgroup of four waves serves RT tiles of 16 rows of one kv-head over a range of
// scale groups (and drafts, 64 an item, at the range's end). Its 16-row chunks of keys
// go to the waves in turn, so the cache is read once for all its rows, straight to
// registers; the waves meet at the end, in LDS, and splits in the merge kernel.
//
//   terms: q . k_t = sum_d v_d (nib_td - zp_d), v = q*s. Per group and row, v is made
//      into a few narrow terms, once for the group's 128 keys, and multiplied by the
//      nibbles as they are stored, where dequantized keys would need two or three terms
//      against as many of the query; the constant sum_d v_d zp_d, in float32, goes in
//      with the exponent's FMA. A product takes 16 keys (A) and 16 rows (B).
//      The terms are in units of a power of two for the largest |v| of the row and the
//      group. 16-bit outputs: two float16 terms of 11 bits (21 of v in all, and down to
//      2^-39 of the largest), for v_mfma_f32_16x16x32_f16 with a nibble at bits 6 to 9 of
//      a float16, the number nib * 2^-18. That instruction aligns a product of a number
//      below 2^-14 as if it were 2^-14 and keeps 24 bits: nibbles in the lowest bits
//      (nib * 2^-24) cost a sum of 32 2^-17 of its largest product, six bits up they cost
//      2^-24, as float32 sums do. Three shifts a word more: 118 us in place of 116 for 64
//      rows of bfloat16 at 16384 tokens.
//      float32 outputs (WIDE): an integer below 2^30, in four balanced base-256 digits
//      for v_mfma_i32_16x16x64_i8, whose exact sums meet in float32: as good as float32
//      products of q and k (2-norm error 3e-7 over 300 keys of 128 channels, 4e-7 with
//      those).
//      The terms are built by the whole workgroup for the next group while the present
//      one is multiplied (two LDS buffers, one barrier a group), from scales that a wave
//      stages for a group of its own every four.
//   softmax: lane (g, r) of a wave holds the logits of row r with keys 4g .. 4g+3, and
//      the value product wants its B operand in the same lanes, so probabilities never
//      leave their registers. The shift is a whole number that moves only when a logit
//      passes it by kSlack (a power of two, so probabilities stay in their type's
//      range); the accumulators are rescaled then and not for every new maximum.
//   values: lane (g, r) loads the channels 8r.. of rows 4g .. 4g+3, byte permutes pair
//      the rows, and one product takes 32 keys. A probability is the sum of two
//      (float16: 22 bits; bfloat16: 16) or three (bfloat16 values, float32 output:
//      24) terms. (16 bits are off by a 64th of a float16 output's half step, a 512th of a
//      bfloat16 one's; a third term took 128 us in place of 118 for 64 rows at 16384
//      tokens, and changed one bfloat16 output in 1300.) float32 values are three bfloat16 terms like it: 58 us, where
//      v_mfma_f32_16x16x4_f32 took 68 (100 drafts of four sequences of up to 3000
//      tokens).
//
// A non-finite value times a probability of zero is NaN, though the row does not see
// it: a workgroup that ends with a NaN goes through its range again, row by row and key
// by key (14 ms where eight sequences of 8192 tokens all do, 71 us otherwise). Rows whose
// query is not finite are NaN without it, if they see anything, and values that no row
// sees are dropped: a batch padded with either is no slower.
//
// What bounds it. Up to 32 rows a kv-head: memory. 8 sequences of 8 kv-heads with 128
// bfloat16 channels and 16 rows read their tokens at 6.5 TB/s once they are many, on top
// of 11 us (launch, the first loads' chain, the waves' and the splits' merges): 37 us at
// 8192 tokens, 64 us at 16384, 5.4 TB/s in all. More rows: each further workgroup of 32
// rows takes its keys again, from L2, and the time follows the rows: 126 us for 64 rows
// at 16384 tokens, 221 us for 128, of which 114 and 204 us remain where all pages lie in
// L2. A step (32 keys by 32 rows, a wave) takes about 7800 cycles, two waves a SIMD,
// with the VALU busy for 54 % of them, the matrix cores for 28 %; the rest waits for LDS,
// dependent results and the barrier.
//
// RT: one tile up to 16 rows (and at 256 channels, whose accumulators fill the registers
// with one), two beyond: 32 rows in one workgroup read the cache once (78 us at 16384
// tokens, 64 us for 16 rows). Four tiles in one workgroup of eight waves were slower
// than two workgroups of two: one barrier for all of them.
// STREAM: non-temporal loads where one workgroup reads a page, cached ones where the
// workgroups of several tiles do, which run on one XCD one after the other.
// Splits: as many as fill the chip twice over with workgroups (two fit a CU).

#include "decode_common.hpp"

namespace fdi4 {

typedef int v4i __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kWaves = 4;

// The kernel's arguments, read again from where they lie: a phase that follows the key
// loop uses this copy, so that its arguments hold no scalar registers in the loop (those
// that do not fit go to lanes of vector registers, which do not fit then).
__device__ __forceinline__ const RowsArgs& late_args() {
  auto p = __builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(p));
  return *(const RowsArgs*)p;
}

template <int D, int VDT, int RT, bool WIDE>
struct RowsGeo {
  static constexpr int ND = WIDE ? 4 : 2;          // terms of q*s
  static constexpr int TB = WIDE ? 1 : 2;          // bytes of a term
  static constexpr int NB = D / 64;                // 64-channel blocks of the key product
  static constexpr int KW = D / 32;                // packed key words per lane per row
  static constexpr int VEB = VDT == kVF32 ? 4 : 2;
  static constexpr int PB = D * VEB / 16 < 16 ? D * VEB / 16 : 16;  // bytes per value load
  static constexpr int NP = D * VEB / (16 * PB);   // value loads per lane per row
  static constexpr int CPP = PB / VEB;             // channels per value load
  static constexpr int NA = D / 16;                // 16-channel output tiles
  static constexpr int CPS = VDT == kVF32 ? 1 : 2; // chunks per step
  static constexpr int M = 16 * RT;           // rows of the workgroup
  static constexpr int NT = kWaves * 64;           // threads
  static constexpr int TPR = NT / M;               // threads per row that build terms
  static constexpr int SPT = D / TPR;              // channels each
  static constexpr int DS = D * TB + 16;           // bytes per row of a term (padded)
  static constexpr int kDig = ND * M * DS;         // a buffer of terms
  static constexpr int AS = D + 4;                 // floats per row of queries and outputs
  // Scales, and zero-points times them, of a group, in slot order; four floats of
  // padding every 16 keep the threads of a row, 16 channels apart, on different banks.
  static constexpr int kSz = D + D / 4;
  // LDS: two buffers of terms, the queries and twice kWaves groups' scales while the keys
  // stream, then the waves' outputs.
  static constexpr int kQ = 2 * kDig;
  static constexpr int kScales = kQ + M * AS * 4;
  static constexpr int kStream = kScales + 2 * kWaves * 2 * kSz * 4;
  static constexpr int kAcc = kWaves * M * AS * 4;
  static constexpr int kSmem = kStream > kAcc ? kStream : kAcc;
  static_assert(TPR >= 4 && TPR <= 16 && (TPR & (TPR - 1)) == 0 && SPT % 4 == 0, "threads");
};

// Position of channel d in the operands' order, of every eight channels (a word of
// nibbles): digits, the even ones (low nibbles) before the odd ones; float16 terms, the
// pairs (j, j + 4) of nibbles that lie 16 bits apart.
template <bool WIDE>
__device__ __forceinline__ int row_slot(int d) {
  return WIDE ? (d & ~7) | ((d & 1) << 2) | ((d & 7) >> 1)
              : (d & ~7) | ((d & 3) << 1) | ((d & 7) >> 2);
}

// Eight channels of a query as float32, from 16-byte loads (VEC) or element by element.
__device__ __forceinline__ void load_query8(const void* q, int64_t i, int dt, bool vec, float* x) {
  if (!vec) {
#pragma unroll
    for (int k = 0; k < 8; ++k) x[k] = load_elem(q, i + k, dt);
  } else if (dt == kEF32) {
    const float* p = static_cast<const float*>(q) + i;
    widen_values<kVF32>(ld16(p), x);
    widen_values<kVF32>(ld16(p + 4), x + 4);
  } else {
    const U32x4 v = ld16(static_cast<const unsigned short*>(q) + i);
    if (dt == kEF16) widen_values<kVF16>(v, x);
    else widen_values<kVBF16>(v, x);
  }
}

// KW words of a key or value row: streamed (non-temporal) where one workgroup reads them,
// through the caches where the workgroups of other rows do too.
template <int KW, bool STREAM>
__device__ __forceinline__ KVec<KW> load_words(const uint8_t* p) {
  if constexpr (STREAM) return load_k<KW>(p);
  return *reinterpret_cast<const KVec<KW>*>(__builtin_assume_aligned(p, 4 * KW));
}

// Value of lane ^ 4: mirrored within 8 lanes, then within 4.
__device__ __forceinline__ unsigned xchg4(unsigned x) {
  return (unsigned)__builtin_amdgcn_mov_dpp(
      __builtin_amdgcn_mov_dpp((int)x, 0x141, 0xF, 0xF, false), 0x1B, 0xF, 0xF, false);
}

// A lane's number as a value of unknown origin: what is computed from it in a loop is
// computed there. (Four digits leave no registers to keep a few addresses in: spilled,
// they made 64 rows of 16-bit values and float32 outputs 85 us in place of 76.)
__device__ __forceinline__ int fresh(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Maximum and sum over the four 16-lane groups.
// (The maximum without the quieting moves that fmax puts before operands of unknown
// origin; the instruction quiets them itself.)
__device__ __forceinline__ float max_of(float x, float y) {
  float r;
  asm("v_max_f32 %0, %1, %2" : "=v"(r) : "v"(x), "v"(y));
  return r;
}

__device__ __forceinline__ float over_groups_max(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = max_of(u2f(r[0]), u2f(r[1]));
  auto s = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return max_of(u2f(s[0]), u2f(s[1]));
}

__device__ __forceinline__ float over_groups_sum(float x) {
  auto r = __builtin_amdgcn_permlane16_swap(f2u(x), f2u(x), false, false);
  x = u2f(r[0]) + u2f(r[1]);
  auto s = __builtin_amdgcn_permlane32_swap(f2u(x), f2u(x), false, false);
  return u2f(s[0]) + u2f(s[1]);
}

// RT: row tiles. WIDE: float32 outputs (four digits of q*s, all 24 bits of a
// probability); otherwise two float16 terms and at least 16 bits. STREAM: keys and values
// are read by one workgroup only (non-temporal loads).
template <int D, int VDT, int RT, bool WIDE, bool STREAM>
__global__ __launch_bounds__(kWaves * 64, 2) void decode_rows_kernel(RowsArgs a) {
  // 16-bit terms of a probability.
  constexpr int TERMS = VDT == kVF32 || (WIDE && VDT == kVBF16) ? 3 : 2;
  using G = RowsGeo<D, VDT, RT, WIDE>;
  constexpr int ND = G::ND, NB = G::NB, CPS = G::CPS, NA = G::NA, M = G::M, NT = G::NT;
  constexpr int TPR = G::TPR, SPT = G::SPT, NS = 4 * CPS;
  // Shift of the probabilities: the largest is 2^kUp when the shift moves, and stays
  // below 2^(kUp + kSlack). float16 terms need the headroom (2^16) and the small end
  // (quantum 2^-24): a probability's terms are exact to 2^-37 of the largest.
  constexpr float kUp = VDT == kVF16 ? 13.f : 0.f;
  constexpr float kSlack = VDT == kVF16 ? 2.f : 8.f;
  constexpr float kLeast = -3.4028235e38f;
  constexpr float kLog2e = 1.44269504088896f;

  const DecodeArgs& c = a.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int n16 = lane & 15, grp = lane >> 4;

  // Tiles of one (sequence, kv-head, split) run on one XCD, one after the other: they
  // read the same pages.
  int wi = (int)blockIdx.x, tile = 0;
  if (a.tiles > 1) {
    const int L = (int)xcd_run_item(blockIdx.x, gridDim.x, (unsigned)a.tiles);
    wi = L / a.tiles;
    tile = L - wi * a.tiles;
  }
  int wj = fdiv(wi, c.div_splits);
  const int split = wi - wj * c.num_splits;
  const int b = fdiv(wj, a.div_heads), hk = wj - b * a.kv_heads;
  const int rows = c.hq_per_kv * a.nodes;          // rows of this kv-head
  const int row0 = tile * M;
  const int live = min(rows - row0, M);            // rows of this workgroup

  __shared__ __align__(16) uint8_t smem[G::kSmem];
  constexpr int kSz = G::kSz;
  auto sz_pos = [](int slot) { return slot + slot / 16 * 4; };
  __shared__ float2 cc_s[2][M];                    // a row's logit unit and constant
  __shared__ int low_s[M];                         // first cached token in a row's window
  __shared__ int ext_s[2];                         // smallest and largest of them
  __shared__ int seen_s[M];                        // a row sees a key of this range
  __shared__ int wild_s[M];                        // its query is not finite
  __shared__ float m_s[kWaves][M], l_s[kWaves][M];
  __shared__ int bad_s;
  float* const q_s = reinterpret_cast<float*>(smem + G::kQ);
  float* const sz_s = reinterpret_cast<float*>(smem + G::kScales);

  // This thread's part of a row of terms: brow's channels part * SPT .. (of eight, the
  // even or the odd ones where SPT is four).
  const int brow = tid / TPR, part = tid % TPR;
  constexpr int NQ = SPT / 8 > 0 ? SPT / 8 : 1;
  float qv[NQ][8];
  {
    const int R = row0 + min(brow, live - 1), hr = fdiv(R, a.div_nodes);
    const int64_t q0 = (int64_t)b * c.q_b + (int64_t)(hk * c.hq_per_kv + hr) * c.q_h +
                       (int64_t)(R - hr * a.nodes) * a.q_n + (part * SPT & ~7);
#pragma unroll
    for (int i = 0; i < NQ; ++i) load_query8(c.q, q0 + 8 * i, c.q_dtype, a.q_vec, qv[i]);
  }

  const int n = seq_len_of(c, b);
  if (c.lens_out && tile == 0 && split == 0 && hk == 0 && tid == 0)
    c.lens_out[b] = c.seq_lens[b];

  // ---- each row's window ----
  int low_min = 0, low_max = 0;
  if (a.window) {
    low_min = low_max = max(n - a.window, 0);
    if (a.mask) {
      // It ends at the node, whose visible drafts count.
      const int R = row0 + min(brow, live - 1), node = R - fdiv(R, a.div_nodes) * a.nodes;
      const uint8_t* mk = a.mask + (int64_t)b * a.mk_b + (int64_t)node * a.mk_i;
      int mine = 0;
      // (Eight in flight: one wait for memory up to 8 * TPR nodes.)
      for (int j0 = part; j0 < a.nodes; j0 += 8 * TPR) {
        uint8_t x[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) x[k] = mk[min(j0 + k * TPR, a.nodes - 1)];
#pragma unroll
        for (int k = 0; k < 8; ++k) mine += (x[k] != 0) & (j0 + k * TPR < a.nodes);
      }
      mine += (int)xchg_u32<1>((unsigned)mine);
      mine += (int)xchg_u32<2>((unsigned)mine);
      if constexpr (TPR > 4) mine += (int)xchg_u32<4>((unsigned)mine);
      if constexpr (TPR > 8) mine += (int)xchg_u32<8>((unsigned)mine);
      const int low = (int)min(max((int64_t)n + mine - a.window, (int64_t)0), (int64_t)n);
      if (tid == 0) {
        ext_s[0] = 0x7FFFFFFF;
        ext_s[1] = 0;
      }
      __syncthreads();
      if (part == 0) {
        low_s[brow] = low;
        atomicMin(&ext_s[0], low);
        atomicMax(&ext_s[1], low);
      }
      __syncthreads();
      low_min = __builtin_amdgcn_readfirstlane(ext_s[0]);
      low_max = __builtin_amdgcn_readfirstlane(ext_s[1]);
    } else if (tid < M) {
      low_s[tid] = low_min;
    }
  } else if (tid < M) {
    low_s[tid] = 0;
  }

  // ---- the items: scale groups of the sinks, of the window, and 64 drafts each ----
  const int group_rows = c.pages_per_group * c.page_rows;
  const int cpp = (c.page_rows + 15) >> 4, cpg = cpp * c.pages_per_group;
  const int gend = fdiv(n + group_rows - 1, a.div_group);
  const int gw0 = a.sinks >= low_min ? 0 : fdiv(low_min, a.div_group);
  const int nsg = min(fdiv(min(a.sinks, n) + group_rows - 1, a.div_group), gw0);
  const int ng = nsg + max(gend - gw0, 0);
  const int nd = a.mask ? (a.nodes + 63) >> 6 : 0;
  const int tot = ng + nd;
  const int i0 = (int)((int64_t)split * tot / c.num_splits);
  const int i1 = (int)((int64_t)(split + 1) * tot / c.num_splits);
  const int it0 = min(i0, ng), it1 = min(i1, ng);
  const int dr0 = max(i0, ng) - ng, dr1 = max(i1, ng) - ng;
  auto group_of = [&](int it) { return it < nsg ? it : it - nsg + gw0; };
  // Whether a row sees a cached token of the range (a group of the sinks begins with
  // one; those of the window follow one another), and no draft yet.
  if (tid < M) {
    const int w0 = max(it0, nsg), t0 = (w0 - nsg + gw0) * group_rows;
    const int t1 = min((it1 - nsg + gw0) * group_rows, n);
    seen_s[tid] = it0 < min(it1, nsg) ||
                  (w0 < it1 && (max(t0, low_s[tid]) < t1 || t0 < min(a.sinks, t1)));
    wild_s[tid] = 0;
  }
  if (tid == 0) bad_s = 0;

  const float* sbase = c.k_scale + (int64_t)b * c.s_b + (int64_t)hk * c.s_h;
  const float* zbase = c.k_zp + (int64_t)b * c.s_b + (int64_t)hk * c.s_h;
  const uint8_t* kbase = c.k_pages + (int64_t)hk * c.k_head;
  const uint8_t* vbase = reinterpret_cast<const uint8_t*>(c.v_pages) +
                         (int64_t)hk * c.v_head * G::VEB;
  const unsigned krow_b = (unsigned)c.k_row, vrow_b = (unsigned)(c.v_row * G::VEB);
  // Offsets of this lane's key row and value rows in a full chunk; a partial one takes
  // the smaller of these and the last valid row's.
  const unsigned k_lane = grp * (D / 8), v_lane = n16 * G::PB;
  const unsigned k_full = k_lane + n16 * krow_b;
  unsigned v_full[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v_full[i] = v_lane + (4 * grp + i) * vrow_b;
  const int32_t* table = c.page_table ? c.page_table + (int64_t)b * c.pt_b : nullptr;

  // ---- a step: CPS chunks of 16 rows of a group, for this wave ----
  const int spg = (cpg + CPS * kWaves - 1) / (CPS * kWaves);
  // The table entries are loaded with the metadata and first used a step later.
  struct Meta {
    int entry[CPS], r0[CPS], nval[CPS], tok0[CPS];
  };
  int li = it0, lp = 0;                            // item and step of the next metadata
  auto next_meta = [&]() __attribute__((always_inline)) -> Meta {
    Meta m;
    const int g = group_of(min(li, it1 - 1));
#pragma unroll
    for (int e = 0; e < CPS; ++e) {
      const int j = (lp * CPS + e) * kWaves + w;
      const int pj = fdiv(j, c.div_cpp);
      const int page = g * c.pages_per_group + pj;
      const int r0 = (j - pj * cpp) * 16;
      const int tok0 = page * c.page_rows + r0;
      int nval = j < cpg && li < it1 ? min(min(16, c.page_rows - r0), n - tok0) : 0;
      // Behind the sinks and before every row's window.
      if (tok0 >= a.sinks && tok0 + nval <= low_min) nval = 0;
      const int at = __builtin_amdgcn_readfirstlane(min(page, c.max_pages - 1));
      m.entry[e] = at;
      if (table) m.entry[e] = ld_ro(table, at);
      m.r0[e] = r0;
      m.nval[e] = __builtin_amdgcn_readfirstlane(nval);
      m.tok0[e] = __builtin_amdgcn_readfirstlane(tok0);
    }
    if (++lp == spg) {
      lp = 0;
      ++li;
    }
    return m;
  };
  auto phys_of = [&](const Meta& m, int e) __attribute__((always_inline)) -> uint64_t {
    return (unsigned)__builtin_amdgcn_readfirstlane(
        min(max(m.entry[e], 0), c.num_pages - 1));
  };

  // Rows past the valid count are loaded from the last valid row, a chunk of none from
  // its first (never out of bounds, and its values are dropped).
  struct Keys {
    unsigned w[CPS][G::KW];
  };
  struct Vals {
    unsigned w[CPS][4][G::NP][G::PB / 4];
  };
  auto load_keys = [&](const Meta& m, Keys& f) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < CPS; ++e) {
      const uint8_t* kb = kbase + (phys_of(m, e) * a.k_page_b +
                                   (uint64_t)(unsigned)m.r0[e] * krow_b);
      const unsigned ko = min(k_full, k_lane + (unsigned)max(m.nval[e] - 1, 0) * krow_b);
      constexpr int KL = G::KW < 4 ? G::KW : 4;
#pragma unroll
      for (int i = 0; i < G::KW / KL; ++i) {
        const KVec<KL> x = load_words<KL, STREAM>(kb + (ko + 16 * i));
#pragma unroll
        for (int k = 0; k < KL; ++k) f.w[e][KL * i + k] = x.w[k];
      }
    }
  };
  auto load_values = [&](const Meta& m, Vals& f) __attribute__((always_inline)) {
#pragma unroll
    for (int e = 0; e < CPS; ++e) {
      const unsigned v_last = v_lane + (unsigned)max(m.nval[e] - 1, 0) * vrow_b;
      const uint8_t* vb = vbase + (phys_of(m, e) * a.v_page_b +
                                   (uint64_t)(unsigned)m.r0[e] * vrow_b);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned vo = min(v_full[i], v_last);
#pragma unroll
        for (int u = 0; u < G::NP; ++u) {
          const KVec<G::PB / 4> x =
              load_words<G::PB / 4, STREAM>(vb + (vo + 16 * G::PB * u));
#pragma unroll
          for (int k = 0; k < G::PB / 4; ++k) f.w[e][i][u][k] = x.w[k];
        }
      }
    }
  };

  // ---- scales of a group to LDS, and the rows' terms ----
  // Lane l holds the scales and zero-points of channels SL * l .. (SL = D / 64).
  constexpr int SL = D / 64;
  struct Scales {
    float s[SL], z[SL];
  };
  auto load_sz = [&](int it) __attribute__((always_inline)) -> Scales {
    const uint64_t off = (uint64_t)(unsigned)group_of(min(it, it1 - 1)) * a.s_group +
                         SL * (WIDE ? fresh(lane) : lane);
    struct alignas(4 * SL) Part {
      float v[SL];
    };
    const Part s = *reinterpret_cast<const Part*>(sbase + off);
    const Part z = *reinterpret_cast<const Part*>(zbase + off);
    Scales r;
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      r.s[k] = s.v[k];
      r.z[k] = z.v[k];
    }
    return r;
  };
  // The scales, and zero-points times them, by one wave to the slot of group it.
  auto slot_of = [&](int it) { return (it - it0) & (2 * kWaves - 1); };
  auto stage_sz = [&](const Scales& x, int it) __attribute__((always_inline)) {
    float* dst = sz_s + slot_of(it) * 2 * kSz;
    const int d0 = SL * (WIDE ? fresh(lane) : lane);
#pragma unroll
    for (int k = 0; k < SL; ++k) {
      const int at = sz_pos(row_slot<WIDE>(d0 + k));
      dst[at] = x.s[k];
      dst[kSz + at] = x.z[k] * x.s[k];
    }
  };
  float qn[SPT];                                   // the row's channels in slot order
  // The row's products with the scales of group it as terms, in units of a power of two
  // for the largest of them. (Not for the largest query times the largest scale, which
  // may lie in different channels: one channel of r times the query and 1/r times the
  // scale beside one of the opposite cost float32 outputs 2e-5 at r = 100 and 2e-3 at
  // 1000, where float32 products have 4e-7.)
  auto build = [&](int it) __attribute__((always_inline)) {
    const int buf = (it - it0) & 1;
    const float* sz = sz_s + slot_of(it) * 2 * kSz;
    const int own = WIDE ? fresh(tid) : tid, brow = own / TPR, part = own % TPR;
    uint8_t* dst = smem + buf * G::kDig + brow * G::DS + part * SPT * G::TB;
    float cg[4] = {0.f, 0.f, 0.f, 0.f}, mx[2] = {0.f, 0.f}, v[SPT];
    constexpr int OW = SPT * G::TB / 4;
    unsigned out[ND][OW];
    static_assert(SPT == 4 || SPT == 8 || SPT == 16, "operand stores");
#pragma unroll
    for (int i = 0; i < SPT; i += 4) {
      const float* src = sz + sz_pos(part * SPT + i);
      const float4 s4 = *reinterpret_cast<const float4*>(src);
      const float4 z4 = *reinterpret_cast<const float4*>(src + kSz);
      const float ss[4] = {s4.x, s4.y, s4.z, s4.w}, zz[4] = {z4.x, z4.y, z4.z, z4.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        cg[k] = __builtin_fmaf(qn[i + k], zz[k], cg[k]);
        v[i + k] = qn[i + k] * ss[k];
      }
#pragma unroll
      for (int k = 0; k < 2; ++k)
        mx[k] = fmaxf(mx[k], fmaxf(fabsf(v[i + k]), fabsf(v[i + k + 2])));
    }
    float top = fmaxf(mx[0], mx[1]);
    top = fmaxf(top, xchg<1>(top));
    top = fmaxf(top, xchg<2>(top));
    if constexpr (TPR > 4) top = fmaxf(top, u2f(xchg4(f2u(top))));
    if constexpr (TPR > 8) top = fmaxf(top, xchg<8>(top));
    // All products are below 2^kBits units. (Of NaN, which the maximum passes over, the
    // constant is NaN too.)
    constexpr unsigned kBits = WIDE ? 30 : 15;
    const unsigned ex = max(f2u(top) >> 23, 32u);
    const float up = u2f((253 + kBits - ex) << 23);
#pragma unroll
    for (int i = 0; i < SPT; i += 4) {
#pragma unroll
      for (int k = 0; k < 4; ++k) v[i + k] *= up;
      if constexpr (WIDE) {
        // The nearest integer, plus a bias that makes its lower bytes digits + 128.
        unsigned x[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (unsigned)(int)__builtin_rintf(v[i + k]) + 0x808080u;
        const unsigned t0 = __builtin_amdgcn_perm(x[1], x[0], 0x05010400u);
        const unsigned u0 = __builtin_amdgcn_perm(x[3], x[2], 0x05010400u);
        const unsigned t1 = __builtin_amdgcn_perm(x[1], x[0], 0x07030602u);
        const unsigned u1 = __builtin_amdgcn_perm(x[3], x[2], 0x07030602u);
        out[0][i / 4] = __builtin_amdgcn_perm(u0, t0, 0x05040100u) ^ 0x80808080u;
        out[1][i / 4] = __builtin_amdgcn_perm(u0, t0, 0x07060302u) ^ 0x80808080u;
        out[2][i / 4] = __builtin_amdgcn_perm(u1, t1, 0x05040100u) ^ 0x80808080u;
        out[3][i / 4] = __builtin_amdgcn_perm(u1, t1, 0x07060302u);
      } else {
        // (The second term is what the first cuts off, in the same units.)
#pragma unroll
        for (int k = 0; k < 4; k += 2) {
          const float x0 = v[i + k], x1 = v[i + k + 1];
          const float h0 = u2f(f2u(x0) & 0xFFFFE000u), h1 = u2f(f2u(x1) & 0xFFFFE000u);
          out[0][(i + k) / 2] =
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(h0, h1));
          out[1][(i + k) / 2] =
              __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(x0 - h0, x1 - h1));
        }
      }
    }
#pragma unroll
    for (int k = 0; k < ND; ++k) {
      uint8_t* o = dst + k * M * G::DS;
      if constexpr (OW == 2) {
        *reinterpret_cast<uint2*>(o) = make_uint2(out[k][0], out[k][1]);
      } else if constexpr (OW == 1) {
        *reinterpret_cast<unsigned*>(o) = out[k][0];
      } else {
#pragma unroll
        for (int i = 0; i < OW; i += 4)
          *reinterpret_cast<uint4*>(o + 4 * i) =
              make_uint4(out[k][i], out[k][i + 1], out[k][i + 2], out[k][i + 3]);
      }
    }
    float cgs = (cg[0] + cg[1]) + (cg[2] + cg[3]);
    cgs += xchg<1>(cgs);
    cgs += xchg<2>(cgs);
    if constexpr (TPR > 4) cgs += u2f(xchg4(f2u(cgs)));
    if constexpr (TPR > 8) cgs += xchg<8>(cgs);
    if (part == 0) {
      // (A product that is not finite makes the row NaN.)
      const float unit = ex == 255u ? u2f(0x7FC00000u) : u2f((ex + 1 - kBits) << 23);
      cc_s[buf][brow] =
          make_float2(unit * (WIDE ? kLog2e : kLog2e * 262144.f), cgs * kLog2e);
    }
  };

  // ---- softmax and values ----
  // (The sum of a row's probabilities is one more output channel, of ones: as an
  // accumulator of the 16-bit products, in every lane; per lane for float32 values.)
  float m_run[RT];
  v4f l_run[RT];
  v4f acc[RT][NA];
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    m_run[rt] = kLeast;
    l_run[rt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NA; ++t) acc[rt][t] = v4f{0.f, 0.f, 0.f, 0.f};
  }
  // Probabilities of a step as the value product's operands.
  constexpr int PW = NS / 2;                       // registers per term
  unsigned pr[RT][PW * TERMS];

  // Scores s (logit = s * c1 - cc, log2 units, c1 >= 0) of keys 4 grp + i of chunk e in
  // s[4 e + i], of which, if masked, those in vis are seen: of all row tiles together,
  // whose chains of dependent instructions run side by side.
  auto softmax = [&](float (*s)[NS], const float* c1, const float* cc, bool masked,
                     const unsigned* vis) __attribute__((always_inline)) {
    float top[RT], sub[RT];
    if (masked) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        top[rt] = kLeast;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
          s[rt][k] =
              (vis[rt] >> k) & 1u ? __builtin_fmaf(s[rt][k], c1[rt], -cc[rt]) : -INFINITY;
          top[rt] = fmaxf(top[rt], s[rt][k]);
        }
      }
    } else {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        top[rt] = kLeast;
#pragma unroll
        for (int k = 0; k < NS; ++k) top[rt] = fmaxf(top[rt], s[rt][k]);
        top[rt] = __builtin_fmaf(top[rt], c1[rt], -cc[rt]);
      }
    }
    bool up[RT], some = false;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      top[rt] = over_groups_max(top[rt]);
      up[rt] = top[rt] > m_run[rt] + (kUp + kSlack);
      some |= up[rt];
    }
    if (__builtin_amdgcn_ballot_w64(some)) {
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const float m_new = up[rt] ? __builtin_ceilf(top[rt]) - kUp : m_run[rt];
        const float corr = __builtin_amdgcn_exp2f(m_run[rt] - m_new);
        m_run[rt] = m_new;
        l_run[rt] *= corr;
#pragma unroll
        for (int t = 0; t < NA; ++t) acc[rt][t] *= corr;
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      if (masked) {
#pragma unroll
        for (int k = 0; k < NS; ++k) s[rt][k] -= m_run[rt];
      } else {
        sub[rt] = -cc[rt] - m_run[rt];
#pragma unroll
        for (int k = 0; k < NS; ++k) s[rt][k] = __builtin_fmaf(s[rt][k], c1[rt], sub[rt]);
      }
    }
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float* p = s[rt];
#pragma unroll
      for (int k = 0; k < NS; ++k) p[k] = __builtin_amdgcn_exp2f(p[k]);
      if constexpr (VDT == kVF32) l_run[rt][0] += (p[0] + p[1]) + (p[2] + p[3]);
#pragma unroll
      for (int h = 0; h < PW; ++h) {
        float y0 = p[2 * h], y1 = p[2 * h + 1];
#pragma unroll
        for (int q = 0; q < TERMS; ++q) {
          if constexpr (VDT == kVF16) {
            const float h0 = q == TERMS - 1 ? y0 : u2f(f2u(y0) & 0xFFFFE000u);
            const float h1 = q == TERMS - 1 ? y1 : u2f(f2u(y1) & 0xFFFFE000u);
            pr[rt][PW * q + h] =
                __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_pkrtz(h0, h1));
            y0 -= h0;
            y1 -= h1;
          } else {
            const unsigned r =
                __builtin_bit_cast(unsigned, __builtin_convertvector(v2f{y0, y1}, v2bf));
            pr[rt][PW * q + h] = r;
            y0 -= u2f(r << 16);
            y1 -= u2f(r & 0xFFFF0000u);
          }
        }
      }
    }
  };

  auto prob = [&](int rt, int q) __attribute__((always_inline)) -> uint4 {
    // (float32 values: terms 0 twice, 1 twice, then 0 and 2.)
    if constexpr (VDT == kVF32)
      return make_uint4(pr[rt][q % 2 * 2], pr[rt][q % 2 * 2 + 1], pr[rt][q * 2 % 6],
                        pr[rt][q * 2 % 6 + 1]);
    return make_uint4(pr[rt][4 * q], pr[rt][4 * q + 1], pr[rt][4 * q + 2], pr[rt][4 * q + 3]);
  };
  auto product = [](uint4 x, uint4 y, v4f o) __attribute__((always_inline)) -> v4f {
    if constexpr (VDT == kVF16)
      return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x),
                                                    __builtin_bit_cast(v8h, y), o, 0, 0, 0);
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x),
                                                   __builtin_bit_cast(v8bf, y), o, 0, 0, 0);
  };
  auto add_values = [&](const Vals& f) __attribute__((always_inline)) {
    if constexpr (VDT != kVF32) {
      constexpr unsigned kOnes = VDT == kVF16 ? 0x3C003C00u : 0x3F803F80u;
      const uint4 ones = make_uint4(kOnes, kOnes, kOnes, kOnes);
#pragma unroll
      for (int q = 0; q < TERMS; ++q)
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) l_run[rt] = product(ones, prob(rt, q), l_run[rt]);
    }
#pragma unroll
    for (int t = 0; t < NA; ++t) {
      const int u = t / G::CPP, j = t % G::CPP;
      if constexpr (VDT == kVF32) {
        // A value is three bfloat16 terms of eight bits (cut off, so exactly), and of the
        // nine products with those of p the six above 2^-24 count, two a product of 32.
        unsigned x[4], tm[3][2];
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = f.w[0][i][u][j];
#pragma unroll
        for (int q = 0; q < 3; ++q) {
          tm[q][0] = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);
          tm[q][1] = __builtin_amdgcn_perm(x[3], x[2], 0x07060302u);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[i] = f2u(u2f(x[i]) - u2f(x[i] & 0xFFFF0000u));
        }
        const uint4 hi = make_uint4(tm[0][0], tm[0][1], tm[1][0], tm[1][1]);
        const uint4 lo = make_uint4(tm[2][0], tm[2][1], tm[0][0], tm[0][1]);
#pragma unroll
        for (int q = 0; q < 3; ++q)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt)
            acc[rt][t] = product(q < 2 ? hi : lo, prob(rt, q), acc[rt][t]);
      } else {
        const unsigned sel = j & 1 ? 0x07060302u : 0x05040100u;
        const uint4 av =
            make_uint4(__builtin_amdgcn_perm(f.w[0][1][u][j / 2], f.w[0][0][u][j / 2], sel),
                       __builtin_amdgcn_perm(f.w[0][3][u][j / 2], f.w[0][2][u][j / 2], sel),
                       __builtin_amdgcn_perm(f.w[CPS - 1][1][u][j / 2],
                                             f.w[CPS - 1][0][u][j / 2], sel),
                       __builtin_amdgcn_perm(f.w[CPS - 1][3][u][j / 2],
                                             f.w[CPS - 1][2][u][j / 2], sel));
#pragma unroll
        for (int q = 0; q < TERMS; ++q)
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) acc[rt][t] = product(av, prob(rt, q), acc[rt][t]);
      }
    }
  };

  if (i0 < i1) {
    const int steps = (it1 - it0) * spg;
    Keys kf;
    Vals vf;
    Meta cur, nxt;
    Scales sz0, szr;
    if (steps > 0) {
      cur = next_meta();
      nxt = next_meta();
      sz0 = load_sz(it0 + w);
      load_keys(cur, kf);
      load_values(cur, vf);
      szr = load_sz(it0 + kWaves + w);
    }
    // The row in slot order (zeros behind the last row), and as it is to LDS for the
    // drafts.
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) qv[i][k] = brow < live ? qv[i][k] : 0.f;
#pragma unroll
    for (int i = 0; i < SPT; ++i) {
      // Channel of slot i of eight, for a thread of the lower and of the upper four.
      auto of = [](int i) { return WIDE ? 2 * (i & 3) + (i >> 2) : 4 * (i & 1) + (i >> 1); };
      if constexpr (SPT >= 8) {
        qn[i] = qv[i / 8][of(i % 8)];
      } else {
        const unsigned up = part & 1 ? ~0u : 0u;
        qn[i] = u2f((f2u(qv[0][of(i + 4)]) & up) | (f2u(qv[0][of(i)]) & ~up));
      }
    }
    if (dr0 < dr1) {
#pragma unroll
      for (int i = 0; i < NQ; ++i) {
        float* dst = q_s + brow * G::AS + (part * SPT & ~7) + 8 * i;
        *reinterpret_cast<float4*>(dst) = make_float4(qv[i][0], qv[i][1], qv[i][2], qv[i][3]);
        *reinterpret_cast<float4*>(dst + 4) = make_float4(qv[i][4], qv[i][5], qv[i][6], qv[i][7]);
      }
    }
    if (steps > 0) stage_sz(sz0, it0 + w);
    __syncthreads();
    // (Every logit of such a row is infinite or NaN, and the row NaN.)
    unsigned big = 0;
#pragma unroll
    for (int i = 0; i < NQ; ++i)
#pragma unroll
      for (int k = 0; k < 8; ++k) big = max(big, f2u(qv[i][k]) & 0x7FFFFFFFu);
    if (big >= 0x7F800000u) wild_s[brow] = 1;
    if (steps > 0) {
      build(it0);
      int it = it0, p = 0;
      for (int done = 0; done < steps; ++done) {
        const int buf = (it - it0) & 1;
        if (p == 0) {
          __syncthreads();
          if (it + 1 < it1) build(it + 1);
          // Every kWaves items, a wave an item: of the next kWaves items the first is built
          // in the last of these, and the slots held items built before.
          if (((it - it0) & (kWaves - 1)) == 0) {
            stage_sz(szr, it + kWaves + w);
            szr = load_sz(it + 2 * kWaves + w);
          }
        }
        // Nibbles of key block kb of chunk e: as bytes, or (eight channels a block) as
        // float16, nib * 2^-18.
        constexpr int KB = WIDE ? NB : G::KW;
        auto key_op = [&](int e, int kb) __attribute__((always_inline)) -> v4i {
          if constexpr (WIDE) {
            const unsigned w0 = kf.w[e][2 * kb], w1 = kf.w[e][2 * kb + 1];
            return v4i{(int)(w0 & 0x0F0F0F0Fu), (int)((w0 >> 4) & 0x0F0F0F0Fu),
                       (int)(w1 & 0x0F0F0F0Fu), (int)((w1 >> 4) & 0x0F0F0F0Fu)};
          }
          const unsigned w0 = kf.w[e][kb];
          return v4i{(int)(w0 << 6 & 0x03C003C0u), (int)(w0 << 2 & 0x03C003C0u),
                     (int)(w0 >> 2 & 0x03C003C0u), (int)(w0 >> 6 & 0x03C003C0u)};
        };
        // With one row tile they are made where they are used (registers), with two
        // once for both, and the next keys are loaded over the words.
        v4i ak[CPS][KB];
        if constexpr (RT > 1) {
#pragma unroll
          for (int e = 0; e < CPS; ++e)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) ak[e][kb] = key_op(e, kb);
          load_keys(nxt, kf);
        }
        bool any = false, masked = false;
#pragma unroll
        for (int e = 0; e < CPS; ++e) {
          any |= cur.nval[e] > 0;
          masked |= (cur.nval[e] < 16) |
                    ((cur.tok0[e] < low_max) & (cur.tok0[e] + 16 > a.sinks));
        }
        if (any) {
          const uint8_t* dg = smem + buf * G::kDig + n16 * G::DS + grp * (D / 4 * G::TB);
          float s[RT][NS];
          if constexpr (WIDE) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              v4i ds[CPS][ND];
#pragma unroll
              for (int kb = 0; kb < KB; ++kb) {
                v4i kop[CPS];
#pragma unroll
                for (int e = 0; e < CPS; ++e) kop[e] = RT > 1 ? ak[e][kb] : key_op(e, kb);
#pragma unroll
                for (int k = 0; k < ND; ++k) {
                  const v4i bq = *reinterpret_cast<const v4i*>(
                      dg + (k * M + rt * 16) * G::DS + 16 * kb);
#pragma unroll
                  for (int e = 0; e < CPS; ++e)
                    ds[e][k] = __builtin_amdgcn_mfma_i32_16x16x64_i8(
                        kop[e], bq, kb == 0 ? v4i{0, 0, 0, 0} : ds[e][k], 0, 0, 0);
                }
              }
#pragma unroll
              for (int e = 0; e < CPS; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  s[rt][4 * e + i] =
                      __builtin_fmaf((float)((ds[e][3][i] << 8) + ds[e][2][i]), 65536.f,
                                     (float)((ds[e][1][i] << 8) + ds[e][0][i]));
            }
          } else {
            v4f ds[RT][CPS];
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
              v4i kop[CPS];
#pragma unroll
              for (int e = 0; e < CPS; ++e) kop[e] = RT > 1 ? ak[e][kb] : key_op(e, kb);
#pragma unroll
              for (int k = ND - 1; k >= 0; --k)
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                  const v4i bq = *reinterpret_cast<const v4i*>(
                      dg + (k * M + rt * 16) * G::DS + 16 * kb);
#pragma unroll
                  for (int e = 0; e < CPS; ++e)
                    ds[rt][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                        __builtin_bit_cast(v8h, kop[e]), __builtin_bit_cast(v8h, bq),
                        kb == 0 && k == ND - 1 ? v4f{0.f, 0.f, 0.f, 0.f} : ds[rt][e], 0, 0, 0);
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
              for (int k = 0; k < NS; ++k) s[rt][k] = ds[rt][k / 4][k % 4];
          }
          if constexpr (RT == 1) load_keys(nxt, kf);
          float c1[RT], cc[RT];
          unsigned vis[RT];
#pragma unroll
          for (int rt = 0; rt < RT; ++rt) {
            const float2 x = cc_s[buf][rt * 16 + n16];
            c1[rt] = x.x;
            cc[rt] = x.y;
            vis[rt] = 0;
          }
          if (masked) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
              const int low = low_s[rt * 16 + n16];
#pragma unroll
              for (int e = 0; e < CPS; ++e)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  const int k = 4 * grp + i, t = cur.tok0[e] + k;
                  vis[rt] |= (unsigned)((k < cur.nval[e]) & ((t < a.sinks) | (t >= low)))
                             << (4 * e + i);
                }
            }
          }
          softmax(s, c1, cc, masked, vis);
          // Keys that no row sees keep no value: a probability of zero times what lies
          // there (a chunk of none holds anything) would be NaN where that is not
          // finite.
          if (masked) {
#pragma unroll
            for (int e = 0; e < CPS; ++e)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int k = 4 * grp + i, t = cur.tok0[e] + k;
                const unsigned keep =
                    (k < cur.nval[e]) & ((t < a.sinks) | (t >= low_min)) ? ~0u : 0u;
#pragma unroll
                for (int u = 0; u < G::NP; ++u)
#pragma unroll
                  for (int x = 0; x < G::PB / 4; ++x) vf.w[e][i][u][x] &= keep;
              }
          }
        } else if constexpr (RT == 1) {
          load_keys(nxt, kf);
        }
        // The table entries of the step after the next: no LDS access, whose waits
        // would wait for them too, follows before the value products.
        const Meta ahead = next_meta();
        if (any) add_values(vf);
        load_values(nxt, vf);
        cur = nxt;
        nxt = ahead;
        if (++p == spg) {
          p = 0;
          ++it;
        }
      }
    }

    // ---- drafts: 16 of them a wave and item, float32 products ----
    // (All of an item's loads are in flight before its first product: one wait for
    // memory an item, at the end of a workgroup's chain.)
    const RowsArgs& a = late_args();
    for (int item = dr0; item < dr1; ++item) {
      const int j0 = (item * kWaves + w) * 16;
      const int nval = min(16, a.nodes - j0);
      if (nval <= 0) break;
      const uint8_t* vb = a.vd + (int64_t)b * a.vd_b + (int64_t)hk * a.vd_h + v_lane;
#pragma unroll
      for (int e = 0; e < CPS; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int u = 0; u < G::NP; ++u) {
            KVec<G::PB / 4> x = {};
            if (e == 0)
              x = load_k<G::PB / 4>(vb + (int64_t)(j0 + min(4 * grp + i, nval - 1)) * a.vd_n +
                                    16 * G::PB * u);
#pragma unroll
            for (int k = 0; k < G::PB / 4; ++k) vf.w[e][i][u][k] = x.w[k];
          }
      const float* kd = a.kd + (int64_t)b * a.kd_b + (int64_t)hk * a.kd_h +
                        (int64_t)(j0 + min(n16, nval - 1)) * a.kd_n + grp * (D / 4);
      float4 kx[D / 16];
#pragma unroll
      for (int d = 0; d < D / 16; ++d) kx[d] = *reinterpret_cast<const float4*>(kd + 4 * d);
      uint8_t mb[RT][4];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        const int R = row0 + min(rt * 16 + n16, live - 1);
        const int node = R - fdiv(R, a.div_nodes) * a.nodes;
        const uint8_t* mk = a.mask + (int64_t)b * a.mk_b + (int64_t)node * a.mk_i + j0;
#pragma unroll
        for (int k = 0; k < 4; ++k) mb[rt][k] = mk[min(4 * grp + k, nval - 1)];
      }
      __builtin_amdgcn_sched_barrier(0);
      v4f ds[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) ds[rt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int d = 0; d < D / 4; d += 4) {
        const float4 k4 = kx[d / 4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
          const float4 q4 = *reinterpret_cast<const float4*>(
              q_s + (rt * 16 + n16) * G::AS + grp * (D / 4) + d);
          ds[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4.x, q4.x, ds[rt], 0, 0, 0);
          ds[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4.y, q4.y, ds[rt], 0, 0, 0);
          ds[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4.z, q4.z, ds[rt], 0, 0, 0);
          ds[rt] = __builtin_amdgcn_mfma_f32_16x16x4f32(k4.w, q4.w, ds[rt], 0, 0, 0);
        }
      }
      float s[RT][NS], c1[RT], cc[RT];
      unsigned vis[RT];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt) {
        c1[rt] = kLog2e;
        cc[rt] = 0.f;
        vis[rt] = 0;
#pragma unroll
        for (int k = 0; k < NS; ++k) s[rt][k] = kLeast;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          vis[rt] |= (unsigned)((mb[rt][k] != 0) & (4 * grp + k < nval)) << k;
          s[rt][k] = ds[rt][k];
        }
        if (vis[rt]) seen_s[rt * 16 + n16] = 1;
      }
      softmax(s, c1, cc, true, vis);
      // Drafts that no row of the workgroup sees keep no value either (a batch of trees
      // may be padded with anything).
      unsigned any = vis[0];
      if constexpr (RT > 1) any |= vis[1];
      any |= xchg_u32<1>(any);
      any |= xchg_u32<2>(any);
      any |= xchg4(any);
      any |= xchg_u32<8>(any);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const unsigned keep = any >> i & 1u ? ~0u : 0u;
#pragma unroll
        for (int u = 0; u < G::NP; ++u)
#pragma unroll
          for (int x = 0; x < G::PB / 4; ++x) vf.w[0][i][u][x] &= keep;
      }
      add_values(vf);
    }
  }

  // The range again for every row by itself, a wave a row and key after key, for the
  // rare workgroup with a NaN or an overflow: a key that a row does not see takes no
  // part in it. (Masking the values of every product instead costs each step what this
  // costs such a workgroup alone.)
  auto plain_rows = [&]() {
    const RowsArgs& a = late_args();
    const DecodeArgs& c = a.c;
    const float* sbase = c.k_scale + (int64_t)b * c.s_b + (int64_t)hk * c.s_h;
    const float* zbase = c.k_zp + (int64_t)b * c.s_b + (int64_t)hk * c.s_h;
    const uint8_t* kbase = c.k_pages + (int64_t)hk * c.k_head;
    const int32_t* table = c.page_table ? c.page_table + (int64_t)b * c.pt_b : nullptr;
    const int group_rows = c.pages_per_group * c.page_rows;
    constexpr int CH = D / 64;
    float* part0 = reinterpret_cast<float*>(smem);
    __syncthreads();
    for (int i = tid; i < kWaves * M; i += NT) {
      m_s[i / M][i % M] = kLeast;
      l_s[i / M][i % M] = 0.f;
    }
    for (int i = tid; i < kWaves * M * G::AS; i += NT) part0[i] = 0.f;
    __syncthreads();
    for (int r = w; r < live; r += NT / 64) {
      if (wild_s[r]) continue;
      const int i = (row0 + r) % a.nodes;
      const int64_t q0 = (int64_t)b * c.q_b +
                         (int64_t)(hk * c.hq_per_kv + (row0 + r) / a.nodes) * c.q_h +
                         (int64_t)i * a.q_n + lane * CH;
      float q[CH], o[CH];
      for (int k = 0; k < CH; ++k) {
        q[k] = load_elem(c.q, q0 + k, c.q_dtype);
        o[k] = 0.f;
      }
      float m = kLeast, l = 0.f;
      auto key = [&](const float* k, const float* v) {
        float x = 0.f;
        for (int d = 0; d < CH; ++d) x = __builtin_fmaf(q[d], k[d], x);
        x = allreduce_sum<1, 64>(x) * kLog2e;
        const float mn = fmaxf(m, x);
        const float f = __builtin_amdgcn_exp2f(m - mn), p = __builtin_amdgcn_exp2f(x - mn);
        m = mn;
        l = __builtin_fmaf(l, f, p);
        for (int d = 0; d < CH; ++d) o[d] = __builtin_fmaf(o[d], f, p * v[d]);
      };
      for (int it = it0; it < it1; ++it) {
        const int g = group_of(it);
        for (int t = g * group_rows; t < min((g + 1) * group_rows, n); ++t) {
          if (t >= a.sinks && t < low_s[r]) continue;
          const int lp = fdiv(t, c.div_rows), tr = t - lp * c.page_rows;
          const int64_t phys = min(max(table ? table[lp] : lp, 0), c.num_pages - 1);
          const uint8_t* kp = kbase + phys * c.k_page + (int64_t)tr * c.k_row;
          const int64_t vo = phys * c.v_page + (int64_t)hk * c.v_head + (int64_t)tr * c.v_row;
          float k[CH], v[CH];
          for (int j = 0; j < CH; ++j) {
            const int d = lane * CH + j;
            const float s = sbase[(int64_t)g * c.s_g + d], z = zbase[(int64_t)g * c.s_g + d];
            k[j] = (float)((kp[d >> 1] >> (4 * (d & 1))) & 15) * s - z * s;
            v[j] = load_elem(c.v_pages, vo + d, VDT);
          }
          key(k, v);
        }
      }
      for (int j = dr0 * 64; j < min(dr1 * 64, a.nodes); ++j) {
        if (!a.mask[(int64_t)b * a.mk_b + (int64_t)i * a.mk_i + j]) continue;
        const float* kd = a.kd + (int64_t)b * a.kd_b + (int64_t)hk * a.kd_h + (int64_t)j * a.kd_n;
        const uint8_t* vd = a.vd + (int64_t)b * a.vd_b + (int64_t)hk * a.vd_h + (int64_t)j * a.vd_n;
        float v[CH];
        for (int d = 0; d < CH; ++d) v[d] = load_elem(vd, lane * CH + d, VDT);
        key(kd + lane * CH, v);
      }
      for (int k = 0; k < CH; ++k) part0[r * G::AS + lane * CH + k] = o[k];
      if (lane == 0) {
        m_s[0][r] = m;
        l_s[0][r] = l;
      }
    }
    __syncthreads();
  };

  // ---- the waves' parts ----
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const float l = VDT == kVF32 ? over_groups_sum(l_run[rt][0]) : l_run[rt][0];
    if (grp == 0) {
      m_s[w][rt * 16 + n16] = m_run[rt];
      l_s[w][rt * 16 + n16] = l;
    }
  }
  __syncthreads();                                 // (the terms are no longer read)
  float* out_w = reinterpret_cast<float*>(smem) + w * M * G::AS;
  float any_nan = 0.f;
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    const int r = rt * 16 + n16;
    float top = m_s[0][r];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, m_s[i][r]);
    const float f = __builtin_amdgcn_exp2f(m_run[rt] - top);
    const bool wild = wild_s[r];
#pragma unroll
    for (int u = 0; u < G::NP; ++u)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float* dst = out_w + r * G::AS + u * 16 * G::CPP + (4 * grp + i) * G::CPP;
#pragma unroll
        for (int j = 0; j < G::CPP; j += 4) {
          const int t = u * G::CPP + j;
          const float4 x = make_float4(acc[rt][t][i] * f, acc[rt][t + 1][i] * f,
                                       acc[rt][t + 2][i] * f, acc[rt][t + 3][i] * f);
          *reinterpret_cast<float4*>(dst + j) = x;
          any_nan += wild ? 0.f : (x.x + x.y) + (x.z + x.w);
        }
      }
  }
  if (!(any_nan - any_nan == 0.f)) bad_s = 1;      // (NaN, or beyond float32)
  __syncthreads();
  if (bad_s) plain_rows();
  const float* parts = reinterpret_cast<const float*>(smem);
  const RowsArgs& za = late_args();
  const DecodeArgs& zc = za.c;
  const int64_t o0 =
      ((int64_t)b * zc.num_q_heads + (int64_t)hk * zc.hq_per_kv) * za.nodes + row0;
  for (int idx = tid * 4; idx < live * D; idx += NT * 4) {
    const int r = idx / D, d = idx % D;
    float top = m_s[0][r];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = fmaxf(top, m_s[i][r]);
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
      l = __builtin_fmaf(__builtin_amdgcn_exp2f(m_s[i][r] - top), l_s[i][r], l);
      const float4 x = *reinterpret_cast<const float4*>(parts + (i * M + r) * G::AS + d);
      o.x += x.x;
      o.y += x.y;
      o.z += x.z;
      o.w += x.w;
    }
    if (wild_s[r]) {
      l = 0.f;
      o = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    // (No finite logit, hence no probability: zero where the row sees nothing, otherwise
    // NaN, 0 / 0 as in the formula.)
    const bool none = l == 0.f, seen = seen_s[r];
    if (zc.final_out) {
      const float os[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        store_elem(zc.out, (o0 + r) * D + d + k, zc.out_dtype,
                   none && !seen ? 0.f : os[k] / l);
    } else {
      const int64_t pi = (o0 + r) * zc.num_splits + split;
      *reinterpret_cast<float4*>(zc.ws_acc + pi * D + d) = o;
      if (d == 0) {
        zc.ws_ml[2 * pi] = !none  ? (double)top * 0.6931471805599453
                           : seen ? kNoFinite
                                  : -INFINITY;
        zc.ws_ml[2 * pi + 1] = (double)l;
      }
    }
  }
}

hipError_t launch_decode_rows(const RowsArgs& a, int D, int v_dtype, int batch, hipStream_t st) {
  const int64_t wgs = (int64_t)a.tiles * a.c.num_splits * (a.c.num_q_heads / a.c.hq_per_kv) *
                      batch;
  if (!grid_fits(wgs, kWaves * 64)) return hipErrorInvalidValue;
  const bool wide = a.c.out_dtype == kEF32;
  const bool stream = a.tiles == 1;
#define FDI4_RW(DD, VV, RR, OO, SS)                                                       \
  if (D == DD && v_dtype == VV && a.row_tiles == RR && wide == OO && stream == SS) {      \
    hipLaunchKernelGGL((decode_rows_kernel<DD, VV, RR, OO, SS>), dim3((unsigned)wgs),      \
                       dim3(kWaves * 64), 0, st, a);                                      \
    return hipGetLastError();                                                             \
  }
#define FDI4_RW_V(DD, RR, SS) \
  FDI4_RW(DD, kVF32, RR, false, SS) FDI4_RW(DD, kVF16, RR, false, SS) \
  FDI4_RW(DD, kVBF16, RR, false, SS) FDI4_RW(DD, kVF32, RR, true, SS) \
  FDI4_RW(DD, kVF16, RR, true, SS) FDI4_RW(DD, kVBF16, RR, true, SS)
  FDI4_RW_V(64, 1, true) FDI4_RW_V(64, 2, true) FDI4_RW_V(64, 2, false)
  FDI4_RW_V(128, 1, true) FDI4_RW_V(128, 2, true) FDI4_RW_V(128, 2, false)
  FDI4_RW_V(256, 1, true) FDI4_RW_V(256, 1, false)
#undef FDI4_RW_V
#undef FDI4_RW
  return hipErrorInvalidValue;
}

}  // namespace fdi4
