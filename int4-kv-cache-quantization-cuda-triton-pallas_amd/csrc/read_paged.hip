// Rows of the paged INT4 cache back as dense tensors (gfx950): for token t in
// [start_b, start_b + length) of sequence b
//   k[b, h, t - start_b, d] = q*s - zp*s     (two rounded float32 products and a
//                                             rounded difference, then one rounding
//                                             to the output type)
//   v[b, h, t - start_b, d] = the stored value, converted
// and zeros behind the sequence's end. The arithmetic is that of
// dequant_kernel (reference src/quantize_int4_ref.py:87-136).
//
// A workgroup takes up to RPS * kReadRows rows of one scale group of one (sequence,
// kv-head): a thread owns eight channels, whose scales it loads once, of kReadRows
// rows, all of whose loads are in flight together (page-table entries, then codes and
// values). Bound by memory: every byte is read once and written once, 5.4 TB/s over 440
// MB of bfloat16 (81 us; a copy of 256 MB runs at 5.5). One row a thread at a time, and
// a workgroup for the whole group, took 85 us there, 31 us against 25 for 1000 tokens
// of 8 sequences (85 MB, to float32) and 15 against 10 for 16 sequences' open groups.

#include <algorithm>

#include "decode_common.hpp"

namespace fdi4 {

constexpr int kReadThreads = 256;

// Eight consecutive elements of type OUT at p.
template <int OUT>
__device__ __forceinline__ void store8(uint8_t* p, const float* x) {
  if constexpr (OUT == kEF32) {
    st16_stream(p, U32x4{f2u(x[0]), f2u(x[1]), f2u(x[2]), f2u(x[3])});
    st16_stream(p + 16, U32x4{f2u(x[4]), f2u(x[5]), f2u(x[6]), f2u(x[7])});
  } else {
    unsigned w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      unsigned lo, hi;
      if constexpr (OUT == kEF16) {
        lo = __builtin_bit_cast(unsigned short, (_Float16)x[2 * k]);
        hi = __builtin_bit_cast(unsigned short, (_Float16)x[2 * k + 1]);
      } else {
        lo = bf16_rne(x[2 * k]);
        hi = bf16_rne(x[2 * k + 1]);
      }
      w[k] = lo | hi << 16;
    }
    st16_stream(p, U32x4{w[0], w[1], w[2], w[3]});
  }
}

constexpr int kReadRows = 4;

template <int D, int VDT, int OUT>
__global__ __launch_bounds__(kReadThreads) void read_paged_kernel(ReadArgs a, int slots,
                                                                  int heads) {
  constexpr int TPR = D / 8;                  // threads per row
  constexpr int RPS = kReadThreads / TPR;     // rows per sweep
  constexpr int U = kReadRows;
  constexpr int VEB = VDT == kVF32 ? 4 : 2;
  constexpr int OEB = OUT == kEF32 ? 4 : 2;
  constexpr int VL = VDT == kVF32 ? 2 : 1;    // 16-byte value loads per row
  const DecodeArgs& c = a.c;
  unsigned wi = blockIdx.x;
  const int slot = (int)(wi % (unsigned)slots);
  wi /= (unsigned)slots;
  const int h = (int)(wi % (unsigned)heads), b = (int)(wi / (unsigned)heads);
  const int cap = c.max_pages * c.page_rows;
  const int G = c.pages_per_group * c.page_rows;
  const int start = a.start ? min(max(a.start[b], 0), cap) : a.start0;
  const int T = seq_len_of(c, b);
  // Rows of this workgroup: a piece of a group, the slot-th from the one that holds the
  // range's start, within the range (64 bits: a range may end anywhere), counted from
  // its start.
  const unsigned pieces = ((unsigned)G + RPS * U - 1) / (RPS * U);
  const unsigned at = (unsigned)(start % G) / (RPS * U) + (unsigned)slot;
  const int g = start / G + (int)(at / pieces);
  const int64_t p0 = (int64_t)g * G + (int64_t)(at % pieces) * (RPS * U);
  const int64_t p1 = min(p0 + RPS * U, (int64_t)(g + 1) * G);
  const int i0 = (int)max(p0 - start, (int64_t)0);
  const int i1 = (int)min(p1 - start, (int64_t)a.length);
  if (i0 >= i1) return;
  const int tid = threadIdx.x, oct = tid % TPR, rsub = tid / TPR;
  uint8_t* ko = reinterpret_cast<uint8_t*>(a.k_out) +
                ((int64_t)b * a.ko_b + (int64_t)h * a.ko_h + 8 * oct) * OEB;
  uint8_t* vo = reinterpret_cast<uint8_t*>(a.v_out) +
                ((int64_t)b * a.vo_b + (int64_t)h * a.vo_h + 8 * oct) * OEB;
  float k[8], v[8];
  if (start + (int64_t)i0 >= T) {
#pragma unroll
    for (int j = 0; j < 8; ++j) k[j] = 0.f;
    for (int i = i0 + rsub; i < i1; i += RPS) {
      store8<OUT>(ko + (int64_t)i * a.ko_t * OEB, k);
      store8<OUT>(vo + (int64_t)i * a.vo_t * OEB, k);
    }
    return;
  }
  // Rows past the range or the sequence load the last valid one.
  // (Sums of positions as unsigned: a capacity may be any 31-bit number.)
  const unsigned s0 = (unsigned)start;
  const unsigned last = min(s0 + (unsigned)i1, (unsigned)T) - 1;
  unsigned q[U];
  U32x4 x[U][VL];
  int phys[U], row[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int t = (int)min(s0 + (unsigned)(i0 + rsub + u * RPS), last);
    const int lp = fdiv(t, c.div_rows);
    row[u] = t - lp * c.page_rows;
    phys[u] = c.page_table ? c.page_table[(int64_t)b * c.pt_b + lp] : lp;
  }
  float s[8], zs[8];
  const int64_t so = (int64_t)b * c.s_b + (int64_t)h * c.s_h + (int64_t)g * c.s_g + 8 * oct;
  widen_values<kVF32>(ld16(c.k_scale + so), s);
  widen_values<kVF32>(ld16(c.k_scale + so + 4), s + 4);
  widen_values<kVF32>(ld16(c.k_zp + so), zs);
  widen_values<kVF32>(ld16(c.k_zp + so + 4), zs + 4);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t p = min(max(phys[u], 0), c.num_pages - 1);
    q[u] = __builtin_nontemporal_load(reinterpret_cast<const unsigned*>(
        c.k_pages + p * c.k_page + (int64_t)h * c.k_head + (int64_t)row[u] * c.k_row + 4 * oct));
    const uint8_t* vp = reinterpret_cast<const uint8_t*>(c.v_pages) +
                        (p * c.v_page + (int64_t)h * c.v_head + (int64_t)row[u] * c.v_row +
                         8 * oct) * VEB;
#pragma unroll
    for (int i = 0; i < VL; ++i) x[u][i] = ld16_stream(vp + 16 * i);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) zs[j] = __fmul_rn(zs[j], s[j]);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int i = i0 + rsub + u * RPS;
    if (i >= i1) continue;
    const bool there = s0 + (unsigned)i < (unsigned)T;
#pragma unroll
    for (int w = 0; w < VL; ++w) widen_values<VDT>(x[u][w], v + w * 4);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      k[j] = __fsub_rn(__fmul_rn((float)((q[u] >> (4 * j)) & 15u), s[j]), zs[j]);
      k[j] = there ? k[j] : 0.f;
      v[j] = there ? v[j] : 0.f;
    }
    store8<OUT>(ko + (int64_t)i * a.ko_t * OEB, k);
    store8<OUT>(vo + (int64_t)i * a.vo_t * OEB, v);
  }
}

hipError_t launch_read_paged(const ReadArgs& a, int D, int v_dtype, int batch, int heads,
                             hipStream_t st) {
  if (batch == 0 || heads == 0 || a.length == 0) return hipSuccess;
  const int64_t G = (int64_t)a.c.pages_per_group * a.c.page_rows;
  const int per = kReadThreads / (D / 8) * kReadRows;
  // Pieces that the range touches: of its groups' pieces as many as begin in it, at most
  // one per `per` rows and one per further group, and the one that holds its start.
  // (Counted from this start, or the most from any.)
  const int64_t pieces = (G + per - 1) / per;
  int64_t slots;
  if (a.start) {
    const int64_t groups = ((int64_t)a.length + 2 * G - 2) / G;
    slots = std::min(groups * pieces, (a.length - 1) / per + 1 + groups);
  } else {
    const int64_t last = a.start0 + (int64_t)a.length - 1;
    slots = (last / G - a.start0 / G) * pieces + last % G / per - a.start0 % G / per + 1;
  }
  const int64_t items = slots * heads * batch;
  if (!grid_fits(items, kReadThreads)) return hipErrorInvalidValue;
#define FDI4_RD(DD, VV, OO)                                                               \
  if (D == DD && v_dtype == VV && a.out_dtype == OO) {                                    \
    hipLaunchKernelGGL((read_paged_kernel<DD, VV, OO>), dim3((unsigned)items),            \
                       dim3(kReadThreads), 0, st, a, (int)slots, heads);     \
    return hipGetLastError();                                                             \
  }
#define FDI4_RD_O(DD, VV) FDI4_RD(DD, VV, kEF32) FDI4_RD(DD, VV, kEF16) FDI4_RD(DD, VV, kEBF16)
#define FDI4_RD_V(DD) FDI4_RD_O(DD, kVF32) FDI4_RD_O(DD, kVF16) FDI4_RD_O(DD, kVBF16)
  FDI4_RD_V(64) FDI4_RD_V(128) FDI4_RD_V(256)
#undef FDI4_RD_V
#undef FDI4_RD_O
#undef FDI4_RD
  return hipErrorInvalidValue;
}

}  // namespace fdi4
