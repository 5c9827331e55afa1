// Row arithmetic of the paged append, shared by the kernels that write K and V
// rows into the cache: where a row's bytes go, and the K rotation, RTN int8 and
// 3-bit Lloyd-Max codec over rows that sit on D / 16 lanes (several rows per
// wave) or on a whole wave.
#pragma once

#include "s8kv_device.h"

namespace s8kv {

// Where a row's bytes go: through the tensor's buffer descriptor at a 32-bit
// offset (per-layer tensors up to 4 GiB), or through a 64-bit pointer (the
// <.., BIG> kernels, a tensor past 4 GiB; rows are checked against the pool
// before any store).  `off` is relative to the row's first byte.
struct BufOut {
  rsrc_t r;
  uint32_t base;
  __device__ void st128(uint32_t off, u32x4_t v) const { bstore128(v, r, base + off); }
  __device__ void st32(uint32_t off, uint32_t v) const { bstore32(v, r, base + off); }
  __device__ void st8(uint32_t off, uint8_t v) const { bstore8(v, r, base + off); }
};
struct PtrOut {
  char* p;
  __device__ void st128(uint32_t off, u32x4_t v) const { *reinterpret_cast<u32x4_t*>(p + off) = v; }
  __device__ void st32(uint32_t off, uint32_t v) const { *reinterpret_cast<uint32_t*>(p + off) = v; }
  __device__ void st8(uint32_t off, uint8_t v) const { p[off] = (char)v; }
};
template <bool BIG>
__device__ __forceinline__ auto row_out(void* base, uint32_t bytes, uint64_t off) {
  if constexpr (BIG)
    return PtrOut{static_cast<char*>(base) + off};
  else
    return BufOut{make_rsrc(base, bytes), (uint32_t)off};
}

// Per-row RTN int8 of the wave's row; writes D bytes at `byte_off` and the scale.
template <int D, class QOut, class SOut>
__device__ __forceinline__ void rtn_store_row(const float (&y)[RowLayout<D>::E], int lane, const QOut& qout,
                                              const SOut& sout) {
  constexpr int E = RowLayout<D>::E;
  int q[E];
  const float scale = rtn_row<D>(y, q);
  if (lane < RowLayout<D>::ACTIVE) {
#pragma unroll
    for (int j = 0; j < E; ++j) qout.st8((uint32_t)(lane + 64 * j), (uint8_t)(int8_t)q[j]);
  }
  if (lane == 0) sout.st32(0u, __builtin_bit_cast(uint32_t, scale));
}

// Several rows per wave: a row's D values sit on LPR = D/16 lanes, 16
// consecutive values per lane, so each lane moves a row part with two 16-byte
// loads and one 16-byte store per tensor and the per-row work (slot lookup,
// addresses, reductions) is shared by 64/LPR rows per instruction.  The K rotation runs the FWHT stages h = 1, 2, 4, 8 in-lane
// and h = 16 .. D/2 across the row's lanes: the stage order and arithmetic of
// fwht_row, so the bytes equal the one-row-per-wave kernel's.  Needs 16-byte
// aligned K and V rows.
//
// Lane placement: part li (values 16 li .. 16 li + 15) of a row.  At head_dim
// 128 li sits on lane bits (b3 b1 b0) and lane bits (b5 b4 b2) number the row,
// so the partners of the three cross-lane stages (li ^ 1, ^ 2, ^ 4) are lanes
// ^ 1, ^ 2, ^ 8, all DPP sources.  Other head dims: li = lane % LPR.
template <int D>
struct RowsLayout {
  static constexpr int LPR = D / 16;   // lanes per row
  static constexpr int RPW = 64 / LPR;  // rows per wave
  static constexpr int LANE4 = D == 128 ? 8 : 4;  // lane xor of part xor 4
  static __device__ __forceinline__ int part(int lane) {
    return D == 128 ? (lane & 3) | ((lane >> 1) & 4) : lane % LPR;
  }
  static __device__ __forceinline__ int row(int lane) {
    return D == 128 ? ((lane >> 2) & 1) | ((lane >> 3) & 6) : lane / LPR;
  }
};

// max over the row's lanes (part xor 1, 2, 4, 8)
template <int D>
__device__ __forceinline__ float rows_max(float v) {
  constexpr int LPR = D / 16;
  if constexpr (LPR > 1) v = fmaxf(v, xor_partner<1>(v));
  if constexpr (LPR > 2) v = fmaxf(v, xor_partner<2>(v));
  if constexpr (LPR > 4) v = fmaxf(v, xor_partner<RowsLayout<D>::LANE4>(v));
  if constexpr (LPR > 8) v = fmaxf(v, xor_partner<8>(v));
  return v;
}

#define S8KV_FMAC_DPP16(CTRL)                                                         \
  "s_nop 1\n"                                                                         \
  "v_fmac_f32_dpp %0, %0, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %1, %1, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %2, %2, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %3, %3, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %4, %4, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %5, %5, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %6, %6, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %7, %7, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %8, %8, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %9, %9, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                  \
  "v_fmac_f32_dpp %10, %10, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                \
  "v_fmac_f32_dpp %11, %11, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                \
  "v_fmac_f32_dpp %12, %12, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                \
  "v_fmac_f32_dpp %13, %13, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                \
  "v_fmac_f32_dpp %14, %14, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                \
  "v_fmac_f32_dpp %15, %15, %16 " CTRL " row_mask:0xf bank_mask:0xf\n"                \
  "s_nop 1"

// One cross-lane FWHT stage over the lane's 16 values, sign-tracked: z += t *
// (z of lane ^ M), t = -1 on the lanes whose part has the stage's bit set,
// else +1.  The lanes hold sigma * (true values), sigma = (-1)^(number of
// earlier stage bits set in the part); partners share sigma, so this is the
// butterfly on the true values (low lane a + b, high lane a - b) with the
// high lanes' sign flipped: RN(b - a) = -RN(a - b), and signed zeros aside
// (a zero quantizes to code 0 either way) the values are the untracked
// form's.  M = 1, 2, 8: one v_fmac_f32 with a DPP source per value (the s_nop
// pairs cover the DPP read-after-VALU-write hazard at the block's edges);
// M = 4 reads the partner through the LDS swizzle.
template <int M>
__device__ __forceinline__ void fwht_stage_tracked(float (&z)[16], float t) {
  if constexpr (M == 4) {
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = __builtin_fmaf(xor_partner<4>(z[i]), t, z[i]);
  } else {
    static_assert(M == 1 || M == 2 || M == 8, "DPP partners: lane ^ 1, ^ 2, ^ 8");
#define S8KV_FMAC_OPERANDS                                                                                       \
  : "+v"(z[0]), "+v"(z[1]), "+v"(z[2]), "+v"(z[3]), "+v"(z[4]), "+v"(z[5]), "+v"(z[6]), "+v"(z[7]), "+v"(z[8]), \
    "+v"(z[9]), "+v"(z[10]), "+v"(z[11]), "+v"(z[12]), "+v"(z[13]), "+v"(z[14]), "+v"(z[15])                    \
  : "v"(t)
    if constexpr (M == 1) asm(S8KV_FMAC_DPP16("quad_perm:[1,0,3,2]") S8KV_FMAC_OPERANDS);
    else if constexpr (M == 2) asm(S8KV_FMAC_DPP16("quad_perm:[2,3,0,1]") S8KV_FMAC_OPERANDS);
    else asm(S8KV_FMAC_DPP16("row_ror:8") S8KV_FMAC_OPERANDS);
#undef S8KV_FMAC_OPERANDS
  }
}
#undef S8KV_FMAC_DPP16

template <int D, class QOut, class SOut>
__device__ __forceinline__ void rows_rtn_store(const float (&y)[16], bool live, int li, const QOut& qout,
                                               const SOut& sout) {
  float amax = 0.0f;
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(y[i]));
  amax = rows_max<D>(amax);
  const float scale = amax / 127.0f;
  const float rscale = rtn_rscale(scale);
  uint32_t w[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    w[k] = pack_low_bytes(rtn_i8_biased(y[4 * k], scale, rscale), rtn_i8_biased(y[4 * k + 1], scale, rscale),
                          rtn_i8_biased(y[4 * k + 2], scale, rscale), rtn_i8_biased(y[4 * k + 3], scale, rscale));
  }
  if (live) {
    qout.st128((uint32_t)li * 16u, u32x4_t{w[0], w[1], w[2], w[3]});
    if (li == 0) sout.st32(0u, __builtin_bit_cast(uint32_t, scale));
  }
}

// 2 w + b in one add with carry-in (the lanes' b as a wave mask).
__device__ __forceinline__ uint32_t shift_in_bit(uint32_t w, bool b) {
  const uint64_t m = __builtin_amdgcn_ballot_w64(b);
  uint32_t r;
  uint64_t carry_out;
  asm("v_addc_co_u32_e64 %0, %1, %2, %2, %3" : "=v"(r), "=s"(carry_out) : "v"(w), "s"(m));
  return r;
}

// Ordered key of an fp32 bit pattern: key(x) < key(y) iff x < y, with -0
// just below +0; the map is its own inverse.
__device__ __forceinline__ int f32_key(int bits) { return bits ^ ((bits >> 31) & 0x7FFFFFFF); }

// Threshold T of the codebook neighbours a = c_{j-1} < b = c_j: the least
// fp32 u for which entry j is strictly nearer than entry j - 1 (fabsf(u - b) <
// fabsf(u - a), lloyd3_search's test).  On [a, b] the two distances are
// RN(b - u), non-increasing in u, and RN(u - a), non-decreasing, so the test
// is monotone there -- false at a, true at b -- and bisection over the keys
// finds T.  Below a the test is false (RN(b - u) >= RN(a - u)) and above b,
// for a codebook accepted by lloyd3_search_ok and |u| <= 1, true; so for
// every u the encoder sees, the test equals u >= T.  (T is never +0: -0 gives
// the same distances and precedes it.)
__device__ __forceinline__ float lloyd3_threshold(float a, float b) {
  int lo = f32_key(__builtin_bit_cast(int, a)), hi = f32_key(__builtin_bit_cast(int, b));
  for (int it = 0; it < 32; ++it) {
    const uint32_t d = (uint32_t)hi - (uint32_t)lo;
    if (d <= 1u) break;
    const int mid = (int)((uint32_t)lo + (d >> 1));
    const float u = __builtin_bit_cast(float, f32_key(mid));
    if (fabsf(u - b) < fabsf(u - a)) hi = mid;
    else lo = mid;
  }
  return __builtin_bit_cast(float, f32_key(hi));
}

// 3-bit Lloyd-Max V of the lane's 16 values (head_dim 128 or 256, blocks of
// 128 = 8 lanes): the block's L2 norm adds the fp32 squares in the order of
// lloydmax3_encode_row (a pairwise tree over neighbours: levels h = 1 .. 8
// in-lane, h = 16, 32, 64 across the parts ^ 1, ^ 2, ^ 4), correctly rounded
// sqrt; u = v / norm (0 for a zero norm) as the Markstein quotient from the
// block's reciprocal, which equals the IEEE quotient for an fp16 v and any
// fp32 norm (checked for every pair of significands); code = first index
// minimising |u - c_j|: with `search` (a codebook accepted by
// lloyd3_search_ok) lloyd3_search's three tests as compares against the
// thresholds thr[j] = T_j, else the sequential scan.  Parts 2g and 2g + 1
// (lanes l and l ^ 1) hold elements 32g .. 32g + 31: each builds 16 bits of
// the three bit-plane words 3g + b, and the even part stores them.  THR false:
// no thresholds (finding them takes a workgroup longer than a row or two):
// lloyd3_search's own tests.
template <int D, bool THR = true, class VOut, class NOut>
__device__ __forceinline__ void rows_lloydmax3_store(const float (&x)[16], bool live, int li, bool search,
                                                     const float (&cb)[8], const float (&thr)[8], const VOut& vout,
                                                     const NOut& nout) {
  float s[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) s[i] = x[i] * x[i];
#pragma unroll
  for (int h = 1; h < 16; h <<= 1) {
#pragma unroll
    for (int i = 0; i < 16; i += 2 * h) s[i] = s[i] + s[i + h];
  }
  float t = s[0];  // the lane's 16 elements; partners hold the neighbouring groups
  t = t + xor_partner<1>(t);
  t = t + xor_partner<2>(t);
  t = t + xor_partner<RowsLayout<D>::LANE4>(t);
  const float nrm = __builtin_sqrtf(t);
  const float rn = rtn_rscale(nrm);  // 1 / norm, 0 for a zero norm (then u = 0)
  float u[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float q0 = materialize(x[i] * rn);
    const float r = __builtin_fmaf(-q0, nrm, x[i]);
    u[i] = __builtin_fmaf(r, rn, q0);
  }
  // bit i of pw[b] = bit b of element i's code (elements shifted in from 15 down)
  uint32_t pw[3] = {0u, 0u, 0u};
  if (search) {
#pragma unroll
    for (int i = 15; i >= 0; --i) {
      bool b2, b1, b0;
      if constexpr (THR) {
        b2 = u[i] >= thr[4];
        b1 = u[i] >= (b2 ? thr[6] : thr[2]);
        const float t_hi = b2 ? thr[7] : thr[3], t_lo = b2 ? thr[5] : thr[1];
        b0 = u[i] >= (b1 ? t_hi : t_lo);
      } else {
        lloyd3_search(u[i], cb, b2, b1, b0);
      }
      pw[0] = shift_in_bit(pw[0], b0);
      pw[1] = shift_in_bit(pw[1], b1);
      pw[2] = shift_in_bit(pw[2], b2);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float best = fabsf(u[i] - cb[0]);
      uint32_t c = 0;
#pragma unroll
      for (int j = 1; j < 8; ++j) {
        const float d = fabsf(u[i] - cb[j]);
        if (d < best) {
          best = d;
          c = (uint32_t)j;
        }
      }
#pragma unroll
      for (int b = 0; b < 3; ++b) pw[b] |= ((c >> b) & 1u) << i;
    }
  }
  uint32_t w[3];
#pragma unroll
  for (int b = 0; b < 3; ++b) {
    const uint32_t odd = (uint32_t)__builtin_amdgcn_mov_dpp((int)pw[b], 0xB1, 0xF, 0xF, false);  // lane ^ 1
    w[b] = pw[b] | (odd << 16);
  }
  if (live && (li & 1) == 0) {
#pragma unroll
    for (int b = 0; b < 3; ++b) vout.st32((uint32_t)(li / 2) * 12u + 4u * b, w[b]);
  }
  if (live && (li & 7) == 0) nout.st32((uint32_t)(li / 8) * 4u, __builtin_bit_cast(uint32_t, nrm));
}

// The K rotation of the lane's 16 values: fp32 FWHT, one multiply by
// 1/sqrt(D), RNE to fp16.  Holds the lane's sign-tracking constants: the stage
// multipliers, and the final sign (-1)^popcount(li) folded into the multiply.
template <int D>
struct RowsHadamard {
  float t1, t2, t4, t8, srn;
  __device__ __forceinline__ RowsHadamard(int li, float rot_norm)
      : t1((li & 1) ? -1.0f : 1.0f),
        t2((li & 2) ? -1.0f : 1.0f),
        t4((li & 4) ? -1.0f : 1.0f),
        t8((li & 8) ? -1.0f : 1.0f),
        srn((__builtin_popcount(li) & 1) ? -rot_norm : rot_norm) {}
  __device__ __forceinline__ void operator()(float (&x)[16]) const {
    constexpr int LPR = RowsLayout<D>::LPR;
#pragma unroll
    for (int hs = 1; hs < 16; hs <<= 1) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        if ((i & hs) == 0) {
          const float p0 = x[i], p1 = x[i + hs];
          x[i] = p0 + p1;
          x[i + hs] = p0 - p1;
        }
      }
    }
    if constexpr (LPR > 1) fwht_stage_tracked<1>(x, t1);
    if constexpr (LPR > 2) fwht_stage_tracked<2>(x, t2);
    if constexpr (LPR > 4) fwht_stage_tracked<RowsLayout<D>::LANE4>(x, t4);
    if constexpr (LPR > 8) fwht_stage_tracked<8>(x, t8);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = (float)(_Float16)materialize(x[i] * srn);
  }
};

}  // namespace s8kv
