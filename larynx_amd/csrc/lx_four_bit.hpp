// Four-bit codes as MFMA operands (lx_q4.hip, lx_kv4.hip).
//
// A dword holds the eight codes of one lane's bf16 fragment (v_mfma_f32_16x16x32_bf16: lane l
// holds row or column l % 16, k = (l / 16) * 8 .. + 7).  Code q becomes the bf16 number 16 + q,
// whose four low bits of significance lie at bits 3..6 above the pattern of 16.0 (0x4180): the
// codes of elements 2r and 2r + 1 are stored at bits 3 + 4r and 19 + 4r (mod 32), so one rotate
// and one and-or make both halves of fragment register r, 7 instructions for eight codes.
// (A signed bf16 number costs a subtraction that gfx950 has no packed bf16 form of.)  What the
// codes stand for is affine in q, so the 16 goes into a constant of the group; it is at most
// half of a code's magnitude, which costs under one bit of the fp32 sums.
#pragma once

#include "lx_gemm_common.hpp"

namespace lx {

typedef unsigned short ushortx4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ unsigned rotr32(unsigned w, int r) {
  return __builtin_amdgcn_alignbit(w, w, r);
}

// The fragment of a dword: element j is 16 + code j.
__device__ __forceinline__ sbf16x8 q4_frag(unsigned w) {
  const uintx4_t f = {(w & 0x00780078u) | 0x41804180u, ((w >> 4) & 0x00780078u) | 0x41804180u,
                      ((w >> 8) & 0x00780078u) | 0x41804180u,
                      (rotr32(w, 12) & 0x00780078u) | 0x41804180u};
  return __builtin_bit_cast(sbf16x8, f);
}

// Bit position of element j's code.
__device__ __forceinline__ int q4_shift(int j) { return (3 + 4 * (j >> 1) + 16 * (j & 1)) & 31; }
// Code q (< 16) at its bits in the dword (element 7's wrap around).
__device__ __forceinline__ unsigned q4_put(unsigned q, int j) {
  const int s = q4_shift(j);
  return s > 28 ? (q << s) | (q >> (32 - s)) : q << s;
}
__device__ __forceinline__ unsigned q4_get(unsigned w, int j) {
  return rotr32(w, q4_shift(j)) & 15u;
}

// x as the sum of three bf16 numbers (exact for normal x: 24 significant bits); contraction
// off, as in pack2_bf16.
__device__ __forceinline__ void split3(const float (&x)[8], sbf16x8 (&p)[3]) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    floatx4 v = {x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]};
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      const bf16x4_t h = __builtin_convertvector(v, bf16x4_t);
#pragma unroll
      for (int j = 0; j < 4; ++j) p[i][4 * e + j] = h[j];
      if (i < 2) v = v - bf16x4_back(h);
    }
  }
}

__device__ __forceinline__ floatx4 mfma_bf16(sbf16x8 a, sbf16x8 b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// fp32 bits of the bf16 in the low or high half of a dword.
__device__ __forceinline__ float bf16_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

}  // namespace lx
