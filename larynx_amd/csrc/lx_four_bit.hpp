// Four-bit codes as MFMA operands (lx_q4.hip, lx_kv4.hip).
//
// A dword holds the eight codes of one lane's fp16 fragment (v_mfma_f32_16x16x32_f16: lane l holds
// row or column l % 16, k = (l / 16) * 8 .. + 7), elements 2r and 2r + 1 at bits 4r and 16 + 4r.
// An and-or with the pattern of 1024.0 makes both halves of a fragment register 1024 + q or 1024 +
// 16 q, a packed fp16 add or fma makes them q - 8, exactly: 9 instructions for eight codes (a
// published method: Kim, Henry, Fahim, Awadalla, "Who Says Elephants Can't Run: Bringing Large
// Scale MoE Models into Cloud Scale Production", 2022).  Signed codes keep the fp32 sums as small
// as the values they stand for; an offset left in and taken off later (bf16 has no packed add: 7
// instructions) cost a digit where values average out, or twice the matrix instructions.  (The bits
// alone are subnormal numbers, five instructions, but the sums of their products lose ten bits.)
//
// The other operand is fp32 data as two fp16 parts, after a power of two of its own per row that
// brings the largest value to 1 .. 2: x = x0 + x1 to within 2^-23 of x, or 2^-25 of the row's
// largest where the second part runs out of fp16's range, fp32's own level.  (Larger numbers
// would gain nothing and cost the sums' range.)
#pragma once

#include "lx_gemm_common.hpp"

namespace lx {

typedef _Float16 half2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8_t __attribute__((ext_vector_type(8)));
typedef unsigned short ushortx4_t __attribute__((ext_vector_type(4)));

// The pattern of 1024.0 in both halves, in a vector register: as a constant known to the compiler
// it becomes a literal, and a literal each for mask and pattern makes two instructions of one.
__device__ __forceinline__ unsigned q4_pattern() {
  unsigned m;
  asm("v_mov_b32 %0, 0x64006400" : "=v"(m));
  return m;
}

__device__ __forceinline__ half8_t q4_frag(unsigned w, unsigned pattern) {
  const half2_t off = {(_Float16)-1032.0f, (_Float16)-1032.0f};
  const half2_t off16 = {(_Float16)-72.0f, (_Float16)-72.0f};
  const half2_t r16 = {(_Float16)0.0625f, (_Float16)0.0625f};
  const unsigned v = w >> 8;
  const half2_t h0 = __builtin_bit_cast(half2_t, (w & 0x000f000fu) | pattern) + off;
  const half2_t h1 = __builtin_elementwise_fma(
      __builtin_bit_cast(half2_t, (w & 0x00f000f0u) | pattern), r16, off16);
  const half2_t h2 = __builtin_bit_cast(half2_t, (v & 0x000f000fu) | pattern) + off;
  const half2_t h3 = __builtin_elementwise_fma(
      __builtin_bit_cast(half2_t, (v & 0x00f000f0u) | pattern), r16, off16);
  const uintx4_t u = {__builtin_bit_cast(unsigned, h0), __builtin_bit_cast(unsigned, h1),
                      __builtin_bit_cast(unsigned, h2), __builtin_bit_cast(unsigned, h3)};
  return __builtin_bit_cast(half8_t, u);
}

// Code q (< 16) at element j's bits in the dword, and back.
__device__ __forceinline__ unsigned q4_put(unsigned q, int j) {
  return q << (4 * (j >> 1) + 16 * (j & 1));
}
__device__ __forceinline__ unsigned q4_get(unsigned w, int j) {
  return (w >> (4 * (j >> 1) + 16 * (j & 1))) & 15u;
}

// x s as two fp16 parts.  The first is pinned: converted anew for the remainder, it costs half
// as many instructions again, and where x is a product folded into one of the two conversions
// the parts belong to different numbers next to a tie (2^-11 off).
__device__ __forceinline__ void split_pair(float x0, float x1, float s, half2_t& p0, half2_t& p1) {
  p0 = half2_t{(_Float16)(x0 * s), (_Float16)(x1 * s)};
  unsigned u = __builtin_bit_cast(unsigned, p0);
  asm("" : "+v"(u));
  p0 = __builtin_bit_cast(half2_t, u);
  p1 = half2_t{(_Float16)fmaf(x0, s, -(float)p0[0]), (_Float16)fmaf(x1, s, -(float)p0[1])};
}
__device__ __forceinline__ void split2(const float (&x)[8], float s, half8_t& p0, half8_t& p1) {
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    half2_t h, l;
    split_pair(x[j], x[j + 1], s, h, l);
    p0[j] = h[0];
    p0[j + 1] = h[1];
    p1[j] = l[0];
    p1[j + 1] = l[1];
  }
}

// The largest magnitudes of the rows that 16 lanes hold eight values each of, n rows a lane, for
// row_scale.  Among lanes as integers, which order as magnitudes do and need no check for a NaN; a
// step of all the rows at once, as a lane's value can cross over two instructions after it is made.
template <int N>
__device__ __forceinline__ void tops16(const float4 (&x)[N][2], float (&top)[N]) {
  unsigned u[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float4 a = x[i][0], b = x[i][1];
    float t = fmaxf(fabsf(a.x), fabsf(a.y));
    t = fmaxf(fmaxf(t, fabsf(a.z)), fabsf(a.w));
    t = fmaxf(fmaxf(t, fabsf(b.x)), fabsf(b.y));
    t = fmaxf(fmaxf(t, fabsf(b.z)), fabsf(b.w));
    u[i] = __float_as_uint(t);
  }
#define LX_TOPS_STEP(CTRL)      \
  _Pragma("unroll") for (int i = 0; i < N; ++i) u[i] = \
      max(u[i], (unsigned)__builtin_amdgcn_update_dpp(0, (int)u[i], CTRL, 0xF, 0xF, true))
  LX_TOPS_STEP(kDppXor1);
  LX_TOPS_STEP(kDppXor2);
  LX_TOPS_STEP(kDppHalfMirror);
  LX_TOPS_STEP(kDppMirror);
#undef LX_TOPS_STEP
#pragma unroll
  for (int i = 0; i < N; ++i) top[i] = __uint_as_float(u[i]);
}

// The power of two that brings a row with largest magnitude `top` to 1 .. 2, and its inverse
// (both normal numbers; an infinite top stays infinite).
__device__ __forceinline__ float row_scale(float top, float* inverse) {
  const unsigned e = min(max(__float_as_uint(top) >> 23 & 255u, 1u), 253u);
  *inverse = __uint_as_float(e << 23);
  return __uint_as_float((254u - e) << 23);
}

__device__ __forceinline__ floatx4 mfma_f16(half8_t a, half8_t b, floatx4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// Whether `rows` rows of ca floats every lda from a and of cb every ldb from b share memory; rows of
// unequal strides that interleave count as sharing.
inline bool rows_overlap(const float* a, long lda, long ca, const float* b, long ldb, long cb,
                         long rows) {
  const intptr_t pa = (intptr_t)a / 4, pb = (intptr_t)b / 4;
  if (pa + (rows - 1) * lda + ca <= pb || pb + (rows - 1) * ldb + cb <= pa) return false;
  if (lda != ldb) return true;
  const long d = ((pb - pa) % lda + lda) % lda;  // the column of a's rows where b's begin
  return d < ca || d + cb > lda;
}

// fp32 bits of the bf16 in the low or high half of a dword.
__device__ __forceinline__ float bf16_lo(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float bf16_hi(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

}  // namespace lx
