// Matrices in 8 bits (lx_q8.hip, lx_q8_linear.hip): layout, and the forming of codes.
//
// Blocks of 128 consecutive elements of a row share 2^e, e the smallest integer >= -127 with
// max|v| <= 448 * 2^e over the finite ones; a code is the e4m3 number nearest to v / 2^e (exact
// but for that one rounding: a power of two, and v_cvt_pk_fp8_f32 rounds to nearest even).  The
// scales are held as bytes e + 127, the exponent field of 2^e.
//
// Memory: tiles of 16 rows x 128 elements, 2 KB each, the blocks of K of a row tile side by side. A
// tile is its first 64 columns, then its last, 1 KB each: 16 rows of four 16-byte chunks, which
// stand at chunk ^ (row / 4 % 4).  That spreads the 16 rows that a ds_read_b128 of a fragment
// touches over all 64 banks, so tiles and halves of them go to LDS as they lie, whole lines at a
// time.  (With a row's 128 bytes as one line a producer of one row writes whole lines, but a kernel
// that takes halves of blocks moves half lines: 1531 x 896 x 4864 19.9 us in place of 18.5, 16 rows
// on 151936 x 896 30.9 in place of 28.7.)  Which elements of a block a lane multiplies in one
// instruction does not matter while both operands agree and a block has one scale: a lane takes
// 16-byte chunks.  Behind the codes the scales, a byte a row: 16 bytes per tile, tiles in the same
// order. Elements past the end of a row are zero; rows past the last may hold anything and only
// reach outputs that are not stored.
#pragma once

#include "lx_common.hpp"
#include "lx_internal.hpp"

namespace lx {

constexpr int kQ8Rows = 16, kQ8Block = 128, kQ8Tile = kQ8Rows * kQ8Block;

inline long q8_tiles(long rows) { return (rows + kQ8Rows - 1) / kQ8Rows; }
inline long q8_blocks(long K) { return (K + kQ8Block - 1) / kQ8Block; }
inline size_t q8_code_bytes(long rows, long K) {
  return (size_t)q8_tiles(rows) * q8_blocks(K) * kQ8Tile;
}

// A matrix in 8 bits as the kernels see it.
struct Q8Mat {
  unsigned char* codes;
  unsigned char* scales;
  int rows, K, kb;  // kb blocks of K
};

inline bool q8_shape_ok(int rows, int K) {
  return rows > 0 && K > 0 && K <= INT_MAX - 127 && rows <= INT_MAX - 15;
}
inline bool q8_ok(const lx_q8* q) {
  return q && q->data && (uintptr_t)q->data % 16 == 0 && q8_shape_ok(q->rows, q->K);
}
inline Q8Mat q8_mat(const lx_q8* q) {
  unsigned char* p = static_cast<unsigned char*>(q->data);
  const int kb = (int)q8_blocks(q->K);
  return Q8Mat{p, p + q8_code_bytes(q->rows, q->K), q->rows, q->K, kb};
}

// Whether `rows` rows of n floats every ld from p share memory with the matrix.
inline bool q8_overlaps(const lx_q8* q, const float* p, long ld, long n, long rows) {
  return rows_overlap(p, ld, n, static_cast<const float*>(q->data), 0,
                      (long)(lx_q8_bytes(q->rows, q->K) / 4), rows);
}

// Where chunk c (0 .. 7) of row r (0 .. 15) stands in a tile.
__device__ __forceinline__ int q8_chunk(int r, int c) {
  return (c >> 2) * (kQ8Tile / 2) + r * (kQ8Block / 2) + (((c & 3) ^ (r >> 2)) << 4);
}

// Byte offset of element k (of its chunk, for k a multiple of 16) of a row.
__device__ __forceinline__ long q8_at(const Q8Mat& q, int row, int k) {
  return ((long)(row >> 4) * q.kb + (k >> 7)) * kQ8Tile + q8_chunk(row & 15, (k >> 4) & 7) +
         (k & 15);
}
__device__ __forceinline__ long q8_scale_at(const Q8Mat& q, int row, int kb) {
  return ((long)(row >> 4) * q.kb + kb) * kQ8Rows + (row & 15);
}

// The e8m0 byte of a block whose largest finite magnitude is `top`: 448 = 1.75 * 2^8.
__device__ __forceinline__ int q8_scale(float top) {
  const unsigned u = __float_as_uint(top);
  return max((int)(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0), 0);
}
__device__ __forceinline__ float q8_power(int byte) {  // 2^(byte - 127)
  return __uint_as_float(byte ? (unsigned)byte << 23 : 0x400000u);
}

// Sixteen lanes hold a block of a row, elements 8 (lane % 16) .. + 7 each: forms its codes and
// scale and stores them at chunk k / 16 of the row.
__device__ __forceinline__ void q8_store_block(const Q8Mat& q, int row, int k, const float (&v)[8]) {
  float top = 0.0f;
  float w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const bool fin = fabsf(v[j]) < __builtin_huge_valf();
    w[j] = fin ? v[j] : __builtin_nanf("");
    top = fmaxf(top, fin ? fabsf(v[j]) : 0.0f);
  }
  top = fmaxf(top, dpp_mov<kDppXor1>(top));
  top = fmaxf(top, dpp_mov<kDppXor2>(top));
  top = fmaxf(top, dpp_mov<kDppHalfMirror>(top));
  top = fmaxf(top, dpp_mov<kDppMirror>(top));
  const int byte = q8_scale(top);
  const float inv = __uint_as_float((unsigned)(254 - byte) << 23);
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] *= inv;
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(w[0], w[1], lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(w[2], w[3], lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(w[4], w[5], hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(w[6], w[7], hi, true);
  *reinterpret_cast<int2*>(q.codes + q8_at(q, row, k)) = make_int2(lo, hi);
  if ((k & 127) == 0) q.scales[q8_scale_at(q, row, k >> 7)] = (unsigned char)byte;
}

}  // namespace lx
