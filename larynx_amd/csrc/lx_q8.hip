// Rows into 8 bits and back: the plain quantiser, the residual's addition with an RMSNorm, the
// read-back.  Layout and codes: lx_q8.hpp.
#include <algorithm>
#include <climits>

#include "lx_q8.hpp"

namespace lx {
namespace {

// Four floats at a 4-byte boundary: gfx950 loads and stores them in one instruction (only whole
// vectors of 16 bytes need no more than dword alignment in global memory).
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));

// Elements k .. k + 7 of a row of n, zero past its end.
__device__ __forceinline__ void load8(const float* row, int k, int n, float (&v)[8]) {
  if (k + 8 <= n) {
    const float4u a = *reinterpret_cast<const float4u*>(row + k);
    const float4u b = *reinterpret_cast<const float4u*>(row + k + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[j] = a[j];
      v[j + 4] = b[j];
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = k + j < n ? row[k + j] : 0.0f;
  }
}
__device__ __forceinline__ void store8(float* row, int k, int n, const float (&v)[8]) {
  if (k + 8 <= n) {
    *reinterpret_cast<float4u*>(row + k) = float4u{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<float4u*>(row + k + 4) = float4u{v[4], v[5], v[6], v[7]};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < n) row[k + j] = v[j];
  }
}

// This thread's row and eight elements of it: sixteen lanes a block, the next sixteen the block of
// the row that shares its lines (8192 x 8192 58 -> 56 us, back 68 -> 65).
__device__ __forceinline__ bool block_of(const Q8Mat& q, int& row, int& k) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, per = (long)q.kb * 32;
  const int in = (int)(i % per);
  row = (int)(i / per) * 2 + (in >> 4 & 1);
  k = (in >> 5) * kQ8Block + (in & 15) * 8;
  return row < q.rows;
}

__global__ __launch_bounds__(256) void q8_quant_kernel(const float* __restrict__ x, long ldx,
                                                       Q8Mat q) {
  int row, k;
  if (!block_of(q, row, k)) return;
  float v[8];
  load8(x + row * ldx, k, q.K, v);
  q8_store_block(q, row, k, v);
}

__global__ __launch_bounds__(256) void q8_dequant_kernel(Q8Mat q, float* __restrict__ x, long ldx) {
  int row, k;
  if (!block_of(q, row, k)) return;
  const int2 c = *reinterpret_cast<const int2*>(q.codes + q8_at(q, row, k));
  const float s = q8_power(q.scales[q8_scale_at(q, row, k >> 7)]);
  typedef float float2v __attribute__((ext_vector_type(2)));
  float v[8];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int w = j ? c.y : c.x;
    const float2v a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const float2v b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    v[4 * j] = a[0] * s;
    v[4 * j + 1] = a[1] * s;
    v[4 * j + 2] = b[0] * s;
    v[4 * j + 3] = b[1] * s;
  }
  store8(x + row * ldx, k, q.K, v);
}

// ---- h = x + add; codes of h / sqrt(mean(h^2) + eps) * w ------------------------------------

template <int CTRL>
__device__ __forceinline__ double dpp_mov64(double v) {
  const int2 u = __builtin_bit_cast(int2, v);
  return __builtin_bit_cast(double, make_int2(__builtin_amdgcn_mov_dpp(u.x, CTRL, 0xF, 0xF, false),
                                              __builtin_amdgcn_mov_dpp(u.y, CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp_mov64<kDppXor1>(v);
  v += dpp_mov64<kDppXor2>(v);
  v += dpp_mov64<kDppHalfMirror>(v);
  v += dpp_mov64<kDppMirror>(v);
  v += __shfl_xor(v, 16);
  v += __shfl_xor(v, 32);
  return v;
}

__device__ __forceinline__ double half_sum64(double v) {
  v += dpp_mov64<kDppXor1>(v);
  v += dpp_mov64<kDppXor2>(v);
  v += dpp_mov64<kDppHalfMirror>(v);
  v += dpp_mov64<kDppMirror>(v);
  v += __shfl_xor(v, 32);
  return v;
}

// d rounded to fp32 towards the odd neighbour: a further rounding to fewer bits than fp32's less
// two, and comparisons with numbers of fewer bits, come out as d's own would.
__device__ __forceinline__ float to_odd(double d) {
  const float f = (float)d;
  unsigned u = __float_as_uint(f);
  if ((double)f != d && !(u & 1)) u = fabs((double)f) > fabs(d) ? u - 1 : u + 1;
  return __uint_as_float(u);
}

struct NormArgs {
  const float *x, *add, *w;
  float* sum;
  long ldx, lda, lds;
  float eps;
  Q8Mat q;
};

// The row of a workgroup that has one: of sixteen, two that share lines go to one XCD (workgroups
// are dealt to them round-robin).  30000 x 2500 102 -> 97.5 us, with add 202 -> 198.
__device__ __forceinline__ int row_of(const Q8Mat& q) {
  const int b = blockIdx.x;
  return b < q.rows / 16 * 16 ? b / 16 * 16 + b % 8 * 2 + (b >> 3 & 1) : b;
}

// G threads a row, each NC chunks of eight elements in registers (one pass over x and add); the
// row's power and the normalised values in 64 bits, where a code next to a border is decided: some
// 40 instructions an element, which a row's bytes hide.  PAIR: a workgroup has the two rows whose
// codes share lines, sixteen lanes of one beside sixteen of the other, so that a wave stores whole
// lines (pairs_pay).  1531 x 896 6.5 us, a launch and one round trip; 8192 x 8192 with add 156 (5.6
// TB/s; a copy: 4.7), without add, whose bytes are half, 80 (4.2 TB/s, the instructions).  Four
// elements a lane need a fifth step of each block's maximum for half the elements: 6 to 20% slower.
template <int G, int NC, bool PAIR>
__global__ __launch_bounds__(PAIR ? 2 * G : 256) void norm_q8_kernel(NormArgs a) {
  const int side = threadIdx.x >> 4 & 1;  // of a pair
  const int t = PAIR ? (threadIdx.x >> 5) * 16 + (threadIdx.x & 15) : threadIdx.x % G;
  const int row = PAIR      ? blockIdx.x * 2 + side
                  : G == 64 ? blockIdx.x * 4 + threadIdx.x / 64
                            : row_of(a.q);
  const int D = a.q.K, chunks = row < a.q.rows ? a.q.kb * 16 : 0;
  __shared__ double part[PAIR ? 2 : 1][PAIR ? 8 : 4];
  if (G == 64 && row >= a.q.rows) return;
  float h[NC][8];
  double s = 0.0;
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int k = (t + G * c) * 8;
    if (t + G * c < chunks) {
      load8(a.x + row * a.ldx, k, D, h[c]);
      if (a.add) {
        float u[8];
        load8(a.add + row * a.lda, k, D, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) h[c][j] += u[j];
        store8(a.sum + row * a.lds, k, D, h[c]);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s = fma((double)h[c][j], (double)h[c][j], s);
    }
  }
  s = PAIR ? half_sum64(s) : wave_sum64(s);
  if constexpr (G > 64) {
    if ((threadIdx.x & (PAIR ? 47 : 63)) == 0) part[PAIR ? side : 0][threadIdx.x >> 6] = s;
    __syncthreads();
    const double* p = part[PAIR ? side : 0];
    s = (p[0] + p[1]) + (p[2] + p[3]);
    if constexpr (PAIR) s += (p[4] + p[5]) + (p[6] + p[7]);
  }
  const double r = 1.0 / sqrt(s / D + (double)a.eps);
#pragma unroll
  for (int c = 0; c < NC; ++c) {
    const int k = (t + G * c) * 8;
    if (t + G * c < chunks) {
      float w[8];
      load8(a.w, k, D, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = to_odd((double)h[c][j] * r * (double)w[j]);
      q8_store_block(a.q, row, k, w);
    }
  }
}

// Rows of any length: the sums (or x) are read a second time.
__global__ __launch_bounds__(256) void norm_q8_long_kernel(NormArgs a) {
  const int row = row_of(a.q), t = threadIdx.x;
  const int D = a.q.K, chunks = a.q.kb * 16;
  __shared__ double part[4];
  double s = 0.0;
  for (int c = t; c < chunks; c += 256) {
    float h[8];
    load8(a.x + row * a.ldx, c * 8, D, h);
    if (a.add) {
      float u[8];
      load8(a.add + row * a.lda, c * 8, D, u);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] += u[j];
      store8(a.sum + row * a.lds, c * 8, D, h);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fma((double)h[j], (double)h[j], s);
  }
  s = wave_sum64(s);
  if ((t & 63) == 0) part[t >> 6] = s;
  __syncthreads();
  s = (part[0] + part[1]) + (part[2] + part[3]);
  const double r = 1.0 / sqrt(s / D + (double)a.eps);
  const float* src = a.add ? a.sum + row * a.lds : a.x + row * a.ldx;  // this thread's own chunks
  for (int c = t; c < chunks; c += 256) {
    float h[8], w[8];
    load8(src, c * 8, D, h);
    load8(a.w, c * 8, D, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = to_odd((double)h[j] * r * (double)w[j]);
    q8_store_block(a.q, row, c * 8, w);
  }
}

}  // namespace
}  // namespace lx

using namespace lx;

extern "C" size_t lx_q8_bytes(int rows, int K) {
  if (!q8_shape_ok(rows, K)) return 0;
  return q8_code_bytes(rows, K) + (size_t)q8_tiles(rows) * q8_blocks(K) * kQ8Rows;
}

namespace {
// Workgroups of 256 threads, sixteen lanes a block of the matrix.
long q8_grid(const Q8Mat& q) { return (((long)q.rows + 1) / 2 * q.kb * 32 + 255) / 256; }
}  // namespace

extern "C" int lx_q8_pack_f32(const float* x, long ldx, const lx_q8* q, hipStream_t stream) {
  LX_REQUIRE(x && q8_ok(q), "q8_pack: null pointer, bad shape or unaligned matrix");
  LX_REQUIRE(ldx >= q->K && (uintptr_t)x % 4 == 0, "q8_pack: bad row stride %ld", ldx);
  const Q8Mat m = q8_mat(q);
  LX_REQUIRE(q8_grid(m) <= INT_MAX / 256, "q8_pack: %d rows of %d are too many", m.rows, m.K);
  LX_REQUIRE(!q8_overlaps(q, x, ldx, m.K, m.rows), "q8_pack: the matrix overlaps x");
  hipLaunchKernelGGL(q8_quant_kernel, dim3((unsigned)q8_grid(m)), dim3(256), 0, stream, x, ldx, m);
  return check_launch("q8_quant_kernel");
}

extern "C" int lx_q8_unpack_f32(const lx_q8* q, float* x, long ldx, hipStream_t stream) {
  LX_REQUIRE(x && q8_ok(q), "q8_unpack: null pointer, bad shape or unaligned matrix");
  LX_REQUIRE(ldx >= q->K && (uintptr_t)x % 4 == 0, "q8_unpack: bad row stride %ld", ldx);
  const Q8Mat m = q8_mat(q);
  LX_REQUIRE(q8_grid(m) <= INT_MAX / 256, "q8_unpack: %d rows of %d are too many", m.rows, m.K);
  LX_REQUIRE(!q8_overlaps(q, x, ldx, m.K, m.rows), "q8_unpack: x overlaps the matrix");
  hipLaunchKernelGGL(q8_dequant_kernel, dim3((unsigned)q8_grid(m)), dim3(256), 0, stream, m, x,
                     ldx);
  return check_launch("q8_dequant_kernel");
}

extern "C" int lx_rmsnorm_q8_f32(const float* x, long ldx, const float* add, long lda, float* sum,
                                 long lds, const float* w, float eps, const lx_q8* q,
                                 hipStream_t stream) {
  LX_REQUIRE(x && w && q8_ok(q), "rmsnorm_q8: null pointer, bad shape or unaligned matrix");
  LX_REQUIRE(!add == !sum, "rmsnorm_q8: add and sum go together");
  LX_REQUIRE(ldx >= q->K && (!add || (lda >= q->K && lds >= q->K)), "rmsnorm_q8: bad row stride");
  LX_REQUIRE(((uintptr_t)x | (uintptr_t)add | (uintptr_t)sum | (uintptr_t)w) % 4 == 0,
             "rmsnorm_q8: unaligned");
  const int rows = q->rows, D = q->K;
  if (add) {
    // in place is fine: each thread reads what it writes first
    LX_REQUIRE((sum == x && lds == ldx) || !rows_overlap(x, ldx, D, sum, lds, D, rows),
               "rmsnorm_q8: sum overlaps x");
    LX_REQUIRE((sum == add && lds == lda) || !rows_overlap(add, lda, D, sum, lds, D, rows),
               "rmsnorm_q8: sum overlaps add");
  }
  LX_REQUIRE((D <= 2048 ? ((long)rows + 3) / 4 : (long)rows) <= INT_MAX / 256,
             "rmsnorm_q8: %d rows of %d are too many", rows, D);
  LX_REQUIRE(!q8_overlaps(q, x, ldx, D, rows) && !q8_overlaps(q, w, D, D, 1) &&
                 (!add || (!q8_overlaps(q, add, lda, D, rows) &&
                           !q8_overlaps(q, sum, lds, D, rows))),
             "rmsnorm_q8: the matrix overlaps x, add, sum or w");
  LX_REQUIRE(!sum || !rows_overlap(sum, lds, D, w, 0, D, rows), "rmsnorm_q8: sum overlaps w");
  NormArgs a{x, add, w, sum, ldx, lda, lds, eps, q8_mat(q)};
  // Rows of 4097 to 8192 two a workgroup?  Where the call's bytes come from memory and, of the four
  // chunks that a thread may hold, more than two are taken (us, one row and two; the same buffers
  // every call, then several in turn, more than the 256 MB of the last cache)
  //    1531 x 8192 163 MB   29.4 30.4   38.7 36.8       8192 x 4100  437 MB   93.6  97.4
  //    2048 x 7000 186      35.0 34.6   46.2 47.8       8192 x 4300  458     101.3 104.7
  //    2048 x 8192 218      37.8 38.4   47.6 44.9       8192 x 4480  477      97.8  94.8
  //    3000 x 6400 250      46.6 46.0   56.3 54.3       8192 x 4864  518     108.1 101.5
  //    4000 x 5000 260      48.7 48.3   58.6 57.3       8192 x 8192  872     176.8 156.1
  //    3000 x 8192 319      63.2 58.8   68.1 62.3      30000 x 4608 1797     372   340
  // Without add the bytes are fewer than the instructions (6000 x 8192 52 and 53).
  const bool pairs_pay = add && D >= 4480 && D <= 8192 && 13.0 * rows * D >= 2e8;
  const dim3 wide((unsigned)rows), four((unsigned)(((long)rows + 3) / 4)), block(256);
  if (D <= 1024)
    hipLaunchKernelGGL((norm_q8_kernel<64, 2, false>), four, block, 0, stream, a);
  else if (D <= 2048)
    hipLaunchKernelGGL((norm_q8_kernel<64, 4, false>), four, block, 0, stream, a);
  else if (D <= 4096)
    hipLaunchKernelGGL((norm_q8_kernel<256, 2, false>), wide, block, 0, stream, a);
  else if (pairs_pay)
    hipLaunchKernelGGL((norm_q8_kernel<256, 4, true>), dim3((unsigned)(((long)rows + 1) / 2)),
                       dim3(512), 0, stream, a);
  else if (D <= 8192)
    hipLaunchKernelGGL((norm_q8_kernel<256, 4, false>), wide, block, 0, stream, a);
  else
    hipLaunchKernelGGL(norm_q8_long_kernel, wide, block, 0, stream, a);
  return check_launch("norm_q8_kernel");
}
