// Projections of few rows on 4-bit weights with group scales.
//
//   w~[n, k] = s[n, k / G] * (q[n, k] - 8),  y = epi(x w~^T + bias),  G = 32, 64 or 128.
//
// What bounds it is the weight stream (half a byte a weight), so the codes go from memory to
// the matrix cores with seven instructions for eight of them (lx_four_bit.hpp) and the scale is
// applied once per group to the fp32 sum, not to the weights: a group's products with 16 + q
// start from -24 times the sum of its x, and the sum times s joins the row's total.  x enters
// as three bf16 parts, so every product is exact and the sums are fp32.
//
// Layout (lx_q4_pack_f32): per tile of 16 rows and block of 128 inputs 1 KB of codes, the 64
// lanes' 16-byte fragments (dword t of lane l: row l % 16, k = 32 t + 8 (l / 16) + 0..7), then
// for all tiles the bf16 scales, per (tile, block) the four row quads' [group][row] runs: a
// lane's accumulators are rows 4 (l / 16) .. + 3, so it reads its scales with one load.  Rows
// and inputs past the matrix have scale 0.
#include <algorithm>
#include <climits>

#include "lx_four_bit.hpp"

namespace lx {
namespace {

constexpr int kTileN = 16;    // rows of a tile
constexpr int kBlockK = 128;  // inputs of a block
constexpr int kMaxRows = 64;
constexpr int kPackedCols = 5;  // rows of x whose three parts fit one fragment's 16 columns

struct Q4Args {
  const float* x;
  long ldx;
  const uintx4_t* codes;
  const unsigned short* scales;
  const float* bias;
  float* y;
  long ldy;
  int M, N, K, kb, epi;
};

__host__ __device__ inline long q4_tiles(int N) { return (N + kTileN - 1) / kTileN; }
__host__ __device__ inline long q4_blocks(int K) { return (K + kBlockK - 1) / kBlockK; }

// ---- quantise and lay out ---------------------------------------------------------------

// One wave per (row tile, block): lane l holds row l % 16, inputs 32 t + 8 (l / 16) + j.
template <int G>
__global__ __launch_bounds__(64) void q4_pack_kernel(const float* __restrict__ W,
                                                     uintx4_t* __restrict__ codes,
                                                     unsigned short* __restrict__ scales, int N,
                                                     int K, int kb) {
  constexpr int TG = G / 32;  // 32-wide steps of a group
  const int lane = threadIdx.x, c = lane >> 4, r = lane & 15;
  const long tile = blockIdx.x;  // row tile * kb + block
  const long n = tile / kb * kTileN + r;
  const int k0 = (int)(tile % kb) * kBlockK;
  float w[4][8];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = k0 + 32 * t + 8 * c + 4 * e;
      const float4 v = n < N && k < K ? *reinterpret_cast<const float4*>(W + n * K + k)
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
      w[t][4 * e] = v.x;
      w[t][4 * e + 1] = v.y;
      w[t][4 * e + 2] = v.z;
      w[t][4 * e + 3] = v.w;
    }
  uintx4_t q = {0, 0, 0, 0};
#pragma unroll
  for (int g = 0; g < 4 / TG; ++g) {
    // the value of largest magnitude, the lowest input among equals
    float best = 0.0f;
    int at = INT_MAX;
    bool bad = false;
#pragma unroll
    for (int t = g * TG; t < (g + 1) * TG; ++t)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        bad |= !(fabsf(w[t][j]) <= 3.402823466e38f);
        if (fabsf(w[t][j]) > fabsf(best)) {
          best = w[t][j];
          at = 32 * t + 8 * c + j;
        }
      }
#pragma unroll
    for (int d = 16; d <= 32; d *= 2) {
      const float ob = d == 16 ? lane_xor16(best) : lane_xor32(best);
      const int oa = __float_as_int(d == 16 ? lane_xor16(__int_as_float(at))
                                            : lane_xor32(__int_as_float(at)));
      const float ox = d == 16 ? lane_xor16(bad ? 1.0f : 0.0f) : lane_xor32(bad ? 1.0f : 0.0f);
      bad |= ox != 0.0f;
      if (fabsf(ob) > fabsf(best) || (fabsf(ob) == fabsf(best) && oa < at)) {
        best = ob;
        at = oa;
      }
    }
    // rounded once, to bf16 (eight bits: the codes are chosen for the rounded scale, so only
    // the largest value of a group sees it, by at most s / 32)
    const __bf16 sb = (__bf16)(best * -0.125f);
    const unsigned short s16 = bad ? 0x7fc0 : __builtin_bit_cast(unsigned short, sb);
    const float s = bad ? 0.0f : (float)sb;
#pragma unroll
    for (int t = g * TG; t < (g + 1) * TG; ++t) {
      unsigned word = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        // in 64 bits: a quotient next to a border decides a whole step
        const double u = s != 0.0f ? rint((double)w[t][j] / (double)s) : 0.0;
        word |= q4_put((unsigned)(int)(fmin(fmax(u, -8.0), 7.0) + 8.0), j);
      }
      q[t] = word;
    }
    if (c == 0) scales[((tile * 4 + (r >> 2)) * (4 / TG) + g) * 4 + (r & 3)] = s16;
  }
  codes[tile * 64 + lane] = q;
}

__global__ __launch_bounds__(256) void q4_unpack_kernel(const unsigned* __restrict__ codes,
                                                        const unsigned short* __restrict__ scales,
                                                        float* __restrict__ W, int N, int K,
                                                        int kb, int G) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x;  // one dword of eight codes
  if (i >= q4_tiles(N) * kb * 256) return;
  const long tile = i >> 8;
  const int lane = (int)(i >> 2) & 63, t = (int)i & 3, c = lane >> 4, r = lane & 15;
  const long n = tile / kb * kTileN + r;
  const int k = (int)(tile % kb) * kBlockK + 32 * t + 8 * c;
  if (n >= N) return;
  const int ng = kBlockK / G;
  const float s = bf16_lo(scales[((tile * 4 + (r >> 2)) * ng + 32 * t / G) * 4 + (r & 3)]);
  const unsigned w = codes[i];
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (k + j < K) W[n * K + k + j] = s * ((float)q4_get(w, j) - 8.0f);
}

// ---- the product ------------------------------------------------------------------------

// A workgroup owns one tile of 16 weight rows against all M rows of x; its waves take the
// blocks of K in turn and their sums meet in LDS, in wave order.  PC: at most 5 rows of x,
// whose three parts are columns 3 m + part of one fragment (one product per 32 inputs); else
// CT column tiles of 16 rows, three products each.
template <int CT, bool PC, int G>
__global__ __launch_bounds__(1024) void q4_linear_kernel(Q4Args a) {
  constexpr int TG = G / 32, NG = 4 / TG, NP = PC ? 1 : 3;
  extern __shared__ float red[];  // [waves][CT * 4][64]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, waves = blockDim.x >> 6;
  const int c = lane >> 4, col = lane & 15;
  const long rt = blockIdx.x;
  const float* xr[CT];
  bool live[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) {
    const int m = PC ? col / 3 : ct * 16 + col;
    live[ct] = m < a.M && (!PC || col < 15);
    xr[ct] = a.x + (long)min(m, a.M - 1) * a.ldx;
  }
  floatx4 tot[CT];
#pragma unroll
  for (int ct = 0; ct < CT; ++ct) tot[ct] = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < a.kb; kb += waves) {
    const long tile = rt * a.kb + kb;
    const uintx4_t w = a.codes[tile * 64 + lane];
    const ushortx4_t* sp =
        reinterpret_cast<const ushortx4_t*>(a.scales) + (tile * 4 + c) * NG;
    ushortx4_t sc[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) sc[g] = sp[g];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      sbf16x8 wf[TG];
#pragma unroll
      for (int t = 0; t < TG; ++t) wf[t] = q4_frag(w[g * TG + t]);
#pragma unroll
      for (int ct = 0; ct < CT; ++ct) {
        sbf16x8 xf[TG][NP];
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < TG; ++t) {
          const int k = kb * kBlockK + (g * TG + t) * 32 + c * 8;
          float v[8];
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float4 u = live[ct] && k + 4 * e < a.K
                                 ? *reinterpret_cast<const float4*>(xr[ct] + k + 4 * e)
                                 : make_float4(0.f, 0.f, 0.f, 0.f);
            v[4 * e] = u.x;
            v[4 * e + 1] = u.y;
            v[4 * e + 2] = u.z;
            v[4 * e + 3] = u.w;
          }
          sbf16x8 p[3];
          split3(v, p);
          if constexpr (PC) {
            const int part = col % 3;
            xf[t][0] = part == 0 ? p[0] : part == 1 ? p[1] : p[2];
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += (float)xf[t][0][j];
          } else {
#pragma unroll
            for (int i = 0; i < 3; ++i) xf[t][i] = p[i];
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += v[j];
          }
        }
        sum += lane_xor16(sum);
        sum += lane_xor32(sum);
        const float c0 = -24.0f * sum;
        floatx4 acc = {c0, c0, c0, c0};
#pragma unroll
        for (int t = 0; t < TG; ++t)
#pragma unroll
          for (int i = NP - 1; i >= 0; --i) acc = mfma_bf16(wf[t], xf[t][i], acc);
#pragma unroll
        for (int i = 0; i < 4; ++i) tot[ct][i] += bf16_lo(sc[g][i]) * acc[i];
      }
    }
  }
#pragma unroll
  for (int ct = 0; ct < CT; ++ct)
#pragma unroll
    for (int i = 0; i < 4; ++i) red[((wave * CT + ct) * 4 + i) * 64 + lane] = tot[ct][i];
  __syncthreads();
  // value of row r of the tile against row m of x
  auto value = [&](int r, int m) {
    float s = 0.0f;
    for (int w = 0; w < waves; ++w) {
      const float* p = red + (w * CT * 4 + (r & 3)) * 64 + (r >> 2) * 16;
      if constexpr (PC) {
        s += (p[3 * m + 2] + p[3 * m + 1]) + p[3 * m];
      } else {
        s += p[(m >> 4) * 256 + (m & 15)];
      }
    }
    return s;
  };
  const int rows = a.epi == LX_EPI_SWIGLU_PAIRED ? kTileN / 2 : kTileN;
  for (int i = tid; i < rows * a.M; i += blockDim.x) {
    const int m = i / rows, r = i % rows;
    if (a.epi == LX_EPI_SWIGLU_PAIRED) {
      const long n = rt * kTileN + 2 * r;
      if (n >= a.N) continue;
      float g = value(2 * r, m), u = value(2 * r + 1, m);
      if (a.bias) {
        g += a.bias[n];
        u += a.bias[n + 1];
      }
      a.y[m * a.ldy + (n >> 1)] = (g / (1.0f + expf(-g))) * u;
    } else {
      const long n = rt * kTileN + r;
      if (n >= a.N) continue;
      float v = value(r, m);
      if (a.bias) v += a.bias[n];
      float* y = a.y + m * a.ldy + n;
      *y = a.epi == LX_EPI_GELU_TANH ? gelu_tanh(v) : a.epi == LX_EPI_RESID ? *y + v : v;
    }
  }
}

template <int CT, bool PC>
int launch_linear(const Q4Args& a, int G, hipStream_t s) {
  const int waves = std::min(PC || CT == 1 ? 16 : 8, a.kb);
  const dim3 grid((unsigned)q4_tiles(a.N)), block(64 * waves);
  const size_t lds = (size_t)waves * CT * 1024;
  if (G == 32)
    hipLaunchKernelGGL((q4_linear_kernel<CT, PC, 32>), grid, block, lds, s, a);
  else if (G == 64)
    hipLaunchKernelGGL((q4_linear_kernel<CT, PC, 64>), grid, block, lds, s, a);
  else
    hipLaunchKernelGGL((q4_linear_kernel<CT, PC, 128>), grid, block, lds, s, a);
  return check_launch("q4_linear_kernel");
}

bool q4_shape_ok(int N, int K, int group) {
  return N > 0 && K > 0 && K % 4 == 0 && (group == 32 || group == 64 || group == 128) &&
         q4_tiles(N) * q4_blocks(K) <= INT_MAX;
}

size_t q4_code_bytes(int N, int K) { return (size_t)q4_tiles(N) * q4_blocks(K) * 1024; }

}  // namespace
}  // namespace lx

using namespace lx;

extern "C" size_t lx_q4_bytes(int N, int K, int group) {
  if (!q4_shape_ok(N, K, group)) return 0;
  return q4_code_bytes(N, K) +
         (size_t)q4_tiles(N) * q4_blocks(K) * (kBlockK / group) * kTileN * sizeof(unsigned short);
}

extern "C" int lx_q4_pack_f32(const float* W, void* Wq, int N, int K, int group,
                              hipStream_t stream) {
  LX_REQUIRE(W && Wq, "q4_pack: null pointer");
  LX_REQUIRE(q4_shape_ok(N, K, group), "q4_pack: bad shape N=%d K=%d group=%d", N, K, group);
  LX_REQUIRE(((uintptr_t)W | (uintptr_t)Wq) % 16 == 0, "q4_pack: unaligned");
  const int kb = (int)q4_blocks(K);
  const dim3 grid((unsigned)(q4_tiles(N) * kb));
  uintx4_t* codes = static_cast<uintx4_t*>(Wq);
  auto* scales =
      reinterpret_cast<unsigned short*>(static_cast<char*>(Wq) + q4_code_bytes(N, K));
  if (group == 32)
    hipLaunchKernelGGL(q4_pack_kernel<32>, grid, dim3(64), 0, stream, W, codes, scales, N, K, kb);
  else if (group == 64)
    hipLaunchKernelGGL(q4_pack_kernel<64>, grid, dim3(64), 0, stream, W, codes, scales, N, K, kb);
  else
    hipLaunchKernelGGL(q4_pack_kernel<128>, grid, dim3(64), 0, stream, W, codes, scales, N, K, kb);
  return check_launch("q4_pack_kernel");
}

extern "C" int lx_q4_unpack_f32(const void* Wq, float* W, int N, int K, int group,
                                hipStream_t stream) {
  LX_REQUIRE(W && Wq, "q4_unpack: null pointer");
  LX_REQUIRE(q4_shape_ok(N, K, group), "q4_unpack: bad shape N=%d K=%d group=%d", N, K, group);
  LX_REQUIRE((uintptr_t)Wq % 16 == 0, "q4_unpack: unaligned");
  const int kb = (int)q4_blocks(K);
  hipLaunchKernelGGL(q4_unpack_kernel, dim3((unsigned)(q4_tiles(N) * kb)), dim3(256), 0, stream,
                     static_cast<const unsigned*>(Wq),
                     reinterpret_cast<const unsigned short*>(static_cast<const char*>(Wq) +
                                                             q4_code_bytes(N, K)),
                     W, N, K, kb, group);
  return check_launch("q4_unpack_kernel");
}

extern "C" int lx_linear_q4_f32(const float* x, long ldx, const void* Wq, int group,
                                const float* bias, float* y, long ldy, int M, int N, int K,
                                const lx_epilogue* epi, hipStream_t stream) {
  LX_REQUIRE(x && Wq && y, "linear_q4: null pointer");
  LX_REQUIRE(q4_shape_ok(N, K, group), "linear_q4: bad shape N=%d K=%d group=%d", N, K, group);
  LX_REQUIRE(M >= 1 && M <= kMaxRows, "linear_q4: %d rows outside [1, %d]", M, kMaxRows);
  const int kind = epi ? epi->kind : LX_EPI_NONE;
  LX_REQUIRE(kind == LX_EPI_NONE || kind == LX_EPI_GELU_TANH || kind == LX_EPI_RESID ||
                 kind == LX_EPI_SWIGLU_PAIRED,
             "linear_q4: epilogue %d (none, GELU, residual or SwiGLU)", kind);
  LX_REQUIRE(kind != LX_EPI_SWIGLU_PAIRED || N % 2 == 0, "linear_q4: SwiGLU needs an even N");
  LX_REQUIRE(ldx >= K && ldx % 4 == 0 && ldy >= (kind == LX_EPI_SWIGLU_PAIRED ? N / 2 : N),
             "linear_q4: bad row stride ldx=%ld ldy=%ld", ldx, ldy);
  LX_REQUIRE(((uintptr_t)x | (uintptr_t)Wq) % 16 == 0 &&
                 ((uintptr_t)y | (uintptr_t)bias) % 4 == 0,
             "linear_q4: x and Wq must be 16-byte aligned");
  Q4Args a{};
  a.x = x;
  a.ldx = ldx;
  a.codes = static_cast<const uintx4_t*>(Wq);
  a.scales = reinterpret_cast<const unsigned short*>(static_cast<const char*>(Wq) +
                                                     q4_code_bytes(N, K));
  a.bias = bias;
  a.y = y;
  a.ldy = ldy;
  a.M = M;
  a.N = N;
  a.K = K;
  a.kb = (int)q4_blocks(K);
  a.epi = kind;
  if (M <= kPackedCols) return launch_linear<1, true>(a, group, stream);
  switch ((M + 15) / 16) {
    case 1: return launch_linear<1, false>(a, group, stream);
    case 2: return launch_linear<2, false>(a, group, stream);
    case 3: return launch_linear<3, false>(a, group, stream);
    default: return launch_linear<4, false>(a, group, stream);
  }
}
