// Projections of few rows on 4-bit weights with group scales.
//
//   w~[n, k] = s[n, k / G] * (q[n, k] - 8),  y = epi(x w~^T + bias),  G = 32, 64 or 128.
//
// What bounds large weights is their stream (half a byte a weight), so the codes go from memory
// to the matrix cores with nine instructions for eight of them (lx_four_bit.hpp) and the scale is
// applied once per group to the fp32 sum, not to the weights.  x enters as two fp16 parts after a
// power of two per row and block of 128 inputs, so every product is exact.  Three kernels: one
// that stages up to 8 rows per wave, one that keeps up to 64 in registers, one for the single
// normalised row of the LM's decode.
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
constexpr long kMaxTiles = (1L << 24) - 1;  // of a weight: every launch below 2^32 threads

struct Q4Args {
  const float* x;
  long ldx;
  const uintx4_t* codes;
  const unsigned short* scales;
  const float* bias;
  float* y;
  long ldy;
  int M, N, K, kb, epi;
  int vec;  // y, its rows and bias 16-byte aligned
  int splits;
  float* ws;
};

__host__ __device__ inline long q4_tiles(int N) { return (N + kTileN - 1) / kTileN; }
__host__ __device__ inline long q4_blocks(int K) { return (K + kBlockK - 1) / kBlockK; }

// ---- quantise and lay out ---------------------------------------------------------------

// One wave per (row tile, block): lane l holds row l % 16, inputs 32 t + 8 (l / 16) + j.  Run once
// a weight; the fp32 matrix bounds it: 8192 x 8192 in groups of 128 66 us (4.6 TB/s; of 32, whose
// scales are four times as many, 76), 151936 x 896 171 us (3.6).  A copy asks 57 and 116.
// neox:// rows 2 i and 2 i + 1 of a head of 64 are its rows i and i + 32, a rotary pair, side by side.
template <int G>
__global__ __launch_bounds__(64) void q4_pack_kernel(const float* __restrict__ W,
                                                     uintx4_t* __restrict__ codes,
                                                     unsigned short* __restrict__ scales, int N,
                                                     int K, int kb, int neox) {
  constexpr int TG = G / 32;  // 32-wide steps of a group
  const int lane = threadIdx.x, c = lane >> 4, r = lane & 15;
  const long tile = blockIdx.x;  // row tile * kb + block
  const long n = tile / kb * kTileN + r;
  const long src = neox ? (n & ~63L) + ((n & 63) >> 1) + (n & 1) * 32 : n;
  const int k0 = (int)(tile % kb) * kBlockK;
  float w[4][8];
#pragma unroll
  for (int t = 0; t < 4; ++t)
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = k0 + 32 * t + 8 * c + 4 * e;
      const float4 v = n < N && k < K ? *reinterpret_cast<const float4*>(W + src * K + k)
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

// One thread per eight codes.  A lane writes 32 bytes of a row, 16 rows a wave: 8192 x 8192 315 us
// (1 TB/s), which a copy moves in 57.  For checks and for going back to fp32; no step runs it.
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

// bias and residual of output (m, n) [SwiGLU: of the pair n, n + 1], and the epilogue.
struct Q4EpiIn {
  float b0, b1, y;
};
__device__ __forceinline__ Q4EpiIn q4_epi_load(const Q4Args& a, int m, long n) {
  Q4EpiIn in = {0.0f, 0.0f, 0.0f};
  if (a.bias) {
    in.b0 = a.bias[n];
    if (a.epi == LX_EPI_SWIGLU_PAIRED) in.b1 = a.bias[n + 1];
  }
  if (a.epi == LX_EPI_RESID) in.y = a.y[m * a.ldy + n];
  return in;
}
__device__ __forceinline__ void q4_epi_store(const Q4Args& a, int m, long n, float v, float v1,
                                             const Q4EpiIn& in) {
  v += in.b0;
  if (a.epi == LX_EPI_SWIGLU_PAIRED) {
    a.y[m * a.ldy + (n >> 1)] = (v / (1.0f + expf(-v))) * (v1 + in.b1);
    return;
  }
  a.y[m * a.ldy + n] = a.epi == LX_EPI_GELU_TANH ? gelu_tanh(v)
                       : a.epi == LX_EPI_RESID   ? in.y + v
                                                 : v;
}

// Outputs n .. n + 3 (n a multiple of 4) of row m.
__device__ __forceinline__ void q4_epi_quad(const Q4Args& a, int m, long n, floatx4 v) {
  if (a.vec && n + 3 < a.N) {
    if (a.bias) v += *reinterpret_cast<const floatx4*>(a.bias + n);
    if (a.epi == LX_EPI_SWIGLU_PAIRED) {
      const float2 o = make_float2((v[0] / (1.0f + expf(-v[0]))) * v[1],
                                   (v[2] / (1.0f + expf(-v[2]))) * v[3]);
      *reinterpret_cast<float2*>(a.y + m * a.ldy + (n >> 1)) = o;
      return;
    }
    floatx4* y = reinterpret_cast<floatx4*>(a.y + m * a.ldy + n);
    if (a.epi == LX_EPI_GELU_TANH)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = gelu_tanh(v[e]);
    if (a.epi == LX_EPI_RESID) v = *y + v;
    *y = v;
    return;
  }
  const int step = a.epi == LX_EPI_SWIGLU_PAIRED ? 2 : 1;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e % step == 0 && n + e < a.N)
      q4_epi_store(a, m, n + e, v[e], v[e | 1], q4_epi_load(a, m, n + e));
}

// At most MB rows of x.  A workgroup owns one tile of 16 weight rows; its waves take the blocks
// of K in turn, each splitting its own 128 inputs of x into a slice of LDS (16 lanes a row, four
// rows at a time), and their sums meet in LDS at the end (in a fixed order).  Column 2 m + part of
// the fragments is a part of row m.  Everything a wave reads is requested before it computes, and
// the next block before this one; what remains is a launch, one memory round trip, the split
// (some 60 instructions a block) and the meeting: in a graph over eight weights in turn 1 row x
// 1152 x 896 3.2 us, x 9728 4.2 (1.1 TB/s), 4 rows x 896 x 4864 4.8, 8 rows x 9728 x 896 5.6, where
// a copy asks 0.1 to 0.9.  (With a lane per row of x each load touched 64 lines: 3 rows x 6761 5.4
// us, now 3.6.)
constexpr int kFewRow = 272;  // bytes of a staged row (128 fp16, and 16 against bank conflicts)

template <int MB>
constexpr int few_bytes() { return 2 * MB * kFewRow + 64; }  // rows, then 16 inverse scales

template <int MB, int G>
struct FewIn {
  static constexpr int NG = kBlockK / G;
  uintx4_t w;
  ushortx4_t sc[NG];
  float4 x[MB / 4][2];
  __device__ __forceinline__ void load(const Q4Args& a, long rt, int kb, int lane) {
    const long tile = rt * a.kb + kb;
    w = a.codes[tile * 64 + lane];
    const ushortx4_t* sp =
        reinterpret_cast<const ushortx4_t*>(a.scales) + (tile * 4 + (lane >> 4)) * NG;
#pragma unroll
    for (int g = 0; g < NG; ++g) sc[g] = sp[g];
    const int k = kb * kBlockK + 8 * (lane & 15);
#pragma unroll
    for (int p = 0; p < MB / 4; ++p) {
      const float* xr = a.x + (long)min(4 * p + (lane >> 4), a.M - 1) * a.ldx;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        x[p][e] = *reinterpret_cast<const float4*>(xr + min(k + 4 * e, a.K - 4));
    }
  }
};

template <int MB, int G>
__global__ __launch_bounds__(1024) void q4_few_kernel(Q4Args a) {
  constexpr int TG = G / 32, NG = kBlockK / G;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // [waves][few_bytes]
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane >> 4, col = lane & 15;
  const unsigned pattern = q4_pattern();
  const long rt = blockIdx.x;
  char* mine = lds + wave * few_bytes<MB>();
  float* finv = reinterpret_cast<float*>(mine + 2 * MB * kFewRow);
  const int step = a.epi == LX_EPI_SWIGLU_PAIRED ? 2 : 1;
  const int rshift = step == 2 ? 3 : 4, nout = a.M << rshift;  // 8 or 16 outputs a row of x
  // four threads an output in the end; what its epilogue reads is requested first
  FewIn<MB, G> in;
  in.load(a, rt, wave, lane);
  Q4EpiIn pre = {0.0f, 0.0f, 0.0f};
  {
    const int i = tid >> 2, m = i >> rshift;
    const long n = rt * kTileN + (i & ((1 << rshift) - 1)) * step;
    if (i < nout && n < a.N) pre = q4_epi_load(a, m, n);
  }
  floatx4 tot = {0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < a.kb; kb += waves) {
    if (kb * kBlockK + kBlockK > a.K) {
      asm volatile("");  // a branch, not a select per value of every block
#pragma unroll
      for (int p = 0; p < MB / 4; ++p)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          if (kb * kBlockK + 8 * col + 4 * e >= a.K) in.x[p][e] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    float top[MB / 4];
    tops16(in.x, top);
#pragma unroll
    for (int p = 0; p < MB / 4; ++p) {
      const float4 x0 = in.x[p][0], x1 = in.x[p][1];
      const float v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
      float inv;
      const float sc = row_scale(top[p], &inv);
      if (col == 0) finv[4 * p + c] = inv;
      half8_t p0, p1;
      split2(v, sc, p0, p1);
      char* row = mine + 2 * (4 * p + c) * kFewRow + col * 16;
      *reinterpret_cast<half8_t*>(row) = p0;
      *reinterpret_cast<half8_t*>(row + kFewRow) = p1;
    }
    const uintx4_t w = in.w;
    ushortx4_t sc[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) sc[g] = in.sc[g];
    if (kb + waves < a.kb) in.load(a, rt, kb + waves, lane);
    // the staged rows are this wave's own: in program order, no barrier
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const char* xr = mine + min(col, 2 * MB - 1) * kFewRow + c * 16;
    const float f = finv[min(col >> 1, MB - 1)];
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = g * TG; t < (g + 1) * TG; ++t) {
        acc = mfma_f16(q4_frag(w[t], pattern), *reinterpret_cast<const half8_t*>(xr + t * 64), acc);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sum[i] = fmaf(bf16_lo(sc[g][i]), acc[i], sum[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) tot[i] = fmaf(f, sum[i], tot[i]);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) reinterpret_cast<float*>(mine)[i * 64 + lane] = tot[i];
  __syncthreads();
  // row r of the tile against row m of x; thread q of four takes every fourth wave
  const int q = tid & 3;
  auto value = [&](int r, int m) {
    float s = 0.0f;
#pragma unroll 2
    for (int w = q; w < waves; w += 4) {
      const float* p = reinterpret_cast<const float*>(lds + w * few_bytes<MB>()) + (r & 3) * 64 +
                       (r >> 2) * 16;
      s += p[2 * m + 1] + p[2 * m];
    }
    s += dpp_mov<kDppXor1>(s);
    s += dpp_mov<kDppXor2>(s);
    return s;
  };
  for (int i = tid >> 2; i < nout; i += blockDim.x >> 2) {
    const int m = i >> rshift, r = (i & ((1 << rshift) - 1)) * step;
    const long n = rt * kTileN + r;
    const float v = value(r, m), v1 = step == 2 ? value(r + 1, m) : 0.0f;
    if (q == 0 && n < a.N)
      q4_epi_store(a, m, n, v, v1, i == tid >> 2 ? pre : q4_epi_load(a, m, n));
  }
}

// One normalised row of x, as the LM's decode runs it (arguments and epilogues of dec_gemv).  W
// waves are one tile of 16 rows, each over its own NB blocks of K: a wave requests all its weights,
// forms its part of the normalised row and the two fp16 parts of that (2 NB values a lane, one
// power of two) and hands them to its lanes as fragments through LDS of its own.  The waves meet
// twice, for the sum of squares and for the sums of the tile.  DEC_QKV_ROPE reads rows laid out in
// rotary pairs (q4_pack_kernel's neox).  The length of a wave's own instructions bounds it: a token
// of the 24-layer LM (hidden 896, cache 1, groups of 64) 488 us with one wave a tile, 474 with two,
// 452 with four, 458 with eight.
constexpr int kRowWaves = 4;  // W

template <int G, int EPI, int NB>
__global__ __launch_bounds__(64 * kRowWaves) void q4_row_kernel(Q4Args a, DecGemvArgs d) {
  constexpr int TG = G / 32, NG = kBlockK / G, ROW = NB * 256 + 16, W = kRowWaves;
  __shared__ __attribute__((aligned(16))) char rows[W][2 * ROW];
  __shared__ float squares[W];
  __shared__ floatx4 sums[W][4];
  const int lane = threadIdx.x & 63, c = lane >> 4, col = lane & 15;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), first = wave * NB;
  char* mine = rows[wave];
  const unsigned pattern = q4_pattern();
  const long rt = blockIdx.x;
  const int kb = a.kb;
  float2 x[NB], g[NB];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int k = min((first + j) * kBlockK + 2 * lane, a.K - 2);
    x[j] = *reinterpret_cast<const float2*>(a.x + k);
    g[j] = *reinterpret_cast<const float2*>(d.norm_w + k);
  }
  uintx4_t w[NB];
  ushortx4_t sc[NB][NG];
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const long tile = rt * kb + min(first + j, kb - 1);
    w[j] = a.codes[tile * 64 + lane];
    const ushortx4_t* sp = reinterpret_cast<const ushortx4_t*>(a.scales) + (tile * 4 + c) * NG;
#pragma unroll
    for (int i = 0; i < NG; ++i) sc[j][i] = sp[i];
  }
  // what the epilogue of the lane's rows n .. n + 3 reads, under the weights' latency
  const long n = rt * kTileN + 4 * c;
  const int head = (int)(n >> 6), hc = (int)(n & 63) >> 1;
  int pos = 0;
  float b[4] = {0.f, 0.f, 0.f, 0.f}, sn[2] = {0.f, 0.f}, cs[2] = {1.f, 1.f};
  if (EPI == DEC_QKV_ROPE && wave == 0) {
    pos = *d.pos;
#pragma unroll
    for (int i = 0; i < 4; ++i) b[i] = d.bias[head * 64 + hc + (i >> 1) + 32 * (i & 1)];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float f = d.inv_freq[hc + i];
      if (head < d.rope_heads) sincosf((float)pos * f, &sn[i], &cs[i]);
    }
  }
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    if ((first + j) * kBlockK + 2 * lane >= a.K) x[j] = make_float2(0.f, 0.f);
    ss += x[j].x * x[j].x + x[j].y * x[j].y;
  }
  ss = wave_sum(ss);
  if (lane == 0) squares[wave] = ss;
  __syncthreads();
  ss = 0.0f;
#pragma unroll
  for (int i = 0; i < W; ++i) ss += squares[i];
  const float rs = 1.0f / sqrtf(ss / (float)a.K + d.eps);
  float top = 0.0f;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    x[j] = make_float2((x[j].x * rs) * g[j].x, (x[j].y * rs) * g[j].y);
    const int k = (first + j) * kBlockK + 2 * lane;
    if (EPI == DEC_HEAD && rt == 0 && d.y2 && k < a.K)
      *reinterpret_cast<float2*>(d.y2 + k) = x[j];
    top = fmaxf(top, fmaxf(fabsf(x[j].x), fabsf(x[j].y)));
  }
  float f;
  const float xs = row_scale(wave_max(top), &f);
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    half2_t p0, p1;
    split_pair(x[j].x, x[j].y, xs, p0, p1);
    *reinterpret_cast<half2_t*>(mine + j * 256 + lane * 4) = p0;
    *reinterpret_cast<half2_t*>(mine + ROW + j * 256 + lane * 4) = p1;
  }
  // the staged row is this wave's own: in program order, no barrier
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  const char* xr = mine + (col & 1) * ROW + c * 16;  // column 0: first parts, 1: second parts
  floatx4 tot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    if (first + j >= kb) break;
#pragma unroll
    for (int i = 0; i < NG; ++i) {
      floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = i * TG; t < (i + 1) * TG; ++t)
        acc = mfma_f16(q4_frag(w[j][t], pattern),
                       *reinterpret_cast<const half8_t*>(xr + j * 256 + t * 64), acc);
#pragma unroll
      for (int e = 0; e < 4; ++e) tot[e] = fmaf(bf16_lo(sc[j][i][e]), acc[e], tot[e]);
    }
  }
  floatx4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    tot[e] *= f;
    v[e] = tot[e] + dpp_mov<kDppXor1>(tot[e]);
  }
  if (col == 0) sums[wave][c] = v;
  __syncthreads();
  if (wave || col) return;
  v = sums[0][c];
#pragma unroll
  for (int i = 1; i < W; ++i) v += sums[i][c];
  if (EPI == DEC_QKV_ROPE) {
    const int cl = head * 64 + hc;
    float* dst = cl < d.q_cols ? d.y + cl
                 : cl < d.q_cols + d.kv_cols
                     ? d.k_cache + (long)pos * d.kv_cols + (cl - d.q_cols)
                     : d.v_cache + (long)pos * d.kv_cols + (cl - d.q_cols - d.kv_cols);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float x0 = v[2 * i] + b[2 * i], x1 = v[2 * i + 1] + b[2 * i + 1];
      dst[i] = x0 * cs[i] - x1 * sn[i];
      dst[32 + i] = x1 * cs[i] + x0 * sn[i];
    }
  } else if (EPI == DEC_SWIGLU) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (n + 2 * i < a.N)
        d.y[(n >> 1) + i] = (v[2 * i] / (1.0f + expf(-v[2 * i]))) * v[2 * i + 1];
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < a.N) d.y[n + e] = v[e];
  }
}

// Up to 64 rows of x in CT column tiles of 16.  The waves of a workgroup own one block of K each,
// of the at most eight of a split: a wave splits its 16 CT rows x 128 inputs of x once, keeps the
// fragments in registers (32 CT of them) and streams the weights of its block past them, RT tiles
// of 16 rows at a time, one group of tiles ahead.  The waves' sums meet in one of two LDS buffers
// (a barrier a group), added in wave order; each thread adds and finishes one quad of outputs.
// More than one split: partial sums into ws (splits, M, N up to 16), which q4_join_kernel adds in
// split order.  16 rows x 151936 x 896, 82 MB: 24 us in a graph over twelve weights in turn (3.4
// TB/s), 21 over three, which the last-level cache holds.  Every 16 rows more cost 8192 x 8192
// about 5 us (eight weights in turn, 16: 16.8, 32: 22.2, 48: 27.9, 64: 31.1, the join's 5 among
// them): their splitting, 100 instructions a lane, then matrix instructions at the clock the power
// limit leaves, and 4 MB of partial sums written and read.  (With x in LDS and whole K ranges a
// wave, every fragment of x is read again for every two tiles: 64 rows 8192 x 8192 33 us, 9728 x
// 896 17 for 11.3 now.  Sums of a group added under the next one's products, with one register
// buffer of weights for two: 33 us.)
constexpr int kManyWaves = 8;
constexpr int kManyTiles = 2;  // RT
constexpr size_t many_bytes(int ct) {
  const size_t sums = (size_t)2 * kManyWaves * kManyTiles * ct * 1024;
  const size_t split = (size_t)kManyWaves * few_bytes<16>();
  return sums > split ? sums : split;
}

template <int CT, int G>
__global__ __launch_bounds__(64 * kManyWaves) __attribute__((
    amdgpu_waves_per_eu(CT == 1 ? 4 : 2))) void q4_many_kernel(Q4Args a) {
  constexpr int TG = G / 32, NG = kBlockK / G, RT = kManyTiles;
  extern __shared__ __attribute__((aligned(16))) char lds[];  // [2][wave][RT][CT][lane] quads
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c = lane >> 4, col = lane & 15;
  const unsigned pattern = q4_pattern();
  const int sp = blockIdx.y, per = (a.kb + a.splits - 1) / a.splits;
  const int nb = min(per, a.kb - sp * per);  // blocks of this split, 1 .. 8: waves that multiply
  const int kb = sp * per + min(wave, nb - 1);
  const long tiles = q4_tiles(a.N);
  const int groups = (int)((tiles + RT - 1) / RT);
  uintx4_t w[RT], wn[RT];
  ushortx4_t sc[RT][NG], scn[RT][NG];
  auto load_w = [&](int group) {  // past the last group: the last
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      const long tile = min((long)group * RT + r, tiles - 1) * a.kb + kb;
      wn[r] = a.codes[tile * 64 + lane];
      const ushortx4_t* p = reinterpret_cast<const ushortx4_t*>(a.scales) + (tile * 4 + c) * NG;
#pragma unroll
      for (int g = 0; g < NG; ++g) scn[r][g] = p[g];
    }
  };
  load_w(blockIdx.x);
  half8_t xf[CT][4][2];
  float f[CT];
  {
    // 16 lanes a row, so that an instruction reads whole lines (a lane a row reads 64 of them:
    // 17000 accesses, 7 us, for 64 rows), then through this wave's slice of LDS
    char* mine = lds + wave * few_bytes<16>();
    float* finv = reinterpret_cast<float*>(mine + 32 * kFewRow);
    float4 u[CT][4][2];  // all requested before the first is used
    const long x4 = 4 * a.ldx;
    const int k0 = kb * kBlockK + 4 * col;
    const float* last = a.x + (a.M - 1) * a.ldx;
    const float* xr = a.x + c * a.ldx;
#pragma unroll
    for (int i = 0; i < 4 * CT; ++i, xr += x4) {
      const float* r = 4 * i + c < a.M ? xr : last;
#pragma unroll
      for (int e = 0; e < 2; ++e)
        u[i >> 2][i & 3][e] = *reinterpret_cast<const float4*>(r + min(k0 + 64 * e, a.K - 4));
    }
    if (kb * kBlockK + kBlockK > a.K) {
      asm volatile("");  // a branch, not a select per value of every block
#pragma unroll
      for (int i = 0; i < 8 * CT; ++i)
        if (k0 + 64 * (i & 1) >= a.K)
          u[i >> 3][i >> 1 & 3][i & 1] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
#pragma unroll
    for (int ct = 0; ct < CT; ++ct) {
      float top[4], inverse = 0.0f;
      tops16(u[ct], top);
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const float4 x0 = u[ct][p][0], x1 = u[ct][p][1];
        const float v[8] = {x0.x, x0.y, x0.z, x0.w, x1.x, x1.y, x1.z, x1.w};
        float inv;
        const float xs = row_scale(top[p], &inv);
        if (col == p) inverse = inv;
        half8_t p0, p1;
        split2(v, xs, p0, p1);
        const uintx4_t b0 = __builtin_bit_cast(uintx4_t, p0), b1 = __builtin_bit_cast(uintx4_t, p1);
        char* row = mine + 2 * (4 * p + c) * kFewRow + col * 8;
        *reinterpret_cast<uintx2_t*>(row) = uintx2_t{b0[0], b0[1]};
        *reinterpret_cast<uintx2_t*>(row + 128) = uintx2_t{b0[2], b0[3]};
        *reinterpret_cast<uintx2_t*>(row + kFewRow) = uintx2_t{b1[0], b1[1]};
        *reinterpret_cast<uintx2_t*>(row + kFewRow + 128) = uintx2_t{b1[2], b1[3]};
      }
      if (col < 4) finv[4 * col + c] = inverse;
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      f[ct] = finv[col];
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          xf[ct][t][p] = *reinterpret_cast<const half8_t*>(mine + (2 * col + p) * kFewRow + t * 64 +
                                                           c * 16);
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();  // the slices become the buffers of sums
  }
  if (wave >= nb)  // no block: zeros for good
#pragma unroll
    for (int i = 0; i < 2 * RT * CT; ++i)
      reinterpret_cast<floatx4*>(lds)[((i & 1) * kManyWaves + wave) * RT * CT * 64 +
                                      (i >> 1) * 64 + lane] = floatx4{0.f, 0.f, 0.f, 0.f};
  int buf = 0;
  for (int group = blockIdx.x; group < groups; group += gridDim.x, buf ^= 1) {
    char* red = lds + (size_t)buf * kManyWaves * RT * CT * 1024;
    if (wave < nb) {
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        w[r] = wn[r];
#pragma unroll
        for (int g = 0; g < NG; ++g) sc[r][g] = scn[r][g];
      }
      if (group + (int)gridDim.x < groups) load_w(group + gridDim.x);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        floatx4 tot[CT];
#pragma unroll
        for (int g = 0; g < NG; ++g) {
          floatx4 acc[CT];
#pragma unroll
          for (int ct = 0; ct < CT; ++ct) acc[ct] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int t = g * TG; t < (g + 1) * TG; ++t) {
            const half8_t wf = q4_frag(w[r][t], pattern);
#pragma unroll
            for (int p = 1; p >= 0; --p)
#pragma unroll
              for (int ct = 0; ct < CT; ++ct) acc[ct] = mfma_f16(wf, xf[ct][t][p], acc[ct]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float s = bf16_lo(sc[r][g][e]);
#pragma unroll
            for (int ct = 0; ct < CT; ++ct)
              tot[ct][e] = g == 0 ? s * acc[ct][e] : fmaf(s, acc[ct][e], tot[ct][e]);
          }
        }
#pragma unroll
        for (int ct = 0; ct < CT; ++ct) {
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[ct][e] *= f[ct];
          reinterpret_cast<floatx4*>(red)[((wave * RT + r) * CT + ct) * 64 + lane] = tot[ct];
        }
      }
    }
    __syncthreads();
    for (int u = tid; u < RT * CT * 64; u += 64 * kManyWaves) {
      const int ct = (u >> 6) % CT, r = (u >> 6) / CT;
      const int m = ct * 16 + col;
      const long tile = (long)group * RT + r, n = tile * kTileN + 4 * c;
      if (m >= a.M || tile >= tiles) continue;
      floatx4 s = reinterpret_cast<const floatx4*>(red)[u];
#pragma unroll
      for (int i = 1; i < kManyWaves; ++i)
        s += reinterpret_cast<const floatx4*>(red)[i * RT * CT * 64 + u];
      if (a.splits > 1)
        *reinterpret_cast<floatx4*>(a.ws + ((long)sp * a.M + m) * (tiles * kTileN) + n) = s;
      else
        q4_epi_quad(a, m, n, s);
    }
  }
}

// The splits' sums added in split order, and the epilogue: one thread per four rows of W (64 rows
// 8192 x 8192: 17 MB of sums in 4.6 us, 3.6 TB/s).
__global__ __launch_bounds__(256) void q4_join_kernel(Q4Args a) {
  const long np4 = q4_tiles(a.N) * (kTileN / 4);
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= np4 * a.M) return;
  const int m = (int)(i / np4);
  const long n = i % np4 * 4;
  const float* p = a.ws + ((long)m * np4) * 4 + n;
  floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k)
    s += *reinterpret_cast<const floatx4*>(p + (long)k * a.M * np4 * 4);
  q4_epi_quad(a, m, n, s);
}

#define LX_Q4_GROUPS(KERNEL, ...)                                        \
  if (G == 32)                                                           \
    hipLaunchKernelGGL((KERNEL<__VA_ARGS__, 32>), grid, block, lds, s, a);  \
  else if (G == 64)                                                      \
    hipLaunchKernelGGL((KERNEL<__VA_ARGS__, 64>), grid, block, lds, s, a);  \
  else                                                                   \
    hipLaunchKernelGGL((KERNEL<__VA_ARGS__, 128>), grid, block, lds, s, a);

template <int MB>
int launch_few(const Q4Args& a, int G, hipStream_t s) {
  const int waves = std::min(std::min(16, a.kb), 64 * 1024 / few_bytes<MB>());
  const dim3 grid((unsigned)q4_tiles(a.N)), block(64 * waves);
  const size_t lds = (size_t)waves * few_bytes<MB>();
  LX_Q4_GROUPS(q4_few_kernel, MB)
  return check_launch("q4_few_kernel");
}

// Splits of K of q4_many_kernel: at most a block a wave.
int many_splits(int K) { return (int)((q4_blocks(K) + kManyWaves - 1) / kManyWaves); }

template <int CT, int G>
int raise_many() {
  static LdsLimit once;
  return raise_lds_limit(reinterpret_cast<const void*>(q4_many_kernel<CT, G>), many_bytes(CT),
                         once, "q4_many_kernel");
}

template <int CT>
int launch_many(const Q4Args& a, int G, hipStream_t s) {
  LX_TRY(G == 32 ? (raise_many<CT, 32>())
                 : G == 64 ? (raise_many<CT, 64>()) : (raise_many<CT, 128>()));
  const long groups = (q4_tiles(a.N) + kManyTiles - 1) / kManyTiles;
  // as many workgroups as the CUs hold at once walk over the groups
  const long slots = (CT == 1 ? 2L : 1L) * device_cus();
  const dim3 grid((unsigned)std::min(groups, std::max(1L, slots / a.splits)), a.splits),
      block(64 * kManyWaves);
  const size_t lds = many_bytes(CT);
  LX_Q4_GROUPS(q4_many_kernel, CT)
  return check_launch("q4_many_kernel");
}
#undef LX_Q4_GROUPS

// Calls that run on q4_few_kernel, which has little fixed cost but splits x again for every tile;
// in units of tile x block, and more where the other kernel needs a second launch (K > 1024).
// Times of both in a graph over eight weights in turn, us (few / many): K = 896, M = 4, N = 27000
// (work 11816) 7.3 / 7.8, N = 32000 (14000) 8.1 / 7.8, N = 40000 9.5 / 8.6; M = 8, N = 9728 (4256)
// 5.6 / 6.3, N = 20000 (8750) 7.6 / 7.0; M = 8, N = 896, K = 4864 5.9 / 6.9, 4096 x 8192 (16384)
// 9.3 / 10.9, 8192 x 8192 (32768) 17.6 / 15.3.
// Up to 4 rows with K > 1024 always run here, since such a call takes no workspace.  M = 4: 896 x
// 4864 (2128) 4.8 / 6.8, 20000 x 1100 (11250) 7.6 / 11.5, 8192 x 8192 (32768) 14.1 / 15.6; past
// some 35000 the other kernel would win: 3 x 70000 x 1100 (39375) 22.7 / 20.7, 28672 x 8192
// (114688) 41.5 / 33.6, 151936 x 2048 (151936) 72.7 / 43.6.
bool q4_takes_few(int M, int N, int K) {
  const long kb = q4_blocks(K), work = q4_tiles(N) * kb;
  if (M <= 4) return kb > kManyWaves || work <= 14000;
  return M <= 8 && work <= (kb > kManyWaves ? 20000 : 6000);
}

bool q4_shape_ok(int N, int K, int group) {
  return N > 0 && K > 0 && K % 4 == 0 && (group == 32 || group == 64 || group == 128) &&
         q4_tiles(N) * q4_blocks(K) <= kMaxTiles;
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

namespace lx {

size_t q4_bytes(int N, int K, int group) { return lx_q4_bytes(N, K, group); }

int q4_pack(const float* W, void* Wq, int N, int K, int group, int neox, hipStream_t stream) {
  LX_REQUIRE(W && Wq, "q4_pack: null pointer");
  LX_REQUIRE(q4_shape_ok(N, K, group) && (!neox || N % 64 == 0),
             "q4_pack: bad shape N=%d K=%d group=%d", N, K, group);
  LX_REQUIRE(((uintptr_t)W | (uintptr_t)Wq) % 16 == 0, "q4_pack: unaligned");
  const int kb = (int)q4_blocks(K);
  const dim3 grid((unsigned)(q4_tiles(N) * kb));
  uintx4_t* codes = static_cast<uintx4_t*>(Wq);
  auto* scales =
      reinterpret_cast<unsigned short*>(static_cast<char*>(Wq) + q4_code_bytes(N, K));
  if (group == 32)
    hipLaunchKernelGGL(q4_pack_kernel<32>, grid, dim3(64), 0, stream, W, codes, scales, N, K, kb,
                       neox);
  else if (group == 64)
    hipLaunchKernelGGL(q4_pack_kernel<64>, grid, dim3(64), 0, stream, W, codes, scales, N, K, kb,
                       neox);
  else
    hipLaunchKernelGGL(q4_pack_kernel<128>, grid, dim3(64), 0, stream, W, codes, scales, N, K, kb,
                       neox);
  return check_launch("q4_pack_kernel");
}

namespace {
template <int EPI, int NB>
int launch_row(const Q4Args& a, const DecGemvArgs& d, int G, hipStream_t s) {
  const dim3 grid((unsigned)q4_tiles(a.N)), block(64 * kRowWaves);
  if (G == 32)
    hipLaunchKernelGGL((q4_row_kernel<32, EPI, NB>), grid, block, 0, s, a, d);
  else if (G == 64)
    hipLaunchKernelGGL((q4_row_kernel<64, EPI, NB>), grid, block, 0, s, a, d);
  else
    hipLaunchKernelGGL((q4_row_kernel<128, EPI, NB>), grid, block, 0, s, a, d);
  return check_launch("q4_row_kernel");
}
}  // namespace

int dec_gemv_q4(int epi, const DecGemvArgs& d, const void* Wq, int group, hipStream_t s) {
  LX_REQUIRE(Wq && d.x && d.y && d.N <= INT_MAX && q4_shape_ok((int)d.N, d.K, group),
             "dec_gemv_q4: bad args");
  const int N = (int)d.N;
  if (epi == DEC_RESID) {
    lx_epilogue resid{};
    resid.kind = LX_EPI_RESID;
    return lx_linear_q4_f32(d.x, d.K, Wq, group, nullptr, d.y, N, 1, N, d.K, &resid, nullptr, 0,
                            s);
  }
  LX_REQUIRE(d.norm_w && d.K <= 2048, "dec_gemv_q4: norm args");
  Q4Args a{};
  a.x = d.x;
  a.codes = static_cast<const uintx4_t*>(Wq);
  a.scales = reinterpret_cast<const unsigned short*>(static_cast<const char*>(Wq) +
                                                     q4_code_bytes(N, d.K));
  a.N = N;
  a.K = d.K;
  a.kb = (int)q4_blocks(d.K);
  const bool wide = a.kb > 8;
  switch (epi) {
    case DEC_QKV_ROPE:
      LX_REQUIRE(N % 64 == 0 && d.bias && d.pos && d.k_cache && d.v_cache && d.inv_freq,
                 "dec_gemv_q4: qkv args");
      return wide ? launch_row<DEC_QKV_ROPE, 16 / kRowWaves>(a, d, group, s)
                  : launch_row<DEC_QKV_ROPE, 8 / kRowWaves>(a, d, group, s);
    case DEC_SWIGLU:
      LX_REQUIRE(N % 2 == 0, "dec_gemv_q4: swiglu needs an even N");
      return wide ? launch_row<DEC_SWIGLU, 16 / kRowWaves>(a, d, group, s)
                  : launch_row<DEC_SWIGLU, 8 / kRowWaves>(a, d, group, s);
    case DEC_HEAD:
      return wide ? launch_row<DEC_HEAD, 16 / kRowWaves>(a, d, group, s)
                  : launch_row<DEC_HEAD, 8 / kRowWaves>(a, d, group, s);
  }
  set_error("dec_gemv_q4: unsupported epilogue %d", epi);
  return LX_ERR_ARG;
}

}  // namespace lx

extern "C" int lx_q4_pack_f32(const float* W, void* Wq, int N, int K, int group,
                              hipStream_t stream) {
  return q4_pack(W, Wq, N, K, group, 0, stream);
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

extern "C" size_t lx_linear_q4_ws_floats(int M, int N, int K) {
  if (M < 1 || M > kMaxRows || !q4_shape_ok(N, K, 64) || q4_takes_few(M, N, K)) return 0;
  const int splits = many_splits(K);
  return splits == 1 ? 0 : (size_t)splits * M * q4_tiles(N) * kTileN;
}

extern "C" int lx_linear_q4_f32(const float* x, long ldx, const void* Wq, int group,
                                const float* bias, float* y, long ldy, int M, int N, int K,
                                const lx_epilogue* epi, float* ws, size_t ws_floats,
                                hipStream_t stream) {
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
  LX_REQUIRE(!rows_overlap(x, ldx, K, y, ldy, kind == LX_EPI_SWIGLU_PAIRED ? N / 2 : N, M),
             "linear_q4: y overlaps x");
  Q4Args a{};
  a.x = x;
  a.ldx = ldx;
  a.codes = static_cast<const uintx4_t*>(Wq);
  a.scales = reinterpret_cast<const unsigned short*>(static_cast<const char*>(Wq) +
                                                     q4_code_bytes(N, K));
  a.bias = bias;
  a.y = y;
  a.ldy = ldy;
  a.vec = ldy % 4 == 0 && ((uintptr_t)y | (uintptr_t)bias) % 16 == 0;
  a.M = M;
  a.N = N;
  a.K = K;
  a.kb = (int)q4_blocks(K);
  a.epi = kind;
  a.splits = 1;
  if (q4_takes_few(M, N, K)) {
    if (M <= 4) return launch_few<4>(a, group, stream);
    return launch_few<8>(a, group, stream);
  }
  a.splits = many_splits(K);
  if (a.splits > 1) {
    LX_REQUIRE(a.splits <= 65535, "linear_q4: K=%d of %d rows too long", K, M);
    const size_t need = (size_t)a.splits * M * q4_tiles(N) * kTileN;
    LX_REQUIRE(ws && ws_floats >= need && (uintptr_t)ws % 16 == 0,
               "linear_q4: workspace of %zu floats, %zu needed", ws ? ws_floats : 0, need);
    a.ws = ws;
  }
  switch ((M + 15) / 16) {
    case 1: LX_TRY(launch_many<1>(a, group, stream)); break;
    case 2: LX_TRY(launch_many<2>(a, group, stream)); break;
    case 3: LX_TRY(launch_many<3>(a, group, stream)); break;
    default: LX_TRY(launch_many<4>(a, group, stream)); break;
  }
  if (a.splits == 1) return LX_OK;
  const long n = q4_tiles(N) * (kTileN / 4) * M;
  hipLaunchKernelGGL(q4_join_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, stream, a);
  return check_launch("q4_join_kernel");
}
