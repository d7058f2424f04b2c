// y = epi(x~ W~^T + bias), both operands in 8 bits with a power of two per block of 128
// (lx_q8.hpp).
#include <algorithm>
#include <climits>

#include "lx_q8.hpp"

namespace lx {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
// floats at a 4-byte boundary: y, bias and resid need no other (their vectors reach memory in one
// instruction on gfx950 all the same; rows of an odd N by single floats cost 30%)
typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef float float2u __attribute__((ext_vector_type(2), aligned(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

struct Q8Lin {
  Q8Mat x, w;
  const float* bias;
  const float* resid;
  float* y;
  long ldr, ldy;
  int epi;
  int tiles_m, tiles_n, band;  // of the launch
};

// x / (1 + e^-x) on the hardware's exponential and reciprocal, each within an ulp or so.  v^2 (1 + r)
// is e^-x: v = 2^y with y the rounded -x log2(e) / 2, r what -x - 2 y ln(2) leaves, so that the
// exponential keeps its relative error far from zero.  (Against expf and a division a third of the
// instructions; 256 x 9728 x 896 12.5 -> 11.9 us.)  1 + v^2 is formed in units of 2^32: nothing
// overflows or leaves the normal numbers before the last products, so that x down to the type's
// lowest value gives -0 (the factor is 0 from -105 on: e^-105 < 2^-150) and x up to the largest, and
// infinity, gives x.
__device__ __forceinline__ float silu_hw(float x) {
  constexpr float kUnit = 0x1p-32f;
  const float c = fminf(fmaxf(x, -105.0f), 105.0f), y = c * -0.7213475204444817f;
  const float r = fmaf(y, 3.80930853e-9f, fmaf(y, -1.3862943611198906f, -c));
  const float v = __builtin_amdgcn_exp2f(y);
  const float d = fmaf(v * kUnit, fmaf(v, r, v), kUnit);
  return x * (__builtin_amdgcn_rcpf(d) * kUnit);
}

// What the residual holds at columns n .. n + 3 of row m.  Asked for ahead of the sums, since it comes
// from memory: 4096 x 896 x 896 18.2 -> 16.1 us.
__device__ __forceinline__ floatx4 resid_quad(const Q8Lin& a, int m, long n) {
  floatx4 r{0.f, 0.f, 0.f, 0.f};
  if (m >= a.x.rows) return r;
  const float* p = a.resid + m * a.ldr + n;
  if (n + 3 < a.w.rows) return *reinterpret_cast<const float4u*>(p);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < a.w.rows) r[e] = p[e];
  return r;
}

__device__ __forceinline__ void epi_one(const Q8Lin& a, int m, long n, float v, float up, float r) {
  if (a.bias) v += a.bias[n];
  if (a.epi == LX_EPI_SWIGLU_PAIRED) {
    if (a.bias) up += a.bias[n + 1];
    a.y[m * a.ldy + (n >> 1)] = silu_hw(v) * up;
    return;
  }
  if (a.epi == LX_EPI_GELU_TANH) v = gelu_tanh(v);
  if (a.epi == LX_EPI_RESID) v = r + v;
  a.y[m * a.ldy + n] = v;
}

// Columns n .. n + 3 (n a multiple of 4) of row m; r: their residual.
__device__ __forceinline__ void epi_quad(const Q8Lin& a, int m, long n, floatx4 v, floatx4 r) {
  if (m >= a.x.rows) return;
  if (n + 3 < a.w.rows) {
    if (a.bias) v += *reinterpret_cast<const float4u*>(a.bias + n);
    if (a.epi == LX_EPI_SWIGLU_PAIRED) {
      *reinterpret_cast<float2u*>(a.y + m * a.ldy + (n >> 1)) = float2u{
          silu_hw(v[0]) * v[1], silu_hw(v[2]) * v[3]};
      return;
    }
    if (a.epi == LX_EPI_GELU_TANH)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = gelu_tanh(v[e]);
    if (a.epi == LX_EPI_RESID) v = r + v;
    *reinterpret_cast<float4u*>(a.y + m * a.ldy + n) = v;
    return;
  }
  const int step = a.epi == LX_EPI_SWIGLU_PAIRED ? 2 : 1;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e % step == 0 && n + e < a.w.rows) epi_one(a, m, n + e, v[e], v[e | 1], r[e]);
}

// Codes as operands of the bf16 matrix instructions: exact, eight bits hold e4m3's four, and the
// power of two comes with the conversion (v_cvt_scalef32_pk_bf16_fp8, two codes an instruction; it
// reads the scale's exponent field alone, so the bits of 0.0f are 2^-127, and what lies between
// bf16's subnormal numbers, multiples of 2^-133, goes to the nearest).
// The 8-bit matrix instructions would take the codes as they are at twice the rate, but they add
// the products of eight neighbours with some 13 bits below the largest of them, 1.5e-5 of a sum
// where these keep fp32's 1e-7.
__device__ __forceinline__ bf16x8_t q8_frag(int lo, int hi, float scale) {
  const bf16x2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false);
  const bf16x2_t b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
  const bf16x2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false);
  const bf16x2_t d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
  return bf16x8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// Up to 16 rows.  A workgroup owns 16 MT rows of x and 16 NT rows of W; its waves take the blocks
// of K in turn, straight from memory to registers, and their sums meet in LDS.  W is the
// instruction's A operand: a lane's four sums are four consecutive columns of one row of y.  Bound
// by the weights' bytes (16 x 8192 x 8192 12.7 us, 5.3 TB/s; 16 x 151936 x 896 28.7, 4.8) or a launch
// and one round trip (1 x 1152 x 896 2.6 us in a graph).
template <int MT, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void q8_stream_kernel(Q8Lin a) {
  extern __shared__ __attribute__((aligned(16))) floatx4 red[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int mt = blockIdx.x % a.tiles_m, nt = blockIdx.x / a.tiles_m;
  const int r = lane & 15, c = lane >> 4;
  const int at = q8_chunk(r, c);
  const int mtiles = (a.x.rows + 15) / 16, ntiles = (a.w.rows + 15) / 16;
  long xt[MT], wt[NT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xt[i] = min(mt * MT + i, mtiles - 1);
#pragma unroll
  for (int i = 0; i < NT; ++i) wt[i] = min(nt * NT + i, ntiles - 1);
  floatx4 acc[NT][MT];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) acc[n][m] = floatx4{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < a.x.kb; kb += WAVES) {
    intx4 xf[MT][2], wf[NT][2];
    float xs[MT], ws[NT];
    const int so = kb * 16 + r;
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const unsigned char* p = a.w.codes + (wt[i] * a.w.kb + kb) * kQ8Tile;
      wf[i][0] = *reinterpret_cast<const intx4*>(p + at);
      wf[i][1] = *reinterpret_cast<const intx4*>(p + at + kQ8Tile / 2);
      ws[i] = __uint_as_float((unsigned)a.w.scales[wt[i] * a.w.kb * 16 + so] << 23);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const unsigned char* p = a.x.codes + (xt[i] * a.x.kb + kb) * kQ8Tile;
      xf[i][0] = *reinterpret_cast<const intx4*>(p + at);
      xf[i][1] = *reinterpret_cast<const intx4*>(p + at + kQ8Tile / 2);
      xs[i] = __uint_as_float((unsigned)a.x.scales[xt[i] * a.x.kb * 16 + so] << 23);
    }
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      bf16x8_t xb[MT];
#pragma unroll
      for (int m = 0; m < MT; ++m)
        xb[m] = q8_frag(xf[m][t >> 1][2 * (t & 1)], xf[m][t >> 1][2 * (t & 1) + 1], xs[m]);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const bf16x8_t wb =
            q8_frag(wf[n][t >> 1][2 * (t & 1)], wf[n][t >> 1][2 * (t & 1) + 1], ws[n]);
#pragma unroll
        for (int m = 0; m < MT; ++m)
          acc[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wb, xb[m], acc[n][m], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int m = 0; m < MT; ++m) red[((wave * NT + n) * MT + m) * 64 + lane] = acc[n][m];
  __syncthreads();
  for (int u = tid; u < NT * MT * 64; u += 64 * WAVES) {
    floatx4 s = red[u];
#pragma unroll
    for (int i = 1; i < WAVES; ++i) s += red[i * NT * MT * 64 + u];
    const int m = (u >> 6) % MT, n = (u >> 6) / MT, l = u & 63;
    const int row = (mt * MT + m) * 16 + (l & 15);
    const long col = (long)(nt * NT + n) * 16 + 4 * (l >> 4);
    floatx4 res{};
    if (a.epi == LX_EPI_RESID) res = resid_quad(a, row, col);
    epi_quad(a, row, col, s, res);
  }
}

// This workgroup's tile of y.  Each XCD (workgroups are dealt to them round-robin) takes a
// contiguous run of tiles, which go down and then along bands of a.band rows of tiles: about a
// square, the fewest bytes for its L2 (4096 x 8192 x 8192 442 -> 423 us against runs of columns).
__device__ __forceinline__ void tile_at(const Q8Lin& a, int& mt, int& nt) {
  int id = blockIdx.x;
  const int full = gridDim.x / 8 * 8;
  if (id < full) id = (id % 8) * (full / 8) + id / 8;
  const int band = id / (a.band * a.tiles_n), in_band = id % (a.band * a.tiles_n);
  const int high = min(a.band, a.tiles_m - band * a.band);
  mt = band * a.band + in_band % high;
  nt = in_band / high;
}
int tile_grid(Q8Lin& a, int rows, int cols, int threads, long* grid) {
  a.tiles_m = (int)(((long)a.x.rows + rows - 1) / rows);
  a.tiles_n = (int)(((long)a.w.rows + cols - 1) / cols);
  *grid = (long)a.tiles_m * a.tiles_n;
  LX_REQUIRE(*grid <= INT_MAX / threads, "linear_q8: %d x %d outputs are too many", a.x.rows,
             a.w.rows);
  a.band = 1;
  while (a.band < a.tiles_m && (long)(a.band + 1) * (a.band + 1) * 8 <= *grid) ++a.band;
  return LX_OK;
}

template <int N>
__device__ __forceinline__ void wait_vm() {  // vmcnt(N) lgkmcnt(0)
  __builtin_amdgcn_s_waitcnt((N & 15) | (N >> 4 & 3) << 14 | 7 << 4);
  asm volatile("" ::: "memory");  // no read of LDS moves in front of it
}

// Many rows.  A workgroup owns (32 RB WM) x (32 CB WN) outputs; both operands go through LDS as
// they lie in memory (no registers, no ds_write), a block of K a stage, two stages.  WK waves share
// each (32 RB) x (32 CB) of the outputs, taking 128 / WK of a stage's 128 each: what a tile costs
// beside its products is the conversion of its operands (8 cycles for 128 codes; an instruction of
// 32 x 32 x 16 takes 32), less of it the larger a wave's tile is, and the way of its WK partial
// sums through LDS (256 x 9728 x 896 on 64 x 64: 2 us of 11.5 with WK = 4, three workgroups a CU;
// 10.7 with WK = 2 and four; 10.6 to 10.9 with 1).  A step is 16 of K; while its products run, the
// next step's codes are converted, and those of the step after are on their way from LDS.  The one
// barrier of a stage stands before its last two steps, whose operands every wave has by then: the
// buffer is free for the stage after the next, and the next stage's first reads return behind those
// steps' products.  4096 x 8192 x 8192 on 256 x 256 tiles: 400-455 us by box and heat, 1.2-1.38
// PFLOP/s, as a bf16 product of the library (1.37): the power limit leaves 1.8 GHz, at which the
// matrix pipe is 0.65 to 0.68 busy; four waves of 128 x 128 and eight of 64 x 128 give the same.
// 1000 x 6761 x 896 on 128 x 128: 18.7 us with eight waves of 64 x 32, 20.0 with four of 64 x 64.
template <int RB, int CB, int WM, int WN, int WK>
struct TileShape {
  static constexpr int WAVES = WM * WN * WK;
  static constexpr int XT = 2 * RB * WM, WT = 2 * CB * WN;  // 16-row tiles of a stage
  static constexpr int PIECES = (XT + WT) * 2;              // 1 KB each, of a stage
  static constexpr int CHUNKS = (PIECES + WAVES - 1) / WAVES;  // a wave's; the last repeat
  static_assert(XT + WT <= 16 * WAVES, "a wave loads the scales of 16 tiles");
  static constexpr int SCALES = WAVES * CHUNKS * 1024;  // of a stage, then 256 bytes a wave
  static constexpr int STAGE = SCALES + 256 * WAVES;
  static constexpr int ROW = 32 * CB + 4;  // floats of a row of outputs in LDS
  static constexpr int OUT = 32 * ROW * 4;  // a wave's 32 rows
  static constexpr int LDS = 2 * STAGE > WAVES * OUT ? 2 * STAGE : WAVES * OUT;
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static_assert(WK <= 2 && CHUNKS + 1 < 64, "four steps or more; vmcnt");
};

template <int RB, int CB, int WM, int WN, int WK, int OCC>
__global__ __launch_bounds__(64 * WM * WN * WK, OCC) void q8_tile_kernel(Q8Lin a) {
  using S = TileShape<RB, CB, WM, WN, WK>;
  constexpr int XT = S::XT, WT = S::WT, CHUNKS = S::CHUNKS, SPW = 4 / WK;
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int wk = wave % WK, wm = wave / WK % WM, wn = wave / (WK * WM);
  int mt, nt;
  tile_at(a, mt, nt);
  const int mtiles = (a.x.rows + 15) / 16, ntiles = (a.w.rows + 15) / 16;
  const int kb = a.x.kb;
  // tile t of a stage: rows of x, then of W; past the last it repeats that
  auto tile_of = [&](int t) {
    return t < XT ? min(mt * XT + t, mtiles - 1) : min(nt * WT + min(t - XT, WT - 1), ntiles - 1);
  };
  const unsigned char* src[CHUNKS];
#pragma unroll
  for (int j = 0; j < CHUNKS; ++j) {
    const int c = wave * CHUNKS + j, t = c >> 1;
    src[j] = (t < XT ? a.x.codes : a.w.codes) + (long)tile_of(t) * kb * kQ8Tile + (c & 1) * 1024 +
             lane * 16;
  }
  const unsigned char* ssrc;
  {
    const int t = wave * 16 + (lane >> 2);
    ssrc = (t < XT ? a.x.scales : a.w.scales) + (long)tile_of(t) * kb * 16 + (lane & 3) * 4;
  }
  typedef const __attribute__((address_space(1))) void* global_ptr;
  typedef __attribute__((address_space(3))) void* lds_ptr;
  auto load = [&](int k, int buf) {
    unsigned char* d = sm + buf * S::STAGE;
#pragma unroll
    for (int j = 0; j < CHUNKS; ++j)
      __builtin_amdgcn_global_load_lds((global_ptr)(src[j] + (long)k * kQ8Tile),
                                       (lds_ptr)(d + (wave * CHUNKS + j) * 1024), 16, 0, 0);
    __builtin_amdgcn_global_load_lds((global_ptr)(ssrc + (long)k * 16),
                                     (lds_ptr)(d + S::SCALES + wave * 256), 4, 0, 0);
  };
  const int r = lane & 15, h = lane >> 5, half = (lane >> 4) & 1;
  int at[SPW];
#pragma unroll
  for (int s = 0; s < SPW; ++s)
    at[s] = half * kQ8Tile + q8_chunk(r, 2 * (wk * SPW + s) + h);
  floatx16 acc[CB][RB];
#pragma unroll
  for (int n = 0; n < CB; ++n)
#pragma unroll
    for (int m = 0; m < RB; ++m)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[n][m][e] = 0.0f;

  intx4 raw[2][RB + CB];
  bf16x8_t frag[2][RB + CB];
  float scale[RB + CB];
  auto read = [&](intx4 (&f)[RB + CB], int buf, int s) {
    const unsigned char* b = sm + buf * S::STAGE + at[s];
#pragma unroll
    for (int i = 0; i < RB; ++i)
      f[i] = *reinterpret_cast<const intx4*>(b + (wm * RB + i) * 2 * kQ8Tile);
#pragma unroll
    for (int i = 0; i < CB; ++i)
      f[RB + i] = *reinterpret_cast<const intx4*>(b + (XT + (wn * CB + i) * 2) * kQ8Tile);
  };
  auto read_scales = [&](unsigned (&u)[RB + CB], int buf) {
    const unsigned char* b = sm + buf * S::STAGE + S::SCALES + half * 16 + r;
#pragma unroll
    for (int i = 0; i < RB; ++i) u[i] = b[(wm * RB + i) * 32];
#pragma unroll
    for (int i = 0; i < CB; ++i) u[RB + i] = b[(XT + (wn * CB + i) * 2) * 16];
  };
  auto convert = [&](bf16x8_t (&f)[RB + CB], const intx4 (&u)[RB + CB], int t) {
#pragma unroll
    for (int i = 0; i < RB + CB; ++i) f[i] = q8_frag(u[i][2 * t], u[i][2 * t + 1], scale[i]);
  };
  load(0, 0);
  if (kb > 1) {
    load(1, 1);
    wait_vm<CHUNKS + 1>();  // the second stage's may be on their way
  } else {
    wait_vm<0>();
  }
  __syncthreads();
  unsigned us[RB + CB];
  read_scales(us, 0);
  read(raw[0], 0, 0);
#pragma unroll
  for (int i = 0; i < RB + CB; ++i) scale[i] = __uint_as_float(us[i] << 23);
  convert(frag[0], raw[0], 0);
#pragma unroll 1
  for (int k = 0; k < kb; ++k) {
    const int buf = k & 1;
#pragma unroll
    for (int u = 0; u < 2 * SPW; ++u) {
      const int s = u >> 1, t = u & 1;
      if (u == 2 * SPW - 2) {
        // the conversions so far stay in front of the branches, beside their step's products
#pragma unroll
        for (int i = 0; i < RB + CB; ++i) asm volatile("" : "+v"(frag[0][i]));
        // this wave's part of the next stage is in LDS, and its reads of this one are done
        if (k + 1 < kb) wait_vm<0>();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (k + 2 < kb) load(k + 2, buf);
        read_scales(us, buf ^ 1);
        read(raw[0], buf ^ 1, 0);  // past the last stage: bytes of a buffer, not used
      } else if (t == 0) {
        read(raw[(s + 1) & 1], buf, s + 1);
      }
      if (u == 2 * SPW - 1)
#pragma unroll
        for (int i = 0; i < RB + CB; ++i) scale[i] = __uint_as_float(us[i] << 23);
      convert(frag[(u + 1) & 1], raw[(s + t) & 1], t ^ 1);
#pragma unroll
      for (int n = 0; n < CB; ++n)
#pragma unroll
        for (int m = 0; m < RB; ++m)
          acc[n][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[u & 1][RB + n], frag[u & 1][m],
                                                              acc[n][m], 0, 0, 0);
      constexpr int CV = (4 * (RB + CB) + RB * CB - 1) / (RB * CB);
      if (t == 0) __builtin_amdgcn_sched_group_barrier(0x100, RB + CB, 0);
      if (u == 2 * SPW - 2) __builtin_amdgcn_sched_group_barrier(0x100, RB + CB, 0);
#pragma unroll
      for (int i = 0; i < RB * CB; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, CV, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  // outputs through LDS, 32 rows a wave at a time: the WK waves' sums meet there, and stores are
  // whole lines of y
  float* out = reinterpret_cast<float*>(sm + (wave - wk) * S::OUT);
#pragma unroll
  for (int m = 0; m < RB; ++m) {
    constexpr int QUADS = 32 * 8 * CB / WK;  // of this wave
    floatx4 res[QUADS / 64];
    if (a.epi == LX_EPI_RESID)
#pragma unroll
      for (int i = 0; i < QUADS / 64; ++i) {
        const int e = wk * QUADS + lane + 64 * i;
        res[i] = resid_quad(a, mt * XT * 16 + (wm * RB + m) * 32 + e / (8 * CB),
                            (long)nt * WT * 16 + wn * CB * 32 + e % (8 * CB) * 4);
      }
    if (m == 0 || WK > 1) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int n = 0; n < CB; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<floatx4*>(out + wk * S::OUT / 4 + (lane & 31) * S::ROW + 32 * n + 8 * q +
                                    4 * h) =
            floatx4{acc[n][m][4 * q], acc[n][m][4 * q + 1], acc[n][m][4 * q + 2],
                    acc[n][m][4 * q + 3]};
    if (WK > 1) {
      __syncthreads();
    } else {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }
#pragma unroll
    for (int i = 0; i < QUADS / 64; ++i) {
      const int e = wk * QUADS + lane + 64 * i, row = e / (8 * CB), col = e % (8 * CB) * 4;
      const float* p = out + row * S::ROW + col;
      floatx4 v = *reinterpret_cast<const floatx4*>(p);
#pragma unroll
      for (int w = 1; w < WK; ++w) v += *reinterpret_cast<const floatx4*>(p + w * S::OUT / 4);
      epi_quad(a, mt * XT * 16 + (wm * RB + m) * 32 + row, (long)nt * WT * 16 + wn * CB * 32 + col,
               v, res[i]);
    }
  }
}

template <int RB, int CB, int WM, int WN, int WK, int OCC>
int launch_tile(Q8Lin& a, hipStream_t s) {
  using S = TileShape<RB, CB, WM, WN, WK>;
  const auto kern = q8_tile_kernel<RB, CB, WM, WN, WK, OCC>;
  long grid;
  LX_TRY(tile_grid(a, 32 * RB * WM, 32 * CB * WN, 64 * S::WAVES, &grid));
  static LdsLimit once;
  LX_TRY(raise_lds_limit(reinterpret_cast<const void*>(kern), S::LDS, once, "q8_tile_kernel"));
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * S::WAVES), S::LDS, s, a);
  return check_launch("q8_tile_kernel");
}

// Fewer tiles than CUs.  A workgroup owns (32 RB) x (32 CB) outputs and each of its W waves takes
// every W-th block of K (H = 2) or half of one (H = 1), through a ring of R slots of LDS of its own:
// no barrier until the waves' sums meet, and R - 1 slots of every wave on their way.  A half
// block's tile is 1 KB, one instruction.  1531 x 896 x 4864 on 96 x 64: 17.5 us (0.76 PFLOP/s; with
// residual as much) where 64 x 64 on the tile kernel takes 22.9; a launch, the first slots and the sums
// alone take 8.2, with the loads 15, with conversions and products but no loads 14.3; three slots
// deep it is the same.  256 x 896 x 4864 on 32 x 32: 7.0, 256 x 896 x 896 3.6 (3.8 on half blocks).
template <int RB, int CB, int W, int H, int R>
struct RingShape {
  static constexpr int T = 2 * (RB + CB);  // 16-row tiles of a slot: rows of x, then of W
  static_assert(T <= 16, "one instruction loads a slot's scales");
  static constexpr int CODES = T * H * 1024;
  static constexpr int SLOT = CODES + 256;  // the scales behind the codes
  static constexpr int ROW = 32 * CB + 4;  // floats of a row of outputs in LDS
  static constexpr int OUT = 32 * RB * ROW * 4;  // a wave's sums
  static constexpr int LDS = W * (R * SLOT > OUT ? R * SLOT : OUT);
  static_assert(LDS <= 160 * 1024, "LDS of a CU");
  static constexpr int QUADS = 32 * RB * 8 * CB;  // of four outputs
  static constexpr int LOADS = T * H + 1;  // instructions that load a slot
  static_assert(H == 1 || H == 2, "half a block or a block");
  static_assert((R - 2) * LOADS < 64, "vmcnt");
};

template <int RB, int CB, int W, int H, int R, int OCC>
__global__ __launch_bounds__(64 * W, OCC) void q8_ring_kernel(Q8Lin a) {
  using S = RingShape<RB, CB, W, H, R>;
  constexpr int T = S::T;
  extern __shared__ __attribute__((aligned(16))) unsigned char sm[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int mt, nt;
  tile_at(a, mt, nt);
  const int mtiles = (a.x.rows + 15) / 16, ntiles = (a.w.rows + 15) / 16;
  const int kb = a.x.kb, slots = (2 * kb / H - wave + W - 1) / W;  // this wave's
  auto tile_of = [&](int t) {
    return t < 2 * RB ? min(mt * 2 * RB + t, mtiles - 1)
                      : min(nt * 2 * CB + min(t - 2 * RB, 2 * CB - 1), ntiles - 1);
  };
  const unsigned char* base[T];
#pragma unroll
  for (int t = 0; t < T; ++t)
    base[t] = (t < 2 * RB ? a.x.codes : a.w.codes) + (long)tile_of(t) * kb * kQ8Tile;
  const unsigned char* sbase;
  {
    const int t = lane >> 2;
    sbase = (t < 2 * RB ? a.x.scales : a.w.scales) + (long)tile_of(t) * kb * 16 + (lane & 3) * 4;
  }
  typedef const __attribute__((address_space(1))) void* global_ptr;
  typedef __attribute__((address_space(3))) void* lds_ptr;
  unsigned char* ring = sm + wave * R * S::SLOT;
  auto load = [&](int i, int slot) {
    const int j = i * W + wave, block = H == 2 ? j : j >> 1;
    const long off = (long)j * (H * 1024) + lane * 16;
    unsigned char* d = ring + slot * S::SLOT;
#pragma unroll
    for (int t = 0; t < T; ++t) {
      __builtin_amdgcn_global_load_lds((global_ptr)(base[t] + off),
                                       (lds_ptr)(d + t * H * 1024), 16, 0, 0);
      if constexpr (H == 2)  // the offset counts on both sides
        __builtin_amdgcn_global_load_lds((global_ptr)(base[t] + off),
                                         (lds_ptr)(d + t * H * 1024), 16, 1024, 0);
    }
    __builtin_amdgcn_global_load_lds((global_ptr)(sbase + (long)block * 16),
                                     (lds_ptr)(d + S::CODES), 4, 0, 0);
  };
  const int r = lane & 15, h = lane >> 5, half = (lane >> 4) & 1;
  int at[2 * H];
#pragma unroll
  for (int s = 0; s < 2 * H; ++s)
    at[s] = half * H * 1024 + q8_chunk(r, 2 * s + h);
  floatx16 acc[CB][RB];
#pragma unroll
  for (int n = 0; n < CB; ++n)
#pragma unroll
    for (int m = 0; m < RB; ++m)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[n][m][e] = 0.0f;
  intx4 raw[2][RB + CB];
  bf16x8_t frag[2][RB + CB];
  float scale[RB + CB];
  unsigned us[RB + CB];
  auto read = [&](intx4 (&f)[RB + CB], int slot, int s) {
    const unsigned char* b = ring + slot * S::SLOT + at[s];
#pragma unroll
    for (int i = 0; i < RB + CB; ++i) f[i] = *reinterpret_cast<const intx4*>(b + i * H * 2048);
  };
  auto read_scales = [&](int slot) {
    const unsigned char* b = ring + slot * S::SLOT + S::CODES + half * 16 + r;
#pragma unroll
    for (int i = 0; i < RB + CB; ++i) us[i] = b[i * 32];
  };
  auto set_scales = [&]() {
#pragma unroll
    for (int i = 0; i < RB + CB; ++i) scale[i] = __uint_as_float(us[i] << 23);
  };
  auto convert = [&](bf16x8_t (&f)[RB + CB], const intx4 (&u)[RB + CB], int t) {
#pragma unroll
    for (int i = 0; i < RB + CB; ++i) f[i] = q8_frag(u[i][2 * t], u[i][2 * t + 1], scale[i]);
  };
  // slot i is in LDS (R - 2 later ones may be on their way), and this wave's reads are done
  auto wait = [&](int i) {
    if (i + R - 2 < slots)
      wait_vm<(R - 2) * S::LOADS>();
    else
      wait_vm<0>();
  };
  // the residual, whose latency would stand alone behind the sums (one load a thread is not worth
  // its instructions here: 256 x 896 x 896 3.7 -> 3.8)
  constexpr int EACH = (S::QUADS + 64 * W - 1) / (64 * W);
  floatx4 res[EACH];
  auto at_quad = [&](int i, int& row, int& col) {
    const int e = tid + 64 * W * i;
    row = e / (8 * CB);
    col = e % (8 * CB) * 4;
    return e < S::QUADS;
  };
  if (EACH > 1 && a.epi == LX_EPI_RESID)
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
      int row, col;
      if (at_quad(i, row, col))
        res[i] = resid_quad(a, mt * RB * 32 + row, (long)nt * CB * 32 + col);
    }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (i < slots) load(i, i);
  if (slots > 0) {
    wait(0);
    read_scales(0);
    read(raw[0], 0, 0);
    set_scales();
    convert(frag[0], raw[0], 0);
  }
  int slot = 0;
#pragma unroll 1
  for (int i = 0; i < slots; ++i) {
    const int next = slot + 1 == R ? 0 : slot + 1;
#pragma unroll
    for (int u = 0; u < 4 * H; ++u) {
      const int s = u >> 1, t = u & 1;
      if (u == 4 * H - 2) {
        // the conversions so far stay in front of the branches, beside their step's products
#pragma unroll
        for (int e = 0; e < RB + CB; ++e) asm volatile("" : "+v"(frag[0][e]));
        if (i + 1 < slots) wait(i + 1);
        if (i + R < slots) load(i + R, slot);
        read_scales(next);
        read(raw[0], next, 0);  // past the last slot: bytes of the ring, not used
      } else if (t == 0) {
        read(raw[(s + 1) & 1], slot, s + 1);
      }
      if (u == 4 * H - 1) set_scales();
      convert(frag[(u + 1) & 1], raw[(s + t) & 1], t ^ 1);
#pragma unroll
      for (int n = 0; n < CB; ++n)
#pragma unroll
        for (int m = 0; m < RB; ++m)
          acc[n][m] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(frag[u & 1][RB + n], frag[u & 1][m],
                                                              acc[n][m], 0, 0, 0);
      constexpr int CV = (4 * (RB + CB) + RB * CB - 1) / (RB * CB);
      if (t == 0) __builtin_amdgcn_sched_group_barrier(0x100, RB + CB, 0);
      if (u == 4 * H - 2) __builtin_amdgcn_sched_group_barrier(0x100, RB + CB, 0);
#pragma unroll
      for (int e = 0; e < RB * CB; ++e) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        __builtin_amdgcn_sched_group_barrier(0x2, CV, 0);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    slot = next;
  }
  // the waves' sums meet in LDS, in the order of the waves
  float* out = reinterpret_cast<float*>(sm);
  __syncthreads();
#pragma unroll
  for (int m = 0; m < RB; ++m)
#pragma unroll
    for (int n = 0; n < CB; ++n)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<floatx4*>(out + wave * S::OUT / 4 + (32 * m + (lane & 31)) * S::ROW +
                                    32 * n + 8 * q + 4 * h) =
            floatx4{acc[n][m][4 * q], acc[n][m][4 * q + 1], acc[n][m][4 * q + 2],
                    acc[n][m][4 * q + 3]};
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    int row, col;
    if (!at_quad(i, row, col)) break;
    const float* p = out + row * S::ROW + col;
    floatx4 v = *reinterpret_cast<const floatx4*>(p);
#pragma unroll
    for (int w = 1; w < W; ++w) v += *reinterpret_cast<const floatx4*>(p + w * S::OUT / 4);
    const int om = mt * RB * 32 + row;
    const long on = (long)nt * CB * 32 + col;
    if (EACH == 1 && a.epi == LX_EPI_RESID) res[i] = resid_quad(a, om, on);
    epi_quad(a, om, on, v, res[i]);
  }
}

template <int RB, int CB, int W, int H, int R, int OCC>
int launch_ring(Q8Lin& a, hipStream_t s) {
  using S = RingShape<RB, CB, W, H, R>;
  const auto kern = q8_ring_kernel<RB, CB, W, H, R, OCC>;
  long grid;
  LX_TRY(tile_grid(a, 32 * RB, 32 * CB, 64 * W, &grid));
  static LdsLimit once;
  LX_TRY(raise_lds_limit(reinterpret_cast<const void*>(kern), S::LDS, once, "q8_ring_kernel"));
  hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(64 * W), S::LDS, s, a);
  return check_launch("q8_ring_kernel");
}

template <int MT, int NT, int WAVES>
int launch_stream(Q8Lin& a, hipStream_t s) {
  constexpr size_t lds = (size_t)MT * NT * WAVES * 1024;
  static_assert(lds <= 65536, "raise the limit");
  long grid;
  LX_TRY(tile_grid(a, 16 * MT, 16 * NT, 64 * WAVES, &grid));
  hipLaunchKernelGGL((q8_stream_kernel<MT, NT, WAVES>), dim3((unsigned)grid), dim3(64 * WAVES), lds,
                     s, a);
  return check_launch("q8_stream_kernel");
}

}  // namespace
}  // namespace lx

using namespace lx;

extern "C" int lx_linear_q8_f32(const lx_q8* x, const lx_q8* w, const float* bias,
                                const lx_epilogue* epi, const float* resid, long ldr, float* y,
                                long ldy, hipStream_t stream) {
  LX_REQUIRE(q8_ok(x) && q8_ok(w) && y, "linear_q8: null pointer, bad shape or unaligned matrix");
  LX_REQUIRE(x->K == w->K, "linear_q8: x has %d columns, w %d", x->K, w->K);
  const int kind = epi ? epi->kind : LX_EPI_NONE;
  LX_REQUIRE(kind == LX_EPI_NONE || kind == LX_EPI_GELU_TANH || kind == LX_EPI_RESID ||
                 kind == LX_EPI_SWIGLU_PAIRED,
             "linear_q8: epilogue %d (none, GELU, residual or SwiGLU)", kind);
  LX_REQUIRE(kind != LX_EPI_SWIGLU_PAIRED || w->rows % 2 == 0,
             "linear_q8: SwiGLU needs an even number of rows of w");
  LX_REQUIRE(!resid || kind == LX_EPI_RESID, "linear_q8: resid without a residual epilogue");
  const int M = x->rows, N = w->rows, cols = kind == LX_EPI_SWIGLU_PAIRED ? N / 2 : N;
  if (!resid) {
    resid = y;
    ldr = ldy;
  }
  LX_REQUIRE(ldy >= cols && ldr >= cols, "linear_q8: bad row stride ldy=%ld ldr=%ld", ldy, ldr);
  LX_REQUIRE(((uintptr_t)y | (uintptr_t)bias | (uintptr_t)resid) % 4 == 0, "linear_q8: unaligned");
  LX_REQUIRE((resid == y && ldr == ldy) || !rows_overlap(resid, ldr, cols, y, ldy, cols, M),
             "linear_q8: y overlaps resid");
  LX_REQUIRE(!q8_overlaps(x, y, ldy, cols, M) && !q8_overlaps(w, y, ldy, cols, M) &&
                 (!bias || !rows_overlap(y, ldy, cols, bias, 0, N, M)),
             "linear_q8: y overlaps x, w or bias");
  Q8Lin a{};
  a.x = q8_mat(x);
  a.w = q8_mat(w);
  a.bias = bias;
  a.resid = resid;
  a.y = y;
  a.ldr = ldr;
  a.ldy = ldy;
  a.epi = kind;
  if (M <= 16) {
    // 16 columns of y a workgroup, 32 where there are thousands of them (8192 x 8192 14.8 -> 12.7
    // us; 9728 x 896 3.8 and 3.9)
    if ((long)N * a.w.kb >= 1 << 18) return launch_stream<1, 2, 8>(a, stream);
    return launch_stream<1, 1, 8>(a, stream);
  }
  const long cus = device_cus();
  auto tiles = [&](long m, long n) { return ((M + m - 1) / m) * ((N + n - 1) / n); };
  // Large tiles while they fill the rounds that they take: a tile of 256 x 256 costs a CU as much as
  // 3.5 of 128 x 128, the first of those as much as 3.3 of 64 x 64 (four of which share a CU, so that
  // their rounds need not be full) and another one 2.5 (256 x 256, 128 x 128, 64 x 64, 32 x 64; us)
  //   4096 x 8192 x 4096   227   260   321         1000 x 6761 x 896  30.7  19.0  22.3  23.7
  //   1531 x 9728 x  896  33.4  35.5  41.9         4096 x 1152 x 896  27.6  17.8  15.8  16.9
  //   1600 x 9728 x  896  57.1  36.9  44.8         1024 x 4096 x 896  27.6  12.7  13.6  15.5
  //   2304 x 8192 x 4096   190   155   173         1531 x 2000 x 896  27.3  12.4  11.4  12.5
  auto rounds = [&](long m, long n) { return (tiles(m, n) + cus - 1) / cus; };
  if (7 * rounds(256, 256) <= 2 * rounds(128, 128))
    return launch_tile<4, 2, 2, 4, 1, 1>(a, stream);
  if (10 * tiles(64, 64) >= (25 * rounds(128, 128) + 8) * cus)
    return launch_tile<2, 1, 2, 4, 1, 2>(a, stream);
  // while the smallest give each CU one at most, and at 12 blocks of K or more (24 for the largest)
  // while larger ones do, every wave on K of its own (32 x 32, 32 x 64, 64 x 64, 96 x 64, 128 x 64
  // on the ring kernel, then 64 x 64 and 32 x 64 on the tile kernel)
  //    256 x  896 x  896   3.6   4.4   5.8   7.1   8.8   5.7   4.6
  //    256 x  896 x 4864   7.0   8.8  13.5  16.0  20.1  19.9  18.2
  //    256 x 1152 x  896   5.6   4.3   5.8   7.2   8.8   5.8   4.7
  //    128 x 4096 x 4864  12.6   9.3  13.7  16.6  20.3  19.9  18.2
  //    500 x 1500 x  896   8.2   7.7   6.2   7.8   9.2   6.2   6.1
  //    500 x 1500 x 1500  10.4   9.4   7.7   9.4  11.3   9.1   8.5
  //   1024 x 1024 x 4864  22.9  16.6  15.2  16.5  20.3  20.5  19.2
  //   1531 x  896 x 1500  18.0  13.4  11.0   9.8  11.6  10.7   9.8
  //   1531 x  896 x 4864  30.6  23.7  22.7  17.5  21.2  22.9  21.4
  //   2000 x 1000 x 1600  25.8  17.9  12.6  18.1  13.3  11.9  13.1
  //   2000 x 1000 x 4864  41.4  31.3  24.8  31.3  23.3  25.8  30.1
  //    256 x 9728 x  896  25.3  18.6  12.7  14.8  18.1  10.6  11.0
  //    177 x 6761 x  896  13.4  11.6   9.0   8.8  10.4   8.5   7.7
  if (tiles(32, 32) <= cus) return launch_ring<1, 1, 8, 2, 2, 1>(a, stream);
  if (tiles(32, 64) <= cus) return launch_ring<1, 2, 8, 1, 2, 2>(a, stream);
  if (a.x.kb >= 12) {
    if (tiles(64, 64) <= cus) return launch_ring<2, 2, 4, 1, 2, 2>(a, stream);
    if (tiles(96, 64) <= cus) return launch_ring<3, 2, 4, 1, 2, 1>(a, stream);
    if (tiles(128, 64) <= cus && a.x.kb >= 24) return launch_ring<4, 2, 4, 1, 3, 1>(a, stream);
  }
  // and where tiles of 64 rows hold few of them (24 x 30000 x 896 8.4 and 7.6, 80 x 20000 x 896 11.6
  // and 10.2)
  if ((a.x.kb < 12 && 2 * tiles(64, 64) < 3 * cus) || 10 * tiles(32, 64) < 17 * tiles(64, 64))
    return launch_tile<1, 1, 1, 2, 2, 5>(a, stream);
  return launch_tile<2, 1, 1, 2, 2, 4>(a, stream);
}
