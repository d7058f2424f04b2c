// y = epi(x~ W~^T + bias), both operands in 8 bits with a power of two per block of 128 (lx_q8.hpp).
#include <algorithm>
#include <climits>

#include "lx_q8.hpp"

namespace lx {
namespace {

typedef int intx4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));

struct Q8Lin {
  Q8Mat x, w;
  const float* bias;
  const float* resid;
  float* y;
  long ldr, ldy;
  int epi, vec;
  int tiles_m, tiles_n;  // of the launch
};

__device__ __forceinline__ void epi_one(const Q8Lin& a, int m, long n, float v, float up) {
  if (a.bias) v += a.bias[n];
  if (a.epi == LX_EPI_SWIGLU_PAIRED) {
    if (a.bias) up += a.bias[n + 1];
    a.y[m * a.ldy + (n >> 1)] = (v / (1.0f + expf(-v))) * up;
    return;
  }
  if (a.epi == LX_EPI_GELU_TANH) v = gelu_tanh(v);
  if (a.epi == LX_EPI_RESID) v = a.resid[m * a.ldr + n] + v;
  a.y[m * a.ldy + n] = v;
}

// Columns n .. n + 3 (n a multiple of 4) of row m.
__device__ __forceinline__ void epi_quad(const Q8Lin& a, int m, long n, floatx4 v) {
  if (m >= a.x.rows) return;
  if (a.vec && n + 3 < a.w.rows) {
    if (a.bias) v += *reinterpret_cast<const floatx4*>(a.bias + n);
    if (a.epi == LX_EPI_SWIGLU_PAIRED) {
      *reinterpret_cast<float2*>(a.y + m * a.ldy + (n >> 1)) =
          make_float2((v[0] / (1.0f + expf(-v[0]))) * v[1], (v[2] / (1.0f + expf(-v[2]))) * v[3]);
      return;
    }
    if (a.epi == LX_EPI_GELU_TANH)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = gelu_tanh(v[e]);
    if (a.epi == LX_EPI_RESID) v = *reinterpret_cast<const floatx4*>(a.resid + m * a.ldr + n) + v;
    *reinterpret_cast<floatx4*>(a.y + m * a.ldy + n) = v;
    return;
  }
  const int step = a.epi == LX_EPI_SWIGLU_PAIRED ? 2 : 1;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (e % step == 0 && n + e < a.w.rows) epi_one(a, m, n + e, v[e], v[e | 1]);
}

// Codes as operands of the bf16 matrix instructions: exact, eight bits hold e4m3's four, and the
// power of two comes with the conversion (v_cvt_scalef32_pk_bf16_fp8, two codes an instruction).
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

// A workgroup owns 16 MT rows of x and 16 NT rows of W; its waves take the blocks of K in turn and
// their sums meet in LDS.  W is the instruction's A operand: a lane's four sums are four
// consecutive columns of one row of y.
template <int MT, int NT, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void q8_stream_kernel(Q8Lin a) {
  extern __shared__ __attribute__((aligned(16))) floatx4 red[];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int mt = blockIdx.x % a.tiles_m, nt = blockIdx.x / a.tiles_m;
  const int r = lane & 15, c = lane >> 4;
  const int at = r * kQ8Block + ((c ^ (r >> 1)) << 4);
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
    const int so = (kb >> 2) * 64 + r * 4 + (kb & 3);
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const unsigned char* p = a.w.codes + (wt[i] * a.w.kb + kb) * kQ8Tile;
      wf[i][0] = *reinterpret_cast<const intx4*>(p + at);
      wf[i][1] = *reinterpret_cast<const intx4*>(p + (at ^ 64));
      ws[i] = __uint_as_float((unsigned)a.w.scales[wt[i] * a.w.kb4 * 64 + so] << 23);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) {
      const unsigned char* p = a.x.codes + (xt[i] * a.x.kb + kb) * kQ8Tile;
      xf[i][0] = *reinterpret_cast<const intx4*>(p + at);
      xf[i][1] = *reinterpret_cast<const intx4*>(p + (at ^ 64));
      xs[i] = __uint_as_float((unsigned)a.x.scales[xt[i] * a.x.kb4 * 64 + so] << 23);
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
    epi_quad(a, (mt * MT + m) * 16 + (l & 15), (long)(nt * NT + n) * 16 + 4 * (l >> 4), s);
  }
}

template <int MT, int NT, int WAVES>
int launch_stream(Q8Lin& a, hipStream_t s) {
  constexpr size_t lds = (size_t)MT * NT * WAVES * 1024;
  static LdsLimit once;
  if (lds > 65536)
    LX_TRY(raise_lds_limit(reinterpret_cast<const void*>(q8_stream_kernel<MT, NT, WAVES>), lds,
                           once, "q8_stream_kernel"));
  a.tiles_m = (a.x.rows + 16 * MT - 1) / (16 * MT);
  a.tiles_n = (a.w.rows + 16 * NT - 1) / (16 * NT);
  const long grid = (long)a.tiles_m * a.tiles_n;
  LX_REQUIRE(grid <= INT_MAX / (64 * WAVES), "linear_q8: %d x %d outputs are too many", a.x.rows,
             a.w.rows);
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
  Q8Lin a{};
  a.x = q8_mat(x);
  a.w = q8_mat(w);
  a.bias = bias;
  a.resid = resid;
  a.y = y;
  a.ldr = ldr;
  a.ldy = ldy;
  a.epi = kind;
  a.vec = ldy % 4 == 0 && ldr % 4 == 0 &&
          ((uintptr_t)y | (uintptr_t)bias | (uintptr_t)resid) % 16 == 0;
  if (M <= 16) return launch_stream<1, 1, 8>(a, stream);
  return launch_stream<4, 4, 4>(a, stream);
}
