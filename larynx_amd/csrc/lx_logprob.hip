// Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits, in
// one pass over the logits.
//
// A workgroup holds up to 8192 logits of a row in registers: their maximum m, s = the sum of e^(x -
// m) over all but one of the maxima, t = the sum of e^(x - m) (x - m), then
//   log sum e^x = m + log1p(s),   entropy = log1p(s) - t / (1 + s)
// (the 1 of the maximum left out of the sum, so that a row with one likely token keeps the digits
// of the rest).  Longer rows are cut into pieces of equal length, whose (m, s, t) and leading keys
// a second launch joins.
//
// Alternatives are ordered by 64-bit keys, unlike for any two logits: the value's bits in an order
// that whole numbers share, then the complement of the index.  In each wave the k-th largest of the
// lanes' own largest keys bounds the k-th largest key from below; the largest of these bounds
// leaves a few more than k candidates, and a candidate's rank among them is its place.
#include <algorithm>
#include <climits>

#include "lx_common.hpp"
#include "lx_internal.hpp"

namespace lx {
namespace {

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned long long key_t64;

constexpr int kPiece = 8192;   // logits of a workgroup
constexpr int kMaxTop = 64;    // a lane each
constexpr int kCand = 1024;    // candidates ranked at once

struct LpArgs {
  const float* x;
  long ld;
  int V, pieces, len, top;  // len: logits of a piece, a multiple of 4
  const int* tokens;
  float *logp, *entropy, *top_logp;
  int* top_ids;
  float4* part;    // (rows, pieces): m, s, t
  key_t64* keys;   // (rows, pieces, top), largest first
};

// The order of fp32 numbers as whole numbers: NaN above everything, both zeros alike.
__device__ __forceinline__ unsigned order_of(float x) {
  const unsigned u = __float_as_uint(x + 0.0f);
  return x != x ? 0xffffffffu : u ^ ((unsigned)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float value_of(unsigned o) {
  if (o == 0xffffffffu) return __builtin_nanf("");
  return __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
}
__device__ __forceinline__ key_t64 key_of(unsigned order, int index) {
  return (key_t64)order << 32 | (unsigned)~index;
}

__device__ __forceinline__ float exp_of(float d) {
  return __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
}

// The k-th largest of the 64 lanes' keys.
__device__ __forceinline__ key_t64 wave_kth(key_t64 key, int k) {
  key_t64 at = 0;
#pragma unroll 1
  for (int b = 63; b >= 0; --b) {
    const key_t64 mid = at | 1ull << b;
    if (__popcll(__ballot(key >= mid)) >= k) at = mid;
  }
  return at;
}

struct LpShared {
  float f[4][4];
  key_t64 bound[4];
  int count;
  key_t64 cand[kCand];
};

// The `top` largest of the keys that `each` calls its argument with (each thread's own), largest
// first, handed to out(place, key).  `mine`: the largest of this thread's keys (0: none).
template <class Each, class Out>
__device__ void block_top(LpShared& sh, int top, key_t64 mine, Each each, Out out) {
  const int tid = threadIdx.x;
  const key_t64 b = wave_kth(mine, top);
  if ((tid & 63) == 0) sh.bound[tid >> 6] = b;
  if (tid == 0) sh.count = 0;
  __syncthreads();
  key_t64 bound = max(max(sh.bound[0], sh.bound[1]), max(sh.bound[2], sh.bound[3]));
  for (;;) {
    each([&](key_t64 key) {
      if (key >= bound && key) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kCand) sh.cand[at] = key;
      }
    });
    __syncthreads();
    if (sh.count <= kCand) break;
    // many large keys in few lanes: the exact bound, bit by bit
    key_t64 at = 0;
#pragma unroll 1
    for (int bit = 63; bit >= 0; --bit) {
      const key_t64 mid = at | 1ull << bit;
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
      int n = 0;
      each([&](key_t64 key) { n += key >= mid; });
      if (n) atomicAdd(&sh.count, n);
      __syncthreads();
      if (sh.count >= top) at = mid;
    }
    bound = at;
    __syncthreads();
    if (tid == 0) sh.count = 0;
    __syncthreads();
  }
  const int n = sh.count;
  for (int i = tid; i < n; i += 256) {
    const key_t64 key = sh.cand[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += sh.cand[j] > key;
    if (rank < top) out(rank, key);
  }
}

struct RowSums {
  float m, s, t;
};
// What a row gives: log1p(s), 0 where no logit is above -inf.
__device__ __forceinline__ bool row_empty(const RowSums& r) {
  return r.m == -__builtin_huge_valf() && r.s == 0.0f;
}
__device__ __forceinline__ float logp_of(const RowSums& r, float ls, float x) {
  if (row_empty(r)) return -__builtin_huge_valf();
  return (float)(((double)x - (double)r.m) - (double)ls);
}
__device__ __forceinline__ void write_row(const LpArgs& a, int row, const RowSums& r, float ls) {
  if (a.logp) {
    const int t = a.tokens[row];
    float v = 0.0f;
    if (t >= a.V || t < -1) v = __builtin_nanf("");
    else if (t >= 0) v = logp_of(r, ls, a.x[row * a.ld + t]);
    a.logp[row] = v;
  }
  if (a.entropy) a.entropy[row] = row_empty(r) ? 0.0f : ls - r.t / (1.0f + r.s);
}

template <int NV, bool TOP>
__global__ __launch_bounds__(256) void logprob_kernel(LpArgs a) {
  __shared__ LpShared sh;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int row = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  const int begin = piece * a.len, n = min(a.len, a.V - begin);
  const float* x = a.x + row * a.ld + begin;
  const float inf = __builtin_huge_valf();
  float v[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (tid + 256 * i) * 4;
    if (k + 4 <= n) {
      const float4u u = *reinterpret_cast<const float4u*>(x + k);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = u[e];
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) v[i][e] = k + e < n ? x[k + e] : -inf;
    }
  }
  float m = -inf;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) m = fmaxf(m, v[i][e]);
  m = wave_max(m);
  if ((tid & 63) == 0) sh.f[wave][0] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sh.f[0][0], sh.f[1][0]), fmaxf(sh.f[2][0], sh.f[3][0]));
  const float ref = m == -inf ? 0.0f : m;
  float s = 0.0f, t = 0.0f, tops = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = v[i][e] - ref;
      const float p = exp_of(d);
      if (d == 0.0f) tops += 1.0f; else s += p;
      t = fmaf(p, fmaxf(d, -200.0f), t);  // far below, p is 0
    }
  s = wave_sum(s);
  t = wave_sum(t);
  tops = wave_sum(tops);
  if ((tid & 63) == 0) {
    sh.f[wave][1] = s;
    sh.f[wave][2] = t;
    sh.f[wave][3] = tops;
  }
  __syncthreads();
  RowSums r;
  r.m = m;
  r.t = (sh.f[0][2] + sh.f[1][2]) + (sh.f[2][2] + sh.f[3][2]);
  tops = (sh.f[0][3] + sh.f[1][3]) + (sh.f[2][3] + sh.f[3][3]);
  r.s = (sh.f[0][1] + sh.f[1][1]) + (sh.f[2][1] + sh.f[3][1]);
  if (tops > 0.0f) r.s += tops - 1.0f;
  const float ls = log1pf(r.s);
  if (a.pieces > 1) {
    if (tid == 0) a.part[blockIdx.x] = make_float4(r.m, r.s, r.t, 0.0f);
  } else if (tid == 0) {
    write_row(a, row, r, ls);
  }
  if constexpr (TOP) {
    key_t64 mine = 0;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        mine = max(mine, key_of(order_of(v[i][e]), begin + (tid + 256 * i) * 4 + e));
    block_top(sh, a.top, mine,
              [&](auto f) {
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                  for (int e = 0; e < 4; ++e)
                    f(key_of(order_of(v[i][e]), begin + (tid + 256 * i) * 4 + e));
              },
              [&](int at, key_t64 key) {
                if (a.pieces > 1) {
                  a.keys[(long)blockIdx.x * a.top + at] = key;
                } else {
                  a.top_ids[(long)row * a.top + at] = (int)~(unsigned)key;
                  a.top_logp[(long)row * a.top + at] =
                      logp_of(r, ls, value_of((unsigned)(key >> 32)));
                }
              });
  }
}

__global__ __launch_bounds__(256) void logprob_join_kernel(LpArgs a) {
  __shared__ LpShared sh;
  const int tid = threadIdx.x, wave = tid >> 6, row = blockIdx.x;
  const float4* part = a.part + (long)row * a.pieces;
  const float inf = __builtin_huge_valf();
  float m = -inf;
  for (int i = tid; i < a.pieces; i += 256) m = fmaxf(m, part[i].x);
  m = wave_max(m);
  if ((tid & 63) == 0) sh.f[wave][0] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sh.f[0][0], sh.f[1][0]), fmaxf(sh.f[2][0], sh.f[3][0]));
  float s = 0.0f, t = 0.0f, tops = 0.0f;
  for (int i = tid; i < a.pieces; i += 256) {
    const float4 p = part[i];
    if (p.x == m) {
      s += p.y;
      t += p.z;
      tops += 1.0f;
    } else if (p.x == -inf) {
      s += p.y;  // 0, or the NaN of such a piece
    } else {
      const float d = p.x - m, w = exp_of(d);
      s = fmaf(w, 1.0f + p.y, s);
      t = fmaf(w, fmaf(1.0f + p.y, fmaxf(d, -200.0f), p.z), t);
    }
  }
  s = wave_sum(s);
  t = wave_sum(t);
  tops = wave_sum(tops);
  if ((tid & 63) == 0) {
    sh.f[wave][1] = s;
    sh.f[wave][2] = t;
    sh.f[wave][3] = tops;
  }
  __syncthreads();
  RowSums r;
  r.m = m;
  r.t = (sh.f[0][2] + sh.f[1][2]) + (sh.f[2][2] + sh.f[3][2]);
  tops = (sh.f[0][3] + sh.f[1][3]) + (sh.f[2][3] + sh.f[3][3]);
  r.s = (sh.f[0][1] + sh.f[1][1]) + (sh.f[2][1] + sh.f[3][1]);
  if (m != -inf) r.s += tops - 1.0f;
  const float ls = log1pf(r.s);
  if (tid == 0) write_row(a, row, r, ls);
  if (a.top) {
    const key_t64* keys = a.keys + (long)row * a.pieces * a.top;
    const int n = a.pieces * a.top;
    key_t64 mine = 0;
    for (int i = tid; i < n; i += 256) mine = max(mine, keys[i]);
    block_top(sh, a.top, mine,
              [&](auto f) {
                for (int i = tid; i < n; i += 256) f(keys[i]);
              },
              [&](int at, key_t64 key) {
                a.top_ids[(long)row * a.top + at] = (int)~(unsigned)key;
                a.top_logp[(long)row * a.top + at] =
                    logp_of(r, ls, value_of((unsigned)(key >> 32)));
              });
  }
}

int lp_pieces(int V) { return (V + kPiece - 1) / kPiece; }
bool lp_shape_ok(int rows, int V, int top) {
  return rows > 0 && V > 0 && V <= 1 << 24 && top >= 0 && top <= std::min(V, kMaxTop) &&
         (long)rows * lp_pieces(V) <= INT_MAX / 256;
}

template <bool TOP>
void launch_logprob(const LpArgs& a, int rows, hipStream_t s) {
  const dim3 grid((unsigned)((long)rows * a.pieces)), block(256);
  if (a.len <= 2048)
    hipLaunchKernelGGL((logprob_kernel<2, TOP>), grid, block, 0, s, a);
  else if (a.len <= 4096)
    hipLaunchKernelGGL((logprob_kernel<4, TOP>), grid, block, 0, s, a);
  else
    hipLaunchKernelGGL((logprob_kernel<8, TOP>), grid, block, 0, s, a);
}

}  // namespace
}  // namespace lx

using namespace lx;

extern "C" size_t lx_token_logprobs_ws_floats(int rows, int V, int top) {
  if (!lp_shape_ok(rows, V, top)) return 0;
  const int pieces = lp_pieces(V);
  return pieces == 1 ? 0 : (size_t)rows * pieces * (4 + 2 * top);
}

extern "C" int lx_token_logprobs_f32(const float* logits, long ld, int rows, int V,
                                     const int* tokens, float* logp, float* entropy, int top,
                                     float* top_logp, int* top_ids, float* ws, size_t ws_floats,
                                     hipStream_t stream) {
  LX_REQUIRE(logits, "token_logprobs: null pointer");
  LX_REQUIRE(lp_shape_ok(rows, V, top), "token_logprobs: bad shape rows=%d V=%d top=%d", rows, V,
             top);
  LX_REQUIRE(ld >= V, "token_logprobs: bad row stride %ld", ld);
  LX_REQUIRE(!tokens == !logp, "token_logprobs: tokens and logp go together");
  LX_REQUIRE(logp || entropy || top, "token_logprobs: nothing asked for");
  LX_REQUIRE(!top || (top_logp && top_ids), "token_logprobs: no room for the alternatives");
  LX_REQUIRE(((uintptr_t)logits | (uintptr_t)tokens | (uintptr_t)logp | (uintptr_t)entropy |
              (uintptr_t)top_logp | (uintptr_t)top_ids) % 4 == 0,
             "token_logprobs: unaligned");
  LpArgs a{};
  a.x = logits;
  a.ld = ld;
  a.V = V;
  a.pieces = lp_pieces(V);
  a.len = ((V + a.pieces - 1) / a.pieces + 3) / 4 * 4;
  a.top = top;
  a.tokens = tokens;
  a.logp = logp;
  a.entropy = entropy;
  a.top_logp = top_logp;
  a.top_ids = top_ids;
  if (a.pieces > 1) {
    const size_t need = lx_token_logprobs_ws_floats(rows, V, top);
    LX_REQUIRE(ws && ws_floats >= need && (uintptr_t)ws % 16 == 0,
               "token_logprobs: workspace of %zu floats, %zu needed", ws ? ws_floats : 0, need);
    a.part = reinterpret_cast<float4*>(ws);
    a.keys = reinterpret_cast<key_t64*>(ws + (size_t)rows * a.pieces * 4);
  }
  if (top)
    launch_logprob<true>(a, rows, stream);
  else
    launch_logprob<false>(a, rows, stream);
  LX_TRY(check_launch("logprob_kernel"));
  if (a.pieces == 1) return LX_OK;
  hipLaunchKernelGGL(logprob_join_kernel, dim3((unsigned)rows), dim3(256), 0, stream, a);
  return check_launch("logprob_join_kernel");
}
