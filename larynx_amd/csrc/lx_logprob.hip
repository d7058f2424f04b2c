// Log probabilities of given tokens, entropy and the most likely alternatives of rows of logits, in
// one pass over the logits.
//
// A workgroup holds up to 8192 logits of a row in registers: their maximum m, s = the sum of e^(x -
// m) over all but one of the maxima, t = the sum of e^(x - m) (x - m), then
//   log sum e^x = m + log1p(s),   entropy = log1p(s) - t / (1 + s)
// (the 1 of the maximum left out of the sum, so that a row with one likely token keeps the digits
// of the rest; where these are below 2^-70 they are summed again in units of 2^-64, in which a
// logit counts down to e^-131 of the maximum).  Longer rows are cut into pieces of equal length,
// whose (m, s, t) and leading keys a second launch joins.
//
// Alternatives are ordered by 64-bit keys, unlike for any two logits: the value's bits in an order
// that whole numbers share, then the complement of the index.  The k-th largest of the 256 threads'
// maxima (its leading 16 bits, found bit by bit with ballots, each wave for itself) bounds the k-th
// largest logit from below and leaves little more than k candidates (21 of 8192 normal logits for
// k = 20, 74 for 64), whose ranks among each other are their places.  Where ties or an order crowd
// more of them into few threads, the exact bound is found the same way over all logits.
//
// Bound by the logits' bytes where rows are many: 1000 x 151936 98-110 us without alternatives (5.5
// to 6.2 TB/s, above a copy's 4.7), 123 with 20 (4.9 TB/s: 883 vector instructions a wave for 32
// logits a lane, 493 without); 1531 x 6761 11-12 us (3.7 TB/s: one generation of workgroups, a
// round trip and a tail), 15 where each row is summed a second time.  One row of 6761: 3.8 us in a
// graph, 6.4 with alternatives.
#include <algorithm>
#include <climits>

#include "lx_common.hpp"
#include "lx_internal.hpp"

namespace lx {
namespace {

typedef float float4u __attribute__((ext_vector_type(4), aligned(4)));
typedef unsigned long long key_t64;

constexpr int kPiece = 8192;   // logits of a workgroup
constexpr int kMaxTop = 64;
constexpr int kCand = 1024;    // candidates ranked at once
constexpr int kSeg = kCand / 4;  // of a wave
constexpr int kJoin = 192;     // candidates ranked by the joining wave

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
// Sums are handed on in units of 2^-64.  Where too_small does not say so, the terms that the plain
// exponential flushes, below 2^-126 each, are less than 2^-32 of their sum (2^24 of them at most).
constexpr float kUnits = 0x1p64f, kUnit = 0x1p-64f;
__device__ __forceinline__ bool too_small(float m, float s) {  // s in units
  return m > -__builtin_huge_valf() && s < 0x1p-6f;
}
// e^d in units, for d < -48 as all terms of such a sum are: y + 64 is exact then, and the argument's
// product with log2(e) is in two parts, at these distances some 2^-18 of the result.
__device__ __forceinline__ float exp_units(float d) {
#pragma clang fp contract(off)
  const float c = fmaxf(d, -200.0f), y = c * 1.4426950408889634f;
  const float lo = fmaf(c, 1.9259629911266175e-8f, fmaf(c, 1.4426950408889634f, -y));
  const float e = __builtin_amdgcn_exp2f(y + 64.0f);
  return fmaf(e, lo * 0.6931471805599453f, e);
}
__device__ __forceinline__ int lanes(bool c) { return __popcll(__ballot(c)); }
// How many of the lanes below this one have their bit in m.
__device__ __forceinline__ int lanes_below(unsigned long long m) {
  return __builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32),
                                   __builtin_amdgcn_mbcnt_lo((unsigned)m, 0));
}

// The largest number of `high` + 1 bits, its bits below `low` zero, that count() says at least k
// of.
template <class Count>
__device__ __forceinline__ unsigned largest_with(int k, int high, int low, Count count) {
  unsigned at = 0;
#pragma unroll 1
  for (int b = high; b >= low; --b) {
    const unsigned mid = at | 1u << b;
    if (count(mid) >= k) at = mid;
  }
  return at;
}

// Candidates in SEGS segments of n[..] keys, ranked by how many of them are larger, four threads
// each: the `top` largest go to out(place, key).  All threads of the workgroup take part.
template <int THREADS, int SEGS, int STRIDE, class Out>
__device__ __forceinline__ void rank_keys(const key_t64* cand, const int (&n)[SEGS], int top,
                                          Out out) {
  const int part = threadIdx.x & 3;
  int total = 0;
#pragma unroll
  for (int w = 0; w < SEGS; ++w) total += n[w];
  for (int i = threadIdx.x >> 2; i < (total + 15) / 16 * 16; i += THREADS / 4) {
    int at = i, seg = 0;
#pragma unroll
    for (int w = 0; w + 1 < SEGS; ++w)
      if (seg == w && at >= n[w]) {
        at -= n[w];
        seg = w + 1;
      }
    const key_t64 key = i < total ? cand[seg * STRIDE + at] : 0;
    int rank = 0;
#pragma unroll
    for (int w = 0; w < SEGS; ++w)
#pragma unroll 4
      for (int j = part; j < n[w]; j += 4) rank += cand[w * STRIDE + j] > key;
    rank += __builtin_amdgcn_mov_dpp(rank, kDppXor1, 0xF, 0xF, false);
    rank += __builtin_amdgcn_mov_dpp(rank, kDppXor2, 0xF, 0xF, false);
    if (part == 0 && i < total && rank < top) out(rank, key);
  }
}

struct LpShared {
  float f[4][4];
  uint4 order[64];  // of the threads' maxima
  int n[2][4];
  key_t64 cand[kCand];
};

// m; s and t in units.
struct RowSums {
  float m, s, t;
};
__device__ __forceinline__ bool row_empty(const RowSums& r) {
  return r.m == -__builtin_huge_valf() && r.s == 0.0f;
}
__device__ __forceinline__ float logp_of(const RowSums& r, float ls, float x) {
  if (row_empty(r)) return -__builtin_huge_valf();
  return (float)(((double)x - (double)r.m) - (double)ls);
}
// A row's token and its logit, asked for first and used last.
struct Given {
  int t;
  float x;
};
__device__ __forceinline__ Given given(const LpArgs& a, int row) {
  Given g{-1, 0.0f};
  if (a.logp) {
    g.t = a.tokens[row];
    if (g.t >= 0 && g.t < a.V) g.x = a.x[row * a.ld + g.t];
  }
  return g;
}
__device__ __forceinline__ void write_row(const LpArgs& a, int row, const Given& g,
                                          const RowSums& r, float ls) {
  if (a.logp) {
    float v = 0.0f;
    if (g.t >= a.V || g.t < -1) v = __builtin_nanf("");
    else if (g.t >= 0) v = logp_of(r, ls, g.x);
    a.logp[row] = v;
  }
  if (a.entropy) a.entropy[row] = row_empty(r) ? 0.0f : ls - r.t * kUnit / (1.0f + r.s * kUnit);
}

template <int NV, bool TOP>
__global__ __launch_bounds__(256) void logprob_kernel(LpArgs a) {
  __shared__ LpShared sh;
  const int tid = threadIdx.x, wave = tid >> 6;
  const int row = blockIdx.x / a.pieces, piece = blockIdx.x % a.pieces;
  const int begin = piece * a.len, n = min(a.len, a.V - begin);
  const float* x = a.x + row * a.ld + begin;
  const float inf = __builtin_huge_valf();
  const Given tok = a.pieces > 1 ? Given{} : given(a, row);
  float v[NV][4];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k = (tid + 256 * i) * 4;
    if (k + 4 <= n) {
      const float4u u = __builtin_nontemporal_load(reinterpret_cast<const float4u*>(x + k));
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
  if constexpr (TOP) {
    // a NaN is no maximum, but the largest logit
    unsigned o = order_of(m);
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) o = v[i][e] != v[i][e] ? 0xffffffffu : o;
    reinterpret_cast<unsigned*>(sh.order)[tid] = o;
  }
  m = wave_max(m);
  if ((tid & 63) == 0) sh.f[wave][0] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sh.f[0][0], sh.f[1][0]), fmaxf(sh.f[2][0], sh.f[3][0]));
  const float ref = m == -inf ? 0.0f : m;
  float s = 0.0f, t = 0.0f;
  int maxima = 0;  // of the wave
#pragma unroll
  for (int i = 0; i < NV; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float d = v[i][e] - ref;
      const float p = exp_of(d);
      const bool is_max = d == 0.0f;
      maxima += lanes(is_max);
      s += is_max ? 0.0f : p;
      t = fmaf(p, fmaxf(d, -200.0f), t);  // far below, p is 0
    }
    asm volatile("" : "+s"(maxima));  // counted here, not kept as 4 NV masks
  }
  s = wave_sum(s);
  t = wave_sum(t);
  float tops = (float)maxima;
  if ((tid & 63) == 0) {
    sh.f[wave][1] = s;
    sh.f[wave][2] = t;
    sh.f[wave][3] = tops;
  }
  __syncthreads();
  RowSums r;
  r.m = m;
  r.t = kUnits * ((sh.f[0][2] + sh.f[1][2]) + (sh.f[2][2] + sh.f[3][2]));
  tops = (sh.f[0][3] + sh.f[1][3]) + (sh.f[2][3] + sh.f[3][3]);
  r.s = (sh.f[0][1] + sh.f[1][1]) + (sh.f[2][1] + sh.f[3][1]);
  if (tops > 0.0f) r.s += tops - 1.0f;
  r.s *= kUnits;
  // rows of one open logit have nothing to sum (1531 x 6761 of these 10.8 us in place of 14.7)
  auto others = [&]() {
    bool c = false;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) c |= v[i][e] > -inf && v[i][e] < m;
    return __syncthreads_or(c);
  };
  if (too_small(m, r.s) && others()) {  // of the whole workgroup
    s = t = 0.0f;
    // read again: kept for this they would cost the usual row its occupancy (1000 x 151936 with 20
    // alternatives 135 -> 156 us)
#pragma unroll 2
    for (int k = 4 * tid; k < n; k += 1024) {
      float4u u{-inf, -inf, -inf, -inf};
      if (k + 4 <= n) {
        u = *reinterpret_cast<const float4u*>(x + k);
      } else {
#pragma unroll
        for (int e = 0; e < 3; ++e)
          if (k + e < n) u[e] = x[k + e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float d = u[e] - m, p = d == 0.0f ? 0.0f : exp_units(d);
        s += p;
        t = fmaf(p, fmaxf(d, -200.0f), t);
      }
    }
    s = wave_sum(s);
    t = wave_sum(t);
    __syncthreads();  // the first sums are read
    if ((tid & 63) == 0) {
      sh.f[wave][1] = s;
      sh.f[wave][2] = t;
    }
    __syncthreads();
    r.s = (sh.f[0][1] + sh.f[1][1]) + (sh.f[2][1] + sh.f[3][1]);
    r.t = (sh.f[0][2] + sh.f[1][2]) + (sh.f[2][2] + sh.f[3][2]);
  }
  const float ls = log1pf(r.s * kUnit);
  if (a.pieces > 1) {
    if (tid == 0) a.part[blockIdx.x] = make_float4(r.m, r.s, r.t, 0.0f);
  } else if (tid == 0) {
    write_row(a, row, tok, r, ls);
  }
  if constexpr (TOP) {
    const int top = a.top;
    const uint4 g = sh.order[tid & 63];
    const unsigned bound = largest_with(top, 31, 16, [&](unsigned mid) {
      return lanes(g.x >= mid) + lanes(g.y >= mid) + lanes(g.z >= mid) + lanes(g.w >= mid);
    });
    // not below the bound as a number: a NaN is never below, and nothing is below a bound that
    // is no number (an order of NaNs, or below that of -inf)
    float from = value_of(bound);
    int last = kPiece;  // of the logits equal to `from`, the ones up to here
    bool nans = false;
    int n[4];
    // Every pass over the logits takes them and their indices anew: what the compiler would keep
    // of one pass for the next (masks, orders, indices: 32 of each) costs the occupancy.
    auto anew = [&](int& t4) {
      asm volatile("" : "+v"(t4));
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) asm volatile("" : "+v"(v[i][e]));
    };
    // into this wave's segment; false if one is too small
    auto gather = [&](auto chosen) {
      int at = 0, t4 = 4 * tid;
      anew(t4);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int k = t4 + 1024 * i + e;
          const bool c = chosen(v[i][e], k);
          const unsigned long long mask = __ballot(c);
          if (mask) {
            const int to = at + lanes_below(mask);
            if (c && to < kSeg)
              sh.cand[wave * kSeg + to] =
                  key_of(nans ? 0xffffffffu : order_of(v[i][e]), begin + k);
            at += __popcll(mask);
          }
        }
      if ((tid & 63) == 0) sh.n[0][wave] = at;
      __syncthreads();
      bool fit = true;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        n[w] = sh.n[0][w];
        fit &= n[w] <= kSeg;
      }
      return fit;
    };
    // counts of all four waves, a barrier each
    int turn = 1;
    auto count = [&](auto f) {
      int c = 0, t4 = 4 * tid;
      anew(t4);
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e) c += lanes(f(v[i][e], t4 + 1024 * i + e));
      if ((tid & 63) == 0) sh.n[turn][wave] = c;
      __syncthreads();
      c = (sh.n[turn][0] + sh.n[turn][1]) + (sh.n[turn][2] + sh.n[turn][3]);
      turn ^= 1;
      return c;
    };
    bool fit;
    if (bound <= order_of(-inf)) {
      // Fewer threads than `top` have a logit that is not masked (the others of a constrained
      // choice, a whole piece of a masked vocabulary): these logits, and of the masked ones the
      // lowest indices, `top` of which stand among as many indices as both together.
      const int open = count([&](float x, int) { return !(x <= -inf); });
      fit = gather([&](float x, int k) { return !(x <= -inf) || k < open + top; });
    } else {
      fit = gather([&](float x, int) { return !(x < from); });
    }
    if (!fit) {
      turn = 1;  // sh.n[0] may still be read
      nans = count([](float x, int) { return x != x; }) >= top;
      if (nans) {
        // NaNs alone, the lowest indices: as infinities, the rest as nothing
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) v[i][e] = v[i][e] != v[i][e] ? inf : -inf;
      }
      // orders up to that of +inf
      const unsigned exact = largest_with(top, 31, 0, [&](unsigned mid) {
        const float at = value_of(mid);
        return mid > 0xff800000u ? 0 : count([&](float x, int) { return !(x < at); });
      });
      from = value_of(exact);
      const int above = count([&](float x, int) { return !(x <= from); });
      last = kPiece - 1 - (int)largest_with(top - above, 12, 0, [&](unsigned mid) {
        return count([&](float x, int k) { return x == from && kPiece - 1 - k >= (int)mid; });
      });
      __syncthreads();  // the last counts are read
      gather([&](float x, int k) { return !(x < from) && (!(x == from) || k <= last); });
    }
    rank_keys<256, 4, kSeg>(sh.cand, n, top, [&](int at, key_t64 key) {
      if (a.pieces > 1) {
        a.keys[(long)blockIdx.x * top + at] = key;
      } else {
        a.top_ids[(long)row * top + at] = (int)~(unsigned)key;
        a.top_logp[(long)row * top + at] = logp_of(r, ls, value_of((unsigned)(key >> 32)));
      }
    });
  }
}

// The pieces of a row, one wave.  NR: keys a lane holds (0: any number, read again for each bit).
template <int NR>
__global__ __launch_bounds__(64) void logprob_join_kernel(LpArgs a) {
  __shared__ key_t64 cand[kJoin];
  const int lane = threadIdx.x, row = blockIdx.x;
  const float4* part = a.part + (long)row * a.pieces;
  const float inf = __builtin_huge_valf();
  const key_t64* keys = a.keys + (long)row * a.pieces * a.top;
  const int n = a.pieces * a.top, each = (n + 63) / 64;
  const Given tok = given(a, row);
  key_t64 own[NR ? NR : 1];
#pragma unroll
  for (int i = 0; i < NR; ++i) own[i] = lane + 64 * i < n ? keys[lane + 64 * i] : 0;
  float m = -inf;
  for (int i = lane; i < a.pieces; i += 64) m = fmaxf(m, part[i].x);
  m = wave_max(m);
  RowSums r;
  r.m = m;
  auto sums = [&](bool small) {
    float s = 0.0f, t = 0.0f, tops = 0.0f;
    for (int i = lane; i < a.pieces; i += 64) {
      const float4 p = part[i];
      if (p.x == m) {
        s += p.y;
        t += p.z;
        tops += 1.0f;
      } else if (p.x == -inf) {
        s += p.y;  // 0, or the NaN of such a piece
      } else {
        const float d = p.x - m, far = fmaxf(d, -200.0f);
        const float w = small ? exp_units(d) : exp_of(d) * kUnits;
        const float one = 1.0f + p.y * kUnit;  // of the piece's own maximum
        s = fmaf(w, one, s);
        t = fmaf(w, fmaf(one, far, p.z * kUnit), t);
      }
    }
    r.t = wave_sum(t);
    r.s = wave_sum(s);
    tops = wave_sum(tops);
    if (m != -inf) r.s += (tops - 1.0f) * kUnits;
  };
  sums(false);
  if (too_small(m, r.s)) sums(true);
  const float ls = log1pf(r.s * kUnit);
  if (lane == 0) write_row(a, row, tok, r, ls);
  if (!a.top) return;
  // every lane calls f with `each` keys, 0 for none
  auto all = [&](auto f) {
    if constexpr (NR) {
#pragma unroll
      for (int i = 0; i < NR; ++i) f(own[i]);
    } else {
      for (int i = 0; i < each; ++i) f(lane + 64 * i < n ? keys[lane + 64 * i] : 0);
    }
  };
  auto count = [&](auto f) {
    int c = 0;
    all([&](key_t64 key) { c += lanes(f(key)); });
    return c;
  };
  auto with = [&](unsigned mid) {
    return count([&](key_t64 key) { return (unsigned)(key >> 32) >= mid; });
  };
  unsigned order = largest_with(a.top, 31, 16, with);
  key_t64 bound = (key_t64)order << 32;
  int c = with(order);
  if (c > kJoin) {  // crowded: the exact order, and of its ties the lowest indices, 24 bits of them
    order = largest_with(a.top, 31, 0, with);
    const int above = count([&](key_t64 key) { return (unsigned)(key >> 32) > order; });
    bound = (key_t64)order << 32 | 0xff000000u;
    bound |= largest_with(a.top - above, 23, 0, [&](unsigned mid) {
      const key_t64 from = bound | mid;
      return count([&](key_t64 key) { return key >= from && (unsigned)(key >> 32) == order; });
    });
    c = a.top;
  }
  int at = 0;
  all([&](key_t64 key) {
    const bool in = key >= bound;
    const unsigned long long mask = __ballot(in);
    if (in) cand[at + lanes_below(mask)] = key;
    at += __popcll(mask);
  });
  __syncthreads();
  const int in_all[1] = {c};
  rank_keys<64, 1, kJoin>(cand, in_all, a.top, [&](int place, key_t64 key) {
    a.top_ids[(long)row * a.top + place] = (int)~(unsigned)key;
    a.top_logp[(long)row * a.top + place] = logp_of(r, ls, value_of((unsigned)(key >> 32)));
  });
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
  // rows of logits may be read behind another row's outputs
  auto over = [&](const void* p, size_t floats) {
    return p && rows_overlap(logits, ld, V, static_cast<const float*>(p), 0, (long)floats, rows);
  };
  const size_t alts = (size_t)rows * top;
  LX_REQUIRE(!over(logp, rows) && !over(entropy, rows) &&
                 !(top && (over(top_logp, alts) || over(top_ids, alts))) &&
                 !(a.pieces > 1 && over(ws, lx_token_logprobs_ws_floats(rows, V, top))),
             "token_logprobs: an output or the workspace overlaps the logits");
  if (top)
    launch_logprob<true>(a, rows, stream);
  else
    launch_logprob<false>(a, rows, stream);
  LX_TRY(check_launch("logprob_kernel"));
  if (a.pieces == 1) return LX_OK;
  const dim3 grid((unsigned)rows), block(64);
  if (a.pieces * a.top <= 8 * 64)
    hipLaunchKernelGGL(logprob_join_kernel<8>, grid, block, 0, stream, a);
  else if (a.pieces * a.top <= 20 * 64)
    hipLaunchKernelGGL(logprob_join_kernel<20>, grid, block, 0, stream, a);
  else
    hipLaunchKernelGGL(logprob_join_kernel<0>, grid, block, 0, stream, a);
  return check_launch("logprob_join_kernel");
}
