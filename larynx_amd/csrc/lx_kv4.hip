// A key/value cache held in 4 bits: append, read back, attention over it.
//
// The 64 channels of a group (one head at head_dim 64, half of one at 128) of one cached row
// share z = the largest bf16 not above their minimum and s = the smallest bf16 not below
// (max - z) / 15; a code q = rint((x - z) / s) stands for x~ = z + s q, so every value lies
// inside the range and is off by at most s / 2.  4.5 bits a value.
//
// Layout: per sequence, kv head and block of 32 rows one record of 2304 bytes a channel group:
// 1 KB of key codes, 1 KB of value codes, then per row the key and the value (s, z) pairs as
// dwords (s low, z high).  Both code planes are MFMA fragments (lx_four_bit.hpp), 16 bytes a
// lane: for S^T = K Q^T the keys are rows and the channels k, for O^T = V^T P^T the channels are
// rows and the keys k.  The order of the 32 keys in V's k index is the one in which a lane
// already holds its scores (4 c .. 4 c + 3 of both 16-key tiles, c = lane / 16), so the softmax
// weights go from one product's result to the other's operand without leaving the lane.
#include <algorithm>
#include <climits>

#include "lx_four_bit.hpp"

namespace lx {
namespace {

constexpr int kBlk = 32;       // rows of a record
constexpr int kGrp = 64;       // channels of a group
constexpr int kCodes = 1024;   // bytes of one group's key (or value) codes in a record
constexpr int kRec = 2 * kCodes + 2 * kBlk * 4;  // bytes of a record, per channel group
constexpr long kMaxThreads = 0xffffff00L;        // of a launch along x

// Record of (sequence, kv head, block): ng groups of key codes, ng of value codes, ng x 32 key
// (s, z), ng x 32 value (s, z).
struct Kv4 {
  char* data;
  int batch, heads, ng, rows, blocks;
  __host__ __device__ size_t record(int b, int h, int blk) const {
    return (((size_t)b * heads + h) * blocks + blk) * ((size_t)ng * kRec);
  }
};

struct AppendArgs {
  Kv4 c;
  const float *k, *v;
  long ldk, ldv;
  int T;
  const int* pos;
};

// z and s of a group with extremes lo and hi (finite).  Both quotients here decide by a border, so
// they are the 64-bit ones; where the fp32 quotient (off by less than 2^-21 of itself) is clear of
// every border, which is all but one in some thousands, it decides the same.
struct Affine {
  float s, z;
};
__device__ __forceinline__ Affine affine(float lo, float hi) {
  unsigned zb = __float_as_uint(lo);
  const unsigned cut = zb & 0xffff0000u;
  zb = lo < 0.0f && cut != zb ? cut + 0x10000u : cut;
  Affine a;
  a.z = __uint_as_float(zb);
  unsigned sb = __float_as_uint((hi - a.z) * (1.0f / 15.0f));
  const unsigned low = sb & 0xffffu;
  if (low < 64u || low > 0xffffu - 64u || sb < 0x01000000u) {  // a bf16 number near, or tiny
    const double r = ((double)hi - (double)a.z) / 15.0;
    const float f = (float)r;
    sb = __float_as_uint(f) + ((double)f < r ? 1u : 0u);
  }
  a.s = __uint_as_float((sb + 0xffffu) & 0xffff0000u);
  return a;
}
__device__ __forceinline__ unsigned affine_code(float x, Affine a) {
  if (!(a.s > 0.0f)) return 0;
  const float u = (x - a.z) * (1.0f / a.s);
  float q = rintf(u);
  // (a subnormal s has no inverse: u is then infinite or NaN)
  if (__any(!(fabsf(fabsf(u - q) - 0.5f) > 1e-4f && u < 64.0f)))
    q = (float)rint(((double)x - (double)a.z) / (double)a.s);
  return (unsigned)(int)fminf(fmaxf(q, 0.0f), 15.0f);
}

// Code and pair of one group, lane = channel.  A group that holds an infinity or a NaN, or whose
// |z| + 16 s passes fp32, stores NaN.
__device__ __forceinline__ unsigned quantise(float x, unsigned* pair) {
  const float hi = wave_max(x), lo = -wave_max(-x);
  const bool bad = __any(!(fabsf(x) <= 3.402823466e38f));
  const Affine a = affine(lo, hi);
  if (bad || !(fmaf(16.0f, a.s, fabsf(a.z)) <= 3.402823466e38f)) {
    *pair = 0x7fc07fc0u;
    return 0;
  }
  *pair = __float_as_uint(a.s) >> 16 | (__float_as_uint(a.z) & 0xffff0000u);
  return affine_code(x, a);
}

// One workgroup of eight waves per (32-row record touched, channel group of a kv head, sequence):
// four for the keys, four for the values, lane = channel.  Wave w of a plane owns the rows whose
// value codes share dwords, 4 w .. 4 w + 3 of both halves; all eight are requested at once.  A wave
// is some 140 instructions a group (two wave-wide extremes, two quotients, the code) after one
// memory round trip, and these bound it: 1531 rows of 2 heads 7.2 us, 1.8 MB; one row 3.3, a launch
// and its chain.
__global__ __launch_bounds__(512) void kv4_append_kernel(AppendArgs a) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6 & 3, plane = threadIdx.x >> 8;
  const int ng = a.c.ng, hg = blockIdx.y, b = blockIdx.z;  // hg: head * ng + group
  const int h = ng == 1 ? hg : hg >> 1, g = ng == 1 ? 0 : hg & 1;
  const long pos = a.pos[b];
  const long blk = max(pos, 0L) / kBlk + blockIdx.x;
  if (blk >= a.c.blocks) return;
  char* rec = a.c.data + a.c.record(b, h, (int)blk);
  const long t0 = blk * kBlk - pos;  // the record's first row in k and v
  auto row_of = [&](int j) { return 4 * w + (j & 3) + 16 * (j >> 2); };
  const float* src = plane ? a.v : a.k;
  const long ld = plane ? a.ldv : a.ldk;
  float x[8];
  bool live[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const long t = t0 + row_of(j);
    live[j] = t >= 0 && t < a.T && blk * kBlk + row_of(j) < a.c.rows;
    x[j] = src[((long)b * a.T + min(max(t, 0L), (long)a.T - 1)) * ld + (long)hg * kGrp + lane];
  }
  unsigned kept = 0, mask = 0, pairs = 0;  // keys: the lane's dword of row lane % 8
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (!live[j]) continue;  // uniform
    unsigned pair;
    const unsigned q = quantise(x[j], &pair);
    if ((lane & 7) == j) pairs = pair;
    if (plane) {
      kept |= q4_put(q, j);
      mask |= q4_put(15u, j);
    } else {
      // eight channels make a dword
      int kw = (int)q4_put(q, lane & 7);
      kw |= __builtin_amdgcn_mov_dpp(kw, kDppXor1, 0xF, 0xF, false);
      kw |= __builtin_amdgcn_mov_dpp(kw, kDppXor2, 0xF, 0xF, false);
      kw |= __builtin_amdgcn_mov_dpp(kw, kDppHalfMirror, 0xF, 0xF, false);
      if ((lane & 7) == j) kept = (unsigned)kw;
    }
  }
  const int j = lane & 7, r = row_of(j), o = lane >> 3;
  const long tj = t0 + r;
  const bool mine = tj >= 0 && tj < a.T && blk * kBlk + r < a.c.rows;
  unsigned* codes = reinterpret_cast<unsigned*>(rec + (plane * ng + g) * kCodes);
  if (plane) {
    if (mask) {
      unsigned* p = codes + (w * 16 + (lane & 15)) * 4 + (lane >> 4);
      *p = mask == ~0u ? kept : (*p & ~mask) | kept;
    }
  } else if (mine) {
    codes[(((o & 3) * 16 + (r & 15)) * 2 + (r >> 4)) * 2 + (o >> 2)] = kept;
  }
  if (lane < 8 && mine)
    reinterpret_cast<unsigned*>(rec + 2 * ng * kCodes)[(plane * ng + g) * kBlk + r] = pairs;
}

struct ReadArgs {
  Kv4 c;
  float *k, *v;
  int T;
  const int* pos;
};

// One thread per (row, channel) of a sequence; rows outside the cache read as zero.  1531 rows of 2
// heads 3.0 us, bound by launch and latency.
__global__ __launch_bounds__(256) void kv4_read_kernel(ReadArgs a) {
  const int hd = a.c.ng * kGrp, width = a.c.heads * hd, b = blockIdx.y;
  const long i = (long)blockIdx.x * 256 + threadIdx.x;
  if (i >= (long)a.T * width) return;
  const long t = i / width;
  const int wc = (int)(i - t * width), h = wc / hd, ch = wc - h * hd;
  const long row = (long)a.pos[b] + t;
  float k = 0.0f, v = 0.0f;
  if (row >= 0 && row < a.c.rows) {
    const char* rec = a.c.data + a.c.record(b, h, (int)(row / kBlk));
    const int r = (int)(row % kBlk), g = ch / kGrp, x = ch % kGrp, ng = a.c.ng;
    const unsigned* kc = reinterpret_cast<const unsigned*>(rec + g * kCodes);
    const unsigned* vc = reinterpret_cast<const unsigned*>(rec + (ng + g) * kCodes);
    const unsigned* pairs = reinterpret_cast<const unsigned*>(rec + 2 * ng * kCodes);
    const unsigned kw = kc[((((x >> 3) & 3) * 16 + (r & 15)) * 2 + (r >> 4)) * 2 + (x >> 5)];
    const unsigned vw = vc[(((r & 15) >> 2) * 16 + (x & 15)) * 4 + (x >> 4)];
    const unsigned kp = pairs[g * kBlk + r], vp = pairs[(ng + g) * kBlk + r];
    k = fmaf(bf16_lo(kp), (float)q4_get(kw, x & 7), bf16_hi(kp));
    v = fmaf(bf16_lo(vp), (float)q4_get(vw, (r & 3) + 4 * (r >> 4)), bf16_hi(vp));
  }
  const long to = (long)b * a.T * width + i;
  a.k[to] = k;
  a.v[to] = v;
}

// ---- attention --------------------------------------------------------------------------

constexpr int kMaxWaves = 8;    // of an attention workgroup
constexpr int kMaxSplits = 64;  // of a sequence's keys
constexpr int kQ = 16;  // columns of a tile: query rows, (t, head of the group) pairs, t-major

struct AttnArgs {
  Kv4 c;
  const float* q;
  long ldq;
  const int* lens;
  float* o;
  long ldo;
  float* ws;
  int Tq, rep, tiles, splits, chunk, causal;
  int kshift;  // log2 of the records side by side; a tile has 16 >> kshift query rows
  float scale2;  // scale * log2(e)
};

// The keys of a tile of query rows, in steps of 1 << kshift records: split sp takes steps [sp *
// per, sp * per + per) of n_step.  A split is a.chunk steps long, so that the workgroups of
// sequences of all lengths have the same work, and longer only where a sequence passes the
// length the launch was sized for.
struct Span {
  int most, least;  // the longest and the shortest run of keys a row of the tile sees
  int n_blk, n_step, per;
};
__device__ __forceinline__ Span attn_span(const AttnArgs& a, int len, int qt, int nrow) {
  Span s;
  s.most = s.least = len;
  if (a.causal && a.Tq > 1) {
    const int rows = kQ >> a.kshift, first = qt * rows;
    const int t_first = first / a.rep, t_last = min(first + rows - 1, nrow - 1) / a.rep;
    s.most = max(len - a.Tq + t_last + 1, 0);
    s.least = max(len - a.Tq + t_first + 1, 0);
  }
  s.n_blk = (s.most + kBlk - 1) / kBlk;
  s.n_step = (s.n_blk + (1 << a.kshift) - 1) >> a.kshift;
  s.per = a.chunk;
  if (s.n_step > a.chunk * a.splits) s.per = (s.n_step + a.splits - 1) / a.splits;
  return s;
}

// Channels chn .. chn + 3 of query row rr: O / L, zero where no key was seen (L = 0).
__device__ __forceinline__ void store_row(const AttnArgs& a, int b, int h, int rr, int chn, int hd,
                                          float4 O, float L) {
  const float inv = L == 0.0f ? 0.0f : 1.0f / L;
  float* dst =
      a.o + ((long)b * a.Tq + rr / a.rep) * a.ldo + (long)(h * a.rep + rr % a.rep) * hd + chn;
  *reinterpret_cast<float4*>(dst) = make_float4(O.x * inv, O.y * inv, O.z * inv, O.w * inv);
}

// Partial states in the workspace, per (sequence, kv head, query tile, split): 16 rows of hd
// unnormalised outputs, then 16 maxima (in units of log2) and 16 sums.
__host__ __device__ constexpr long part_floats(int ng) { return (long)kQ * (ng * kGrp + 2); }

// Among the four lanes of a column, l, l ^ 16, l ^ 32 and l ^ 48 (a swap leaves each lane with
// its own and the other's value, in either order).
template <class F>
__device__ __forceinline__ float over_column(float v, F f) {
  const unsigned a = __float_as_uint(v);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const unsigned b = __float_as_uint(f(__uint_as_float(r[0]), __uint_as_float(r[1])));
  const auto q = __builtin_amdgcn_permlane32_swap(b, b, false, false);
  return f(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float column_max(float v) {
  return over_column(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ float column_sum(float v) {
  return over_column(v, [](float a, float b) { return a + b; });
}

// The weights p s of one group's values as fp16 parts: a column's carry a power of two, `lift`,
// that brings the largest of them so far to 2^6 .. 2^7, where the second part ends 2^-31 below it.
// bound: 256 times that largest product; the lift lasts until a product passes it (2^15; fp16 ends
// at 2^16).  Moves the lift to a new bound; returns what sums that carried the old one, and kept
// `keep` of themselves, are multiplied by.
__device__ __forceinline__ float move_lift(float bound, float keep, float& lift) {
  const int e = (int)(__float_as_uint(bound) >> 23 & 255u);
  const int now = min(141 - e, 126), was = (int)(__float_as_uint(lift) >> 23) - 127;
  lift = __uint_as_float((unsigned)(now + 127) << 23);
  return ldexpf(keep, now - was);
}

// One workgroup of up to kMaxWaves waves per (sequence, kv head, tile of query rows, split of the
// keys).  A tile has 16 / KP query rows, the columns of the matrix instructions; with KP > 1 (few
// query rows: single tokens) the rows stand KP times side by side and a step takes KP records, the
// i-th set of columns the softmax of the i-th record, so that no lane works on a row that is not
// there.  The waves take the steps in turn, each column with a running softmax of its own.
// Scores are transposed: lane l holds column l % 16.  Codes count from their middle, x~ = (z + 8
// s) + s (q - 8).  q carries scale * log2 e and the power of two that its two fp16 parts want (S'
// = S / f, f a constant of the row).  The weights p s of the values want one too, a running
// reference like the maximum (move_lift).  It follows the products: taken from the scales alone, a
// row of large values that weighs nothing pushes the others' parts out of fp16's range (2^20 times
// as large: outputs off by 5e-4).
// Half a byte a value and one read of it: the vector instructions beside the products bound long
// contexts, some 920 a step of four 128-channel records (codes to fragments 576, the softmax and
// the weights' two parts most of the rest; the matrix pipe is 0.13 busy): 2 sequences of 65536
// rows, 8 kv heads, 114 MB in 33 us, 3.4 TB/s, and 4 to 5 for the join; 64 sequences of all lengths
// up to 4096, 153 MB, 53 us with the join, 2.9 TB/s.  Short ones are latency: 1 sequence of 2001
// rows 5.2 us and 3.1 for the join, 7.6 for both in a graph.
// A spilled register costs more than a wave gains: the registers follow from NG and KP.
template <int NG, int KP>
__global__ __launch_bounds__(64 * kMaxWaves) __attribute__((
    amdgpu_waves_per_eu(NG == 2 ? 2 : KP == 4 ? 3 : 4))) void kv4_attn_kernel(AttnArgs a) {
  constexpr int HD = NG * kGrp, R = kQ / KP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  float (*om)[kQ][HD + 4] = reinterpret_cast<float (*)[kQ][HD + 4]>(lds);
  const int tid = threadIdx.x, lane = tid & 63, waves = blockDim.x >> 6;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  float (*ml)[2][kQ] =
      reinterpret_cast<float (*)[2][kQ]>(lds + (size_t)waves * kQ * (HD + 4) * sizeof(float));
  const int col = lane & 15, c = lane >> 4, set = col / R;
  const unsigned pattern = q4_pattern();
  const int h = blockIdx.y, b = blockIdx.z;
  int sp = blockIdx.x, qt = 0;
  if (KP == 1 && a.tiles > 1) {
    qt = sp / a.splits;
    sp -= qt * a.splits;
  }
  const int nrow = a.Tq * a.rep;
  const int row = qt * R + col % R;        // the lane's query row
  int t = 0, hr = min(row, nrow - 1);
  if (a.Tq > 1) {
    t = hr / a.rep;
    hr -= t * a.rep;
  }
  // the query first: it is on its way while the length and the records arrive
  float4 qx[NG][2][2];
  {
    const float* q = a.q + ((long)b * a.Tq + t) * a.ldq + (long)(h * a.rep + hr) * HD + c * 8;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          qx[g][ks][e] = *reinterpret_cast<const float4*>(q + g * kGrp + ks * 32 + 4 * e);
  }
  const int len = min(max(a.lens[b], 0), a.c.rows);
  const Span n = attn_span(a, len, qt, nrow);
  const int s0 = sp * n.per, s1 = min(s0 + n.per, n.n_step);
  if (sp > 0 && s0 >= s1) return;
  // keys the row sees: [0, limit)
  const int limit = row >= nrow ? 0 : a.causal ? max(len - a.Tq + t + 1, 0) : len;

  const size_t rstride = (size_t)NG * kRec;
  const char* recs = a.c.data + a.c.record(b, h, 0);
  // a step's operands: the codes of KP records, and the (s, z) pairs of the lane's own one, keys 4
  // c + e and 16 + 4 c + e.  Past the last record the last one stands in, masked by its index.
  uintx4_t kc[KP][NG], vc[KP][NG], kp[NG][2], vp[NG][2];
  auto load = [&](int st, int plane, uintx4_t (&codes)[KP][NG], uintx4_t (&pairs)[NG][2]) {
    const char* own = recs + min(st * KP + set, n.n_blk - 1) * rstride;
#pragma unroll
    for (int g = 0; g < NG; ++g) {
#pragma unroll
      for (int r = 0; r < KP; ++r)
        codes[r][g] = reinterpret_cast<const uintx4_t*>(
            recs + min(st * KP + r, n.n_blk - 1) * rstride + (plane * NG + g) * kCodes)[lane];
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pairs[g][i] = reinterpret_cast<const uintx4_t*>(
            own + 2 * NG * kCodes)[(plane * NG + g) * 8 + i * 4 + c];
    }
  };
  if (s0 + wave < s1) {
    load(s0 + wave, 0, kc, kp);
    load(s0 + wave, 1, vc, vp);
  }

  // every wave splits the whole tile's query the same way; two groups of it would hold 32
  // registers, so with two they stay in LDS (wave 0's)
  half8_t qf[NG][2][2];
  half8_t* ql = reinterpret_cast<half8_t*>(ml + waves) + lane;
  float qsum[NG], f;
  {
    float x[NG][2][8], top = 0.0f;
#pragma unroll
    for (int g = 0; g < NG; ++g)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 u = qx[g][ks][e];
          x[g][ks][4 * e] = u.x * a.scale2;
          x[g][ks][4 * e + 1] = u.y * a.scale2;
          x[g][ks][4 * e + 2] = u.z * a.scale2;
          x[g][ks][4 * e + 3] = u.w * a.scale2;
#pragma unroll
          for (int j = 0; j < 4; ++j) top = fmaxf(top, fabsf(x[g][ks][4 * e + j]));
        }
    const float sc = row_scale(column_max(top), &f);
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float s = 0.0f;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(x[g][ks][j], sc, s);
        split2(x[g][ks], sc, qf[g][ks][0], qf[g][ks][1]);
        if (NG == 2 && wave == 0) {
          ql[(g * 4 + ks * 2) * 64] = qf[g][ks][0];
          ql[(g * 4 + ks * 2 + 1) * 64] = qf[g][ks][1];
        }
      }
      qsum[g] = column_sum(s);
    }
    if (NG == 2) __syncthreads();
  }
  floatx4 o[NG][4];
  float zsum[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    zsum[g] = 0.0f;
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) o[g][ct] = floatx4{0.f, 0.f, 0.f, 0.f};
  }
  // m: the largest S' so far; o[g] carries lift[g]
  float m = -INFINITY, l = 0.0f, bound[NG], lift[NG];
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    bound[g] = 0.0f;
    lift[g] = 0x1p126f;
  }

  for (int st = s0 + wave; st < s1; st += waves) {
    float s[8];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      if constexpr (NG == 2) {
        asm volatile("" ::: "memory");  // read here, not ahead of the loop
#pragma unroll
        for (int i = 0; i < 4; ++i) qf[g][i >> 1][i & 1] = ql[(g * 4 + i) * 64];
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        floatx4 dot = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int r = 0; r < KP; ++r) {
          const half8_t k0 = q4_frag(kc[r][g][i * 2], pattern);
          const half8_t k1 = q4_frag(kc[r][g][i * 2 + 1], pattern);
          floatx4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int p = 1; p >= 0; --p)
            acc = mfma_f16(k1, qf[g][1][p], mfma_f16(k0, qf[g][0][p], acc));
#pragma unroll
          for (int e = 0; e < 4; ++e) dot[e] = r == 0 || set == r ? acc[e] : dot[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float ss = bf16_lo(kp[g][i][e]), z = bf16_hi(kp[g][i][e]);
          const float v = fmaf(ss, dot[e], fmaf(8.0f, ss, z) * qsum[g]);
          s[i * 4 + e] = g == 0 ? v : s[i * 4 + e] + v;
        }
      }
    }
    const bool more = st + waves < s1;
    if (more) load(st + waves, 0, kc, kp);
    if ((st + 1) * (KP * kBlk) > n.least) {
      // a key the row does not see may hold anything (NaN, rows never written): neither its
      // score nor its value takes part
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if ((st * KP + set) * kBlk + 16 * (j >> 2) + 4 * c + (j & 3) >= limit) {
          s[j] = -INFINITY;
#pragma unroll
          for (int g = 0; g < NG; ++g) vp[g][j >> 2][j & 3] = 0;
        }
    }
    float mx = s[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) mx = fmaxf(mx, s[j]);
    if (__any(mx > m)) {
      // the sums so far move to the new maximum of their column
      const float mn = fmaxf(m, column_max(mx));
      const float al = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f((m - mn) * f);
      m = mn;
      l *= al;
#pragma unroll
      for (int g = 0; g < NG; ++g) {
        zsum[g] *= al;
        bound[g] *= al;
        const float alo = move_lift(bound[g], al, lift[g]);
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) o[g][ct] *= alo;
      }
    }
    // a row that has seen no key yet: every weight exp2(-inf) = 0.  The difference comes first,
    // so that no weight passes 1 however large the scores
    const float ref = m == -INFINITY ? 0.0f : m;
    float p[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      p[j] = __builtin_amdgcn_exp2f((s[j] - ref) * f);
      l += p[j];
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
      float ps[8], top = 0.0f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float ss = bf16_lo(vp[g][j >> 2][j & 3]), z = bf16_hi(vp[g][j >> 2][j & 3]);
        ps[j] = p[j] * ss;
        top = fmaxf(top, ps[j]);
        zsum[g] = fmaf(p[j], fmaf(8.0f, ss, z), zsum[g]);
      }
      if (__any(top > bound[g])) {
        bound[g] = fmaxf(bound[g], fminf(256.0f * column_max(top), 0x1p127f));
        const float up = move_lift(bound[g], 1.0f, lift[g]);
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) o[g][ct] *= up;
      }
      half8_t p0, p1;
      split2(ps, lift[g], p0, p1);
#pragma unroll
      for (int r = 0; r < KP; ++r) {
        // the weights of this record's columns alone: the others' belong to other values
        const half8_t none = {};
        const half8_t r0 = KP == 1 || set == r ? p0 : none, r1 = KP == 1 || set == r ? p1 : none;
#pragma unroll
        for (int ct = 0; ct < 4; ++ct) {
          const half8_t vf = q4_frag(vc[r][g][ct], pattern);
          o[g][ct] = mfma_f16(vf, r0, mfma_f16(vf, r1, o[g][ct]));
        }
      }
    }
    if (more) load(st + waves, 1, vc, vp);
  }
  // the lane's sums over its keys -> the column's, without the lift
  l = column_sum(l);
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float drop = __uint_as_float((254u << 23) - __float_as_uint(lift[g]));
    zsum[g] = column_sum(zsum[g]);
#pragma unroll
    for (int ct = 0; ct < 4; ++ct) {
      floatx4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = fmaf(o[g][ct][e], drop, zsum[g]);
      *reinterpret_cast<floatx4*>(&om[wave][col][g * kGrp + ct * 16 + 4 * c]) = v;
    }
  }
  if (c == 0) {
    ml[wave][0][col] = m * f;
    ml[wave][1][col] = l;
  }
  __syncthreads();
  // the states of the waves and column sets joined, four threads an output taking every fourth,
  // in a fixed order
  float* part =
      a.ws + ((((long)b * a.c.heads + h) * a.tiles + qt) * a.splits + sp) * part_floats(NG);
  const int qd = tid & 3;
  for (int i = tid >> 2; i < R * (HD / 4); i += blockDim.x >> 2) {
    const int r = i / (HD / 4), chn = i % (HD / 4) * 4, rr = qt * R + r;
    if (rr >= nrow) break;
    float M = -INFINITY;
    for (int e = qd; e < waves * KP; e += 4) M = fmaxf(M, ml[e / KP][0][e % KP * R + r]);
    M = fmaxf(M, dpp_mov<kDppXor1>(M));
    M = fmaxf(M, dpp_mov<kDppXor2>(M));
    const float ref = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int e = qd; e < waves * KP; e += 4) {
      const int w = e / KP, k = e % KP * R + r;
      const float fw = __builtin_amdgcn_exp2f(ml[w][0][k] - ref);
      const float4 u = *reinterpret_cast<const float4*>(&om[w][k][chn]);
      L += fw * ml[w][1][k];
      O.x += fw * u.x;
      O.y += fw * u.y;
      O.z += fw * u.z;
      O.w += fw * u.w;
    }
    auto quad = [](float x) {
      x += dpp_mov<kDppXor1>(x);
      return x + dpp_mov<kDppXor2>(x);
    };
    L = quad(L);
    O = make_float4(quad(O.x), quad(O.y), quad(O.z), quad(O.w));
    if (qd) continue;
    if (a.splits == 1) {
      store_row(a, b, h, rr, chn, HD, O, L);
    } else {
      *reinterpret_cast<float4*>(part + r * HD + chn) = O;
      if (chn == 0) {
        part[kQ * HD + r] = M;
        part[kQ * HD + kQ + r] = L;
      }
    }
  }
}

// The splits' states of a row joined: one workgroup a row, HD / 4 lanes of four channels, the
// other lanes' groups taking every kG-th split; the groups' states are joined in group order, so
// the result does not depend on timing.  A launch and one round trip: 3.1 us for 14 rows, 3.9
// for 672.
template <int NG>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttnArgs a) {
  constexpr int HD = NG * kGrp, L4 = HD / 4, kG = 256 / L4;
  __shared__ float om[kG][HD + 4];
  __shared__ float ml[2][kG];
  const int chn = (int)(threadIdx.x % L4) * 4, gr = (int)(threadIdx.x / L4);
  const int rr = blockIdx.x, h = blockIdx.y, b = blockIdx.z, nrow = a.Tq * a.rep;
  const int qt = rr >> (4 - a.kshift), r = rr - (qt << (4 - a.kshift));
  const float* p =
      a.ws + (((long)b * a.c.heads + h) * a.tiles + qt) * a.splits * part_floats(NG);
  float M = -INFINITY, L = 0.0f;
  float4 O = make_float4(0.f, 0.f, 0.f, 0.f);
  // every state of a group requested before the first is used, and before the length says how
  // many there are
  constexpr int U = kMaxSplits / kG;
  float ms[U], ls[U];
  float4 u[U];
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const float* ps = p + min(gr + i * kG, a.splits - 1) * part_floats(NG);
    ms[i] = ps[kQ * HD + r];
    ls[i] = ps[kQ * HD + kQ + r];
    u[i] = *reinterpret_cast<const float4*>(ps + r * HD + chn);
  }
  const Span n = attn_span(a, min(max(a.lens[b], 0), a.c.rows), qt, nrow);
  const int count = max((n.n_step + n.per - 1) / n.per, 1);
#pragma unroll
  for (int i = 0; i < U; ++i) {
    if (gr + i * kG >= count) {  // no such state
      ms[i] = -INFINITY;
      ls[i] = 0.0f;
      u[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    M = fmaxf(M, ms[i]);
  }
  const float base = M == -INFINITY ? 0.0f : M;
#pragma unroll
  for (int i = 0; i < U; ++i) {
    const float f = __builtin_amdgcn_exp2f(ms[i] - base);
    L += f * ls[i];
    O.x += f * u[i].x;
    O.y += f * u[i].y;
    O.z += f * u[i].z;
    O.w += f * u[i].w;
  }
  *reinterpret_cast<float4*>(&om[gr][chn]) = O;
  if (chn == 0) {
    ml[0][gr] = M;
    ml[1][gr] = L;
  }
  __syncthreads();
  if (gr) return;
  M = -INFINITY;
#pragma unroll
  for (int g = 0; g < kG; ++g) M = fmaxf(M, ml[0][g]);
  const float ref = M == -INFINITY ? 0.0f : M;
  L = 0.0f;
  O = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
  for (int g = 0; g < kG; ++g) {
    const float f = __builtin_amdgcn_exp2f(ml[0][g] - ref);
    const float4 u = *reinterpret_cast<const float4*>(&om[g][chn]);
    L += f * ml[1][g];
    O.x += f * u.x;
    O.y += f * u.y;
    O.z += f * u.z;
    O.w += f * u.w;
  }
  store_row(a, b, h, rr, chn, HD, O, L);
}

// How a call runs: records side by side, tiles of query rows, waves a workgroup, splits of the
// keys and steps of one.
struct AttnPlan {
  int kp, tiles, waves, splits, chunk;
};

AttnPlan attn_plan(const Kv4& c, int nrow, int max_len) {
  AttnPlan p;
  p.kp = nrow <= 4 ? 4 : nrow <= 8 ? 2 : 1;
  p.tiles = (nrow + kQ / p.kp - 1) / (kQ / p.kp);
  const int cus = device_cus(), len = max_len <= 0 || max_len > c.rows ? c.rows : max_len;
  const long wgs = (long)p.tiles * c.batch * c.heads;
  const int steps = (len + kBlk * p.kp - 1) / (kBlk * p.kp);
  // Splits take four waves, one per SIMD, a call without splits up to eight.  The time in
  // sixteenths of a wave's step: workgroups a CU x (steps a wave, and half of one for its start),
  // an eighth less where two waves cover each other's waits, and five steps for the join's
  // launch.  (1 sequence of 2001 rows, 2 kv heads: one split 11.2 us, eight 7.9 with the join; 48
  // of up to 4000: two 17.9, eight 15.0; 2 of 65536, 8 kv heads of 128 channels: 16 37.1, 32 33.9;
  // 64 query rows over 16384: four 33.8, eight 29.9; a prompt chunk of 156 tiles over 1708 rows:
  // one 14.1, two 21.0.)
  constexpr int kWaves = 4, kJoin = 80;
  long best = LONG_MAX;
  p.splits = 1;
  for (const int s : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 40, 48, 64}) {
    if (s > steps) break;
    const long each = (wgs * s + cus - 1) / cus;
    const int waves = s > 1 ? kWaves : kMaxWaves, n = (steps + waves * s - 1) / (waves * s);
    const long half = s > 1 ? 2L * n + 1 : 4L * n + 1;
    const long t = each * half * (each > 1 || s == 1 ? 7 : 8) + (s > 1 ? kJoin : 0);
    if (t < best) {
      best = t;
      p.splits = s;
    }
  }
  p.chunk = (steps + p.splits - 1) / p.splits;
  p.splits = (steps + p.chunk - 1) / p.chunk;
  p.waves = p.splits > 1 ? kWaves : kMaxWaves;
  while (p.waves > 1 && p.waves / 2 >= p.chunk) p.waves /= 2;
  return p;
}

template <int NG, int KP>
int launch_attn(const AttnArgs& a, const AttnPlan& p, hipStream_t s) {
  // states, and the query's fragments with two groups
  constexpr size_t kState = kQ * (NG * kGrp + 6) * sizeof(float), kQuery = NG == 2 ? 8192 : 0;
  const size_t lds = p.waves * kState + kQuery;
  static LdsLimit once;
  LX_TRY(raise_lds_limit(reinterpret_cast<const void*>(kv4_attn_kernel<NG, KP>),
                         kMaxWaves * kState + kQuery, once, "kv4_attn_kernel"));
  hipLaunchKernelGGL((kv4_attn_kernel<NG, KP>),
                     dim3((unsigned)(p.tiles * p.splits), a.c.heads, a.c.batch),
                     dim3(64 * p.waves), lds, s, a);
  return check_launch("kv4_attn_kernel");
}

bool kv4_shape_ok(int batch, int heads, int hd, int rows) {
  return batch > 0 && batch <= 65535 && heads > 0 && heads <= 32767 && (hd == 64 || hd == 128) &&
         rows > 0 && rows <= INT_MAX - 4 * kBlk;  // a step of four records past the last row
}

int kv4_view(const lx_kv4* c, const char* what, Kv4* out) {
  LX_REQUIRE(c && c->data, "%s: null cache", what);
  LX_REQUIRE(kv4_shape_ok(c->batch, c->n_kv_heads, c->head_dim, c->max_rows),
             "%s: bad cache (%d sequences, %d heads of %d, %d rows)", what, c->batch,
             c->n_kv_heads, c->head_dim, c->max_rows);
  LX_REQUIRE((uintptr_t)c->data % 16 == 0, "%s: unaligned cache", what);
  *out = Kv4{static_cast<char*>(c->data), c->batch, c->n_kv_heads, c->head_dim / kGrp, c->max_rows,
             (c->max_rows + kBlk - 1) / kBlk};
  return LX_OK;
}

}  // namespace
}  // namespace lx

using namespace lx;

extern "C" size_t lx_kv4_bytes(int batch, int n_kv_heads, int head_dim, int max_rows) {
  if (!kv4_shape_ok(batch, n_kv_heads, head_dim, max_rows)) return 0;
  return (size_t)batch * n_kv_heads * ((max_rows + kBlk - 1) / kBlk) * (head_dim / kGrp) * kRec;
}

extern "C" int lx_kv4_append_f32(const lx_kv4* cache, const float* k, long ldk, const float* v,
                                 long ldv, int T, const int* pos, hipStream_t stream) {
  AppendArgs a{};
  LX_TRY(kv4_view(cache, "kv4_append", &a.c));
  LX_REQUIRE(k && v && pos, "kv4_append: null pointer");
  const long width = (long)cache->n_kv_heads * cache->head_dim;
  LX_REQUIRE(T > 0 && ldk >= width && ldv >= width, "kv4_append: bad shape T=%d ldk=%ld ldv=%ld",
             T, ldk, ldv);
  a.k = k;
  a.v = v;
  a.ldk = ldk;
  a.ldv = ldv;
  a.T = T;
  a.pos = pos;
  // records that T rows can touch, wherever they begin
  const long touched = std::min<long>(((long)T + kBlk - 2) / kBlk + 1, a.c.blocks);
  LX_REQUIRE(touched * 512 <= kMaxThreads, "kv4_append: T=%d too long", T);
  hipLaunchKernelGGL(kv4_append_kernel,
                     dim3((unsigned)touched, a.c.heads * a.c.ng, cache->batch), dim3(512), 0,
                     stream, a);
  return check_launch("kv4_append_kernel");
}

extern "C" int lx_kv4_read_f32(const lx_kv4* cache, float* k, float* v, int T, const int* pos,
                               hipStream_t stream) {
  ReadArgs a{};
  LX_TRY(kv4_view(cache, "kv4_read", &a.c));
  LX_REQUIRE(k && v && pos, "kv4_read: null pointer");
  LX_REQUIRE(T > 0, "kv4_read: bad shape T=%d", T);
  a.k = k;
  a.v = v;
  a.T = T;
  a.pos = pos;
  const long n = (long)T * cache->n_kv_heads * cache->head_dim;
  LX_REQUIRE(n <= kMaxThreads, "kv4_read: %ld values a sequence", n);
  hipLaunchKernelGGL(kv4_read_kernel, dim3((unsigned)((n + 255) / 256), a.c.batch), dim3(256), 0,
                     stream, a);
  return check_launch("kv4_read_kernel");
}

extern "C" size_t lx_attention_kv4_ws_floats(const lx_kv4* cache, int Tq, int n_heads,
                                             int max_len) {
  Kv4 c;
  if (kv4_view(cache, "attention_kv4_ws_floats", &c) != LX_OK || Tq <= 0 || n_heads <= 0 ||
      n_heads % c.heads || (long)Tq * (n_heads / c.heads) > INT_MAX - kQ)
    return 0;
  const AttnPlan p = attn_plan(c, Tq * (n_heads / c.heads), max_len);
  return p.splits == 1 ? 0
                       : (size_t)p.tiles * c.batch * c.heads * p.splits * part_floats(c.ng);
}

extern "C" int lx_attention_kv4_f32(const float* q, long ldq, const lx_kv4* cache, const int* lens,
                                    float* o, long ldo, int Tq, int n_heads, float scale,
                                    int causal, int max_len, float* ws, size_t ws_floats,
                                    hipStream_t stream) {
  AttnArgs a{};
  LX_TRY(kv4_view(cache, "attention_kv4", &a.c));
  LX_REQUIRE(q && lens && o, "attention_kv4: null pointer");
  const long width = (long)n_heads * cache->head_dim;
  LX_REQUIRE(Tq > 0 && n_heads > 0 && n_heads % a.c.heads == 0 && ldq >= width && ldo >= width &&
                 ldq % 4 == 0 && ldo % 4 == 0,
             "attention_kv4: bad shape Tq=%d heads=%d/%d ldq=%ld ldo=%ld", Tq, n_heads, a.c.heads,
             ldq, ldo);
  LX_REQUIRE(((uintptr_t)q | (uintptr_t)o) % 16 == 0, "attention_kv4: q and o must be 16-byte "
             "aligned");
  LX_REQUIRE((long)Tq * (n_heads / a.c.heads) <= INT_MAX - kQ, "attention_kv4: Tq=%d too long",
             Tq);
  LX_REQUIRE(!rows_overlap(q, ldq, width, o, ldo, width, (long)a.c.batch * Tq),
             "attention_kv4: o overlaps q");
  a.q = q;
  a.ldq = ldq;
  a.lens = lens;
  a.o = o;
  a.ldo = ldo;
  a.Tq = Tq;
  a.rep = n_heads / a.c.heads;
  a.causal = causal != 0;
  a.scale2 = scale * 1.4426950408889634f;
  const AttnPlan p = attn_plan(a.c, Tq * a.rep, max_len);
  a.tiles = p.tiles;
  a.kshift = p.kp == 4 ? 2 : p.kp == 2 ? 1 : 0;
  a.splits = p.splits;
  a.chunk = p.chunk;
  const long wgs = (long)p.tiles * a.c.batch * a.c.heads;
  LX_REQUIRE((long)p.tiles * p.splits * 64 * p.waves <= kMaxThreads &&
                 (long)Tq * a.rep * 256 <= kMaxThreads,
             "attention_kv4: Tq=%d too long", Tq);
  if (p.splits > 1) {
    const size_t need = (size_t)wgs * p.splits * part_floats(a.c.ng);
    LX_REQUIRE(ws && ws_floats >= need && (uintptr_t)ws % 16 == 0,
               "attention_kv4: workspace of %zu floats, %zu needed", ws ? ws_floats : 0, need);
    a.ws = ws;
  }
  if (a.c.ng == 1)
    LX_TRY(p.kp == 4   ? (launch_attn<1, 4>(a, p, stream))
           : p.kp == 2 ? (launch_attn<1, 2>(a, p, stream))
                       : (launch_attn<1, 1>(a, p, stream)));
  else
    LX_TRY(p.kp == 4   ? (launch_attn<2, 4>(a, p, stream))
           : p.kp == 2 ? (launch_attn<2, 2>(a, p, stream))
                       : (launch_attn<2, 1>(a, p, stream)));
  if (p.splits == 1) return LX_OK;
  const dim3 rows((unsigned)(Tq * a.rep), a.c.heads, a.c.batch);
  if (a.c.ng == 1)
    hipLaunchKernelGGL(kv4_join_kernel<1>, rows, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL(kv4_join_kernel<2>, rows, dim3(256), 0, stream, a);
  return check_launch("kv4_join_kernel");
}
