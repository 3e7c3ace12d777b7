// Which tokens of a drafted chain stand, and the token after them, from given
// random numbers, so that what comes out is distributed as the model's own samples.
// (The reference decodes one token per step, dropkv_cache.py:609-617.)
//
// Node i of a chain was drawn from q_{i-1}, the draft model's distribution after
// node i - 1 (or was given: all of q on it); p_{i-1} is the model's there.  Node i
// stands while u_i q(x_i) < p(x_i); after the last node that stands, the next token
// is drawn by u_0 from max(p - q, 0) if a node failed there, from p otherwise: the
// first one whose running sum, in the order of the vocabulary, exceeds u_0 times
// the whole sum.  p and q are e^(x / temperature) over their sums.
//
// A random number may lie next to the border of two tokens, and p - q is a
// difference of near values, so all weights and sums are in 64 bits.  The exponential
// is 2^(k/32), from a table and the exponent, times the Taylor sum of 2^f, |f| <= 1/64,
// to the 4th power, which leaves 10^-12 of it (and moves a border past a given u_0 in
// one sample of 10^6 at the most, with a vocabulary of 150,000), in 9 operations of 64
// bits and 8 others.  32 entries of 8 bytes are one for each pair of LDS banks: no lanes
// wait for one another.
//
// Bound by that arithmetic: the pass over 136 rows of 151936 in bf16 takes 18.3 us,
// whose bytes take 8 (26 us with one sum over |f| <= 1/2, 45 operations): 25 operations
// an element in all, of four cycles each, are 13.5 us.  Over 704 rows of 32003 in fp32 it
// takes 19 to 21, whose bytes take 17.
//
// First the maximum and sum of every row, in segments; then the walk, the sums of the
// weights that are sampled, over pieces of the one row of each sequence, and the token:
// in one kernel for short chains, else in three.
#include "dkv_common.h"
#include "dkv_internal.h"
#include "dkv_select_dev.h"

#include <algorithm>

namespace dkv {

constexpr int kVfThreads = 256;
constexpr int kVfElems = 16;  // elements per thread and tile
constexpr int kVfTile = kVfThreads * kVfElems;
constexpr int kVfMaxSegs = 64;  // a lane each where they are joined

struct VfPart {
  double s;
  float m;
  int pad;
};
struct VfSeq {           // what the walk leaves of a sequence
  double p_mul, q_mul;   // 1 / sum of the sampled node's row, and of its draft's
  float p_m, q_m;        // their maxima
  int last, token;       // the node; the token that failed there, or -1
};
struct VerifyArgs {
  const void* x;  // logits [B, T, V]
  int64_t x_sb, x_st;
  const void* y;  // draft logits [B, T - 1, V], or null
  int64_t y_sb, y_st;
  const int64_t* tokens;  // [B, T]
  const float* u;         // [B, T]
  int B, T, V, S, seg;    // segments per row, elements per segment (whole tiles)
  int pieces, groups;     // of the sampled rows: pieces, and workgroups of eight of them
  double mul;             // log2 e / temperature
  float deep;             // 990 / mul
  VfPart* part;           // [B, T, S], then [B, T - 1, S] of the drafts
  VfSeq* seq;             // [B]
  uint32_t* arrived;      // [B] at arrived_s: workgroups done, of a call in two kernels; null: they do not fit
  int arrived_s;
  double* sums;           // [B, pieces, 2]: of the weights, and of p alone
  int64_t* choice;        // [B, T]
  int* accepted;          // [B]
  float* logprob;         // [B, T]
};

constexpr double kLn2 = 0.693147180559945309417232121458;
constexpr int kVfTable = 32;
// 2^(i / 32), from products of the square roots of 2 that the bits of i name; with
// i / 32 less in the exponent's place, so that adding 32 e + i there makes 2^e of it.
struct Exp2Table {
  uint64_t t[kVfTable];
  constexpr Exp2Table() : t() {
    double root[5] = {};
    double x = 2.;
    for (int b = 4; b >= 0; --b) {  // 2^(1/2), 2^(1/4), ..
      double y = x;
      for (int i = 0; i < 60; ++i) y = 0.5 * (y + x / y);
      root[b] = x = y;
    }
    for (int i = 0; i < kVfTable; ++i) {
      double v = 1.;
      for (int b = 0; b < 5; ++b)
        if (i >> b & 1) v *= root[b];
      t[i] = __builtin_bit_cast(uint64_t, v) - ((uint64_t)i << 47);
    }
  }
};
__device__ constexpr Exp2Table kExp2Table{};
__device__ __forceinline__ void vf_table(uint64_t* lds) {  // (then a barrier)
  if (threadIdx.x < kVfTable) lds[threadIdx.x] = kExp2Table.t[threadIdx.x];
}
constexpr double kVfRound = 1.5 * 140737488355328.;  // 2^47: sums with it are whole 32nds
// 2^(d + f), |f| <= 1/64, d the whole 32nds in the last bits of t, -1000 <= d + f <= 0
// or so; NaN where f is.
__device__ __forceinline__ double exp2_parts(double t, double f, const uint64_t* table) {
  constexpr double c1 = kLn2, c2 = c1 * kLn2 / 2, c3 = c2 * kLn2 / 3, c4 = c3 * kLn2 / 4;
  const uint32_t k = (uint32_t)__builtin_bit_cast(uint64_t, t);
  const u32x2 e = __builtin_bit_cast(u32x2, table[k & (kVfTable - 1)]);
  double p = __builtin_fma(c4, f, c3);
  p = __builtin_fma(p, f, c2);
  p = __builtin_fma(p, f, c1);
  p = __builtin_fma(p, f, 1.);
  return p * __builtin_bit_cast(double, u32x2{e[0], e[1] + (k << 15)});
}
__device__ __forceinline__ double exp2_64(double z, const uint64_t* table) {  // -1000 <= z <= 1, or NaN
  const double t = z + kVfRound;
  return exp2_parts(t, z - (t - kVfRound), table);
}

// DPP moves of eight bytes, sums over the wave and inclusive sums along its lanes.
template <int kCtrl, int kRowMask, int kBankMask>
__device__ __forceinline__ double dpp_d(double x) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = dpp_z<kCtrl, kRowMask, kBankMask>((uint32_t)b), hi = dpp_z<kCtrl, kRowMask, kBankMask>((uint32_t)(b >> 32));
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double read_lane_d(double x, int l) {
  const uint64_t b = __builtin_bit_cast(uint64_t, x);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)b, l), hi = (uint32_t)__builtin_amdgcn_readlane((int)(b >> 32), l);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum_d(double x) {
  x += dpp_d<kDppQuadSwap1, 0xf, 0xf>(x);
  x += dpp_d<kDppQuadSwap2, 0xf, 0xf>(x);
  x += dpp_d<kDppHalfMirror, 0xf, 0xf>(x);
  x += dpp_d<kDppMirror, 0xf, 0xf>(x);
  return (read_lane_d(x, 0) + read_lane_d(x, 16)) + (read_lane_d(x, 32) + read_lane_d(x, 48));
}
__device__ __forceinline__ double wave_scan_d(double x) {
  double t = x + dpp_d<kDppRowShr1, 0xf, 0xf>(x);
  t += dpp_d<kDppRowShr2, 0xf, 0xf>(x);
  t += dpp_d<kDppRowShr3, 0xf, 0xf>(x);
  t += dpp_d<kDppRowShr4, 0xf, 0xe>(t);
  t += dpp_d<kDppRowShr8, 0xf, 0xc>(t);
  t += dpp_d<kDppRowBcast15, 0xa, 0xf>(t);
  t += dpp_d<kDppRowBcast31, 0xc, 0xf>(t);
  return t;
}

// Elements j .. j + 16 / sizeof(T) - 1 of a row as floats, -inf from `hi` on.
template <typename T>
__device__ __forceinline__ void vf_load(const T* x, int j, int hi, float* v) {
  constexpr int EPV = 16 / (int)sizeof(T);
  struct __attribute__((packed, aligned(sizeof(T)))) Raw {
    T e[EPV];
  };
  if (j + EPV <= hi) {
    const Raw r = *reinterpret_cast<const Raw*>(x + j);
#pragma unroll
    for (int e = 0; e < EPV; ++e) v[e] = static_cast<float>(r.e[e]);
  } else {
#pragma unroll
    for (int e = 0; e < EPV; ++e) v[e] = j + e < hi ? static_cast<float>(x[j + e]) : -INFINITY;
  }
}

// e^((v - m) / temperature); 0 below 2^-1000.
__device__ __forceinline__ double vf_weight(float v, float m, double mul, const uint64_t* table) {
#pragma clang fp contract(off)
  const double z = ((double)v - (double)m) * mul, e = exp2_64(z, table);
  return z < -1000. ? 0. : e;
}

// A sum of weights against m, against the larger maximum `to` (both may be -inf, where
// nothing has been seen).
__device__ __forceinline__ double vf_turned(double s, float m, float to, double mul, const uint64_t* table) {
  return m == to ? s : s * vf_weight(m, to, mul, table);
}

// Maximum and sum of a segment of a row.
template <typename T>
__global__ void __launch_bounds__(kVfThreads) verify_stats_kernel(VerifyArgs a) {
  constexpr int EPV = 16 / (int)sizeof(T), NV = kVfElems / EPV;
  __shared__ float wm[kVfThreads / 64];
  __shared__ double ws[kVfThreads / 64];
  __shared__ uint64_t table[kVfTable];
  const int tid = threadIdx.x, sg = blockIdx.x % a.S, row = blockIdx.x / a.S;
  const T* x;
  if (row < a.B * a.T) {
    x = static_cast<const T*>(a.x) + (row / a.T) * a.x_sb + (row % a.T) * a.x_st;
  } else {
    const int r = row - a.B * a.T;
    x = static_cast<const T*>(a.y) + (r / (a.T - 1)) * a.y_sb + (r % (a.T - 1)) * a.y_st;
  }
  const int lo = sg * a.seg, hi = min(a.V, lo + a.seg);
  vf_table(table);
  __syncthreads();
  float m = -INFINITY;
  double s = 0.;
  for (int j0 = lo; j0 < hi; j0 += kVfTile) {
    float v[kVfElems];
#pragma unroll
    for (int q = 0; q < NV; ++q) vf_load<T>(x, j0 + (q * kVfThreads + tid) * EPV, hi, v + q * EPV);
    float top = v[0];
#pragma unroll
    for (int e = 1; e < kVfElems; ++e) top = fmaxf(top, v[e]);
    if (top > m) {
      s = vf_turned(s, m, top, a.mul, table);
      m = top;
    }
    if (m == -INFINITY) {  // nothing but -inf so far, or NaN
#pragma unroll
      for (int e = 0; e < kVfElems; ++e) s += v[e] == v[e] ? 0. : (double)v[e];
    } else if (fabs((double)m * a.mul) < 0x1p27) {
      // Against 2^R, R the whole 32nds next to m's exponent, so that a product's 32nds
      // and its rest (exact) take one operation each.  (2^-990 of the largest and below
      // are all 2^-990, which no sum notices: cheaper than a zero each.  A NaN stays
      // one.  In fp32 `least` is off by up to 2^-24 of m, 8 powers of two here; beyond,
      // it might be m itself.)
      const float least = m - a.deep;
      const double R = ((double)m * a.mul + kVfRound) - kVfRound, round = kVfRound - R;
      double sum = 0.;
#pragma unroll
      for (int e = 0; e < kVfElems; ++e) {
        const double x = __builtin_elementwise_maximum(v[e], least), t = __builtin_fma(x, a.mul, round);
        sum += exp2_parts(t, __builtin_fma(x, a.mul, round - t), table);
      }
      s += sum * exp2_64(__builtin_fma(-(double)m, a.mul, R), table);
    } else {
#pragma unroll 1
      for (int e = 0; e < kVfElems; ++e) s += vf_weight(v[e], m, a.mul, table);
    }
  }
  const float wave_m = wave_max_dpp(m);
  s = wave_sum_d(vf_turned(s, m, wave_m, a.mul, table));
  if ((tid & 63) == 0) {
    wm[tid >> 6] = wave_m;
    ws[tid >> 6] = s;
  }
  __syncthreads();
  if (tid == 0) {
    float all = wm[0];
    for (int w = 1; w < kVfThreads / 64; ++w) all = fmaxf(all, wm[w]);
    double sum = 0.;
    for (int w = 0; w < kVfThreads / 64; ++w) sum += vf_turned(ws[w], wm[w], all, a.mul, table);
    a.part[(int64_t)row * a.S + sg] = VfPart{sum, all, 0};
  }
}

// A row's maximum and sum from its segments, lane s segment s.
__device__ __forceinline__ void vf_join(const VerifyArgs& a, int64_t row, int lane, const uint64_t* table, float* m, double* s) {
  VfPart p{0., -INFINITY, 0};
  if (lane < a.S) p = a.part[row * a.S + lane];
  *m = wave_max_dpp(p.m);
  *s = wave_sum_d(vf_turned(p.s, p.m, *m, a.mul, table));
}

// Which nodes of sequence b stand: a wave of the workgroup (kVfWide threads) per node at
// a time.  With `write` the outputs of the nodes but the last that stands; returns
// (to every thread) what the sampling needs.
constexpr int kVfWide = 512;
struct VfWalk {
  double s[kTreeMaxT], qs[kTreeMaxT];
  float m[kTreeMaxT], qm[kTreeMaxT];
  int first;  // the first node that does not stand
};
template <typename T>
__device__ __forceinline__ VfSeq vf_walk(const VerifyArgs& a, int b, bool write, const uint64_t* table, VfWalk* sh) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t* tokens = a.tokens + (int64_t)b * a.T;
  if (tid == 0) sh->first = a.T;
  __syncthreads();
  for (int i = 1 + wave; i <= a.T; i += kVfWide / 64) {  // (node T: its parent's row alone)
    const int64_t token = i < a.T ? tokens[i] : -1;
    const bool real = token >= 0 && token < a.V;
    const int64_t at = real ? token : 0;
    const bool draft = a.y && i < a.T;
    const float x = static_cast<float>(static_cast<const T*>(a.x)[b * a.x_sb + (i - 1) * a.x_st + at]);
    const float u = a.u[(int64_t)b * a.T + min(i, a.T - 1)];
    float y = 0.f, m, qm = 0.f;
    if (draft) y = static_cast<float>(static_cast<const T*>(a.y)[b * a.y_sb + (i - 1) * a.y_st + at]);
    double s, qs = 1., q = 1.;
    vf_join(a, (int64_t)b * a.T + i - 1, lane, table, &m, &s);
    if (draft) {
      vf_join(a, (int64_t)a.B * a.T + (int64_t)b * (a.T - 1) + i - 1, lane, table, &qm, &qs);
      q = vf_weight(y, qm, a.mul, table) / qs;
    }
    const bool stands = real && (double)u * q < vf_weight(x, m, a.mul, table) / s;
    if (lane == 0) {
      sh->m[i - 1] = m;
      sh->s[i - 1] = s;
      sh->qm[i - 1] = qm;
      sh->qs[i - 1] = qs;
      if (!stands && i < a.T) atomicMin(&sh->first, i);
    }
    if (write && stands && lane == 0) {
      a.choice[(int64_t)b * a.T + i - 1] = token;
      a.logprob[(int64_t)b * a.T + i - 1] = (float)(((double)x - (double)m) * (a.mul * kLn2) - log(s));
    }
  }
  __syncthreads();
  const int last = sh->first - 1;
  const int64_t failed = last + 1 < a.T ? tokens[last + 1] : -1;
  if (write) {
    for (int i = last + 1 + tid; i < a.T; i += kVfWide) {
      a.choice[(int64_t)b * a.T + i] = -1;
      a.logprob[(int64_t)b * a.T + i] = 0.f;
    }
    if (tid == 0) a.accepted[b] = last + 1;
  }
  return VfSeq{1. / sh->s[last], 1. / sh->qs[last], sh->m[last], sh->qm[last], last, failed >= 0 && failed < a.V ? (int)failed : -1};
}

// Weights of N places from j on of the sampled row: of what is left of p, and of p.
// (Each operation rounded by itself, here and in vf_weight.  A difference of products by
// fma would leave the rounding of one of them, 2^-54 of p, on tokens that both models
// hold equally likely, and u_0 = 0 would draw the first of those.  And a piece that has a
// weight here for its sum has it again where its tokens are looked at one by one.)
template <typename T, int N>
__device__ __forceinline__ void vf_weights(const VerifyArgs& a, int b, const VfSeq& q, int j, int hi, const uint64_t* table,
                                           float* v, double* w, double* p) {
#pragma clang fp contract(off)
  constexpr int EPV = 16 / (int)sizeof(T);
  float z[N];
  const T* x = static_cast<const T*>(a.x) + b * a.x_sb + q.last * a.x_st;
  const T* y = static_cast<const T*>(a.y) + b * a.y_sb + q.last * a.y_st;
  const bool rest = q.token >= 0 && a.y;
  if (N == 1) {
    v[0] = j < hi ? static_cast<float>(x[j]) : -INFINITY;
    if (rest) z[0] = j < hi ? static_cast<float>(y[j]) : -INFINITY;
  } else {
#pragma unroll
    for (int i = 0; i < N; i += EPV) vf_load<T>(x, j + i, hi, v + i);
    if (rest)
#pragma unroll
      for (int i = 0; i < N; i += EPV) vf_load<T>(y, j + i, hi, z + i);
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    p[e] = vf_weight(v[e], q.p_m, a.mul, table) * q.p_mul;
    // (A difference that is NaN counts for nothing: with a draft row that is not
    // finite p itself is sampled.)
    w[e] = rest ? fmax(p[e] - vf_weight(z[e], q.q_m, a.mul, table) * q.q_mul, 0.) : j + e == q.token ? 0. : p[e];
  }
}

// Sums of both over piece `piece` of kVfPiece places, by a wave.
constexpr int kVfPiece = 512;
template <typename T>
__device__ __forceinline__ void vf_piece(const VerifyArgs& a, int b, const VfSeq& q, int piece, int lane,
                                         const uint64_t* table, bool across) {
  constexpr int N = kVfPiece / 64;
  float v[N];
  double w[N], p[N], sw = 0., sp = 0.;
  vf_weights<T, N>(a, b, q, piece * kVfPiece + lane * N, a.V, table, v, w, p);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    sw += w[e];
    sp += p[e];
  }
  sw = wave_sum_d(sw);
  sp = wave_sum_d(sp);
  double* to = a.sums + ((int64_t)b * a.pieces + piece) * 2 + lane;
  if (lane >= 2) return;
  if (across)
    st_dev(reinterpret_cast<uint64_t*>(to), __builtin_bit_cast(uint64_t, lane ? sp : sw));
  else
    *to = lane ? sp : sw;
}

// The workgroup's first thread with a weight that is past the target, and its last
// with a weight.
__device__ __forceinline__ void vf_mark(bool some, bool past, int lane, int wave, int* first, int* any) {
  const uint64_t has = __builtin_amdgcn_ballot_w64(some), hit = __builtin_amdgcn_ballot_w64(some && past);
  if (lane != 0) return;
  if (hit) atomicMin(first, 64 * wave + __builtin_ctzll(hit));
  if (has) atomicMax(any, 64 * wave + 63 - __builtin_clzll(has));
}

// The token: the piece whose running sum passes u_0 times the whole, and the place in
// it.  A thread holds one piece (of up to 262144 tokens), then one place.
static_assert(kVfPiece == kVfWide, "a thread each");
struct VfToken {
  double sum_w[kVfWide / 64], sum_p[kVfWide / 64], base;
  int first, any, piece;
};
template <typename T>
__device__ __forceinline__ void vf_token(const VerifyArgs& a, int b, const VfSeq& q, const uint64_t* table, VfToken* sh) {
  constexpr int W = kVfWide / 64;
  double *sum_w = sh->sum_w, *sum_p = sh->sum_p;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const double* sums = a.sums + (int64_t)b * a.pieces * 2;
  const int per = (a.pieces + kVfPiece - 1) / kVfPiece, p0 = tid * per, p1 = min(p0 + per, a.pieces);
  double sw = 0., sp = 0.;
  for (int i = p0; i < p1; ++i) {
    sw += sums[2 * i];
    sp += sums[2 * i + 1];
  }
  const double ln_s = -log(q.p_mul);
  if (tid == 0) {
    sh->first = kVfPiece;
    sh->any = -1;
  }
  double cw = wave_scan_d(sw), cp = wave_scan_d(sp);
  if (lane == 63) {
    sum_w[wave] = cw;
    sum_p[wave] = cp;
  }
  __syncthreads();
  double all_w = 0., all_p = 0.;
#pragma unroll
  for (int k = 0; k < W; ++k) {
    if (k == wave) {
      cw += all_w;
      cp += all_p;
    }
    all_w += sum_w[k];
    all_p += sum_p[k];
  }
  // (Where nothing is left of p, all of p.)
  const bool left = all_w > 0.;
  const double mine = left ? sw : sp, upto = left ? cw : cp, total = left ? all_w : all_p;
  if (!(total > 0.) || !(total < __builtin_inf())) {  // (a row that is not finite; every thread alike)
    if (tid == 0) {
      a.choice[(int64_t)b * a.T + q.last] = -1;
      a.logprob[(int64_t)b * a.T + q.last] = __builtin_nanf("");
    }
    return;
  }
  const double target = (double)a.u[(int64_t)b * a.T] * total;
  // The first thread past the target, else the last one with any weight.
  vf_mark(mine > 0., upto > target, lane, wave, &sh->first, &sh->any);
  __syncthreads();
  if (tid == (sh->first < kVfPiece ? sh->first : sh->any)) {
    double run = upto - mine, base = run;
    int at = p0;  // the first of its pieces past the target, else its last with any weight
    for (int i = p0; i < p1 && per > 1; ++i) {
      const double x = left ? sums[2 * i] : sums[2 * i + 1];
      if (x > 0.) {
        at = i;
        base = run;
        if (run + x > target) break;
      }
      run += x;
    }
    sh->piece = at;
    sh->base = base;
  }
  __syncthreads();
  if (tid == 0) {
    sh->first = kVfPiece;
    sh->any = -1;
  }
  const int j = sh->piece * kVfPiece + tid;
  float x;
  double w, p;
  vf_weights<T, 1>(a, b, q, j, a.V, table, &x, &w, &p);
  w = left ? w : p;
  double run = wave_scan_d(w);
  if (lane == 63) sum_w[wave] = run;
  __syncthreads();
  run += sh->base;
  for (int k = 0; k < wave; ++k) run += sum_w[k];
  vf_mark(w > 0., run > target, lane, wave, &sh->first, &sh->any);
  __syncthreads();
  if (tid == (sh->first < kVfPiece ? sh->first : sh->any)) {
    a.choice[(int64_t)b * a.T + q.last] = j;
    a.logprob[(int64_t)b * a.T + q.last] = (float)(((double)x - (double)q.p_m) * (a.mul * kLn2) - ln_s);
  }
}

// The walk, the sums and the token by a kernel each.
template <typename T>
__global__ void __launch_bounds__(kVfWide) verify_walk_kernel(VerifyArgs a) {
  __shared__ uint64_t table[kVfTable];
  __shared__ VfWalk walk;
  vf_table(table);
  const VfSeq q = vf_walk<T>(a, blockIdx.x, true, table, &walk);
  if (threadIdx.x == 0) a.seq[blockIdx.x] = q;
}
template <typename T>
__global__ void __launch_bounds__(kVfWide) verify_sums_kernel(VerifyArgs a) {
  __shared__ uint64_t table[kVfTable];
  const int b = blockIdx.x / a.groups, piece = (blockIdx.x % a.groups) * (kVfWide / 64) + (threadIdx.x >> 6);
  vf_table(table);
  __syncthreads();
  if (piece < a.pieces) vf_piece<T>(a, b, a.seq[b], piece, threadIdx.x & 63, table, false);
}
template <typename T>
__global__ void __launch_bounds__(kVfWide) verify_token_kernel(VerifyArgs a) {
  __shared__ uint64_t table[kVfTable];
  __shared__ VfToken token;
  vf_table(table);
  vf_token<T>(a, blockIdx.x, a.seq[blockIdx.x], table, &token);
}

// The three in one, for short chains: each workgroup of a sequence makes the walk for
// itself, and the last one to arrive draws the token (its counter is zero before the
// call and wraps to zero).  8 nodes of one sequence: 8.1 us where the three kernels take
// 12 and their gaps, of which 3.8 are a kernel that does nothing, 1.5 the walk and the
// sums and 2.8 the token, each step a round trip of memory; 8 sequences of 9: 12.7.
template <typename T>
__global__ void __launch_bounds__(kVfWide) verify_rest_kernel(VerifyArgs a) {
  __shared__ uint64_t table[kVfTable];
  __shared__ VfWalk walk;
  __shared__ VfToken token;
  __shared__ int last;
  const int b = blockIdx.x / a.groups, group = blockIdx.x % a.groups, piece = group * (kVfWide / 64) + (threadIdx.x >> 6);
  vf_table(table);
  const VfSeq q = vf_walk<T>(a, b, group == 0, table, &walk);
  if (piece < a.pieces) vf_piece<T>(a, b, q, piece, threadIdx.x & 63, table, true);
  // (Every wave's sums are out first.)
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicInc(a.arrived + b * a.arrived_s, (uint32_t)a.groups - 1u) == (uint32_t)a.groups - 1u;
    if (last) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  }
  __syncthreads();
  if (last) vf_token<T>(a, b, q, table, &token);
}

// Workgroups of a call: enough to fill the GPU where a row can be cut.
constexpr int64_t kVfGroups = 2048;
// Nodes up to which every workgroup of a sequence walks for itself (two a wave).
constexpr int kVfShort = 16;

struct VerifyPlan {
  int S, seg;
  size_t bytes;
};
static VerifyPlan verify_plan(int64_t B, int64_t T, int64_t V, bool draft) {
  const int64_t rows = B * (draft ? 2 * T - 1 : T), tiles = (V + kVfTile - 1) / kVfTile;
  const int64_t want = std::min<int64_t>({tiles, kVfMaxSegs, std::max<int64_t>(1, kVfGroups / rows)});
  const int64_t per = (tiles + want - 1) / want;
  VerifyPlan p;
  p.S = (int)((tiles + per - 1) / per);
  p.seg = (int)std::min<int64_t>(per * kVfTile, INT32_MAX - kVfTile);
  p.bytes = kSyncBytes + 256 + (size_t)rows * p.S * sizeof(VfPart) +
            (size_t)B * (sizeof(VfSeq) + (size_t)((V + kVfPiece - 1) / kVfPiece) * 16);
  return p;
}
size_t verify_workspace_bytes(int64_t B, int64_t T, int64_t V, bool draft) { return verify_plan(B, T, V, draft).bytes; }

template <typename T>
static hipError_t launch_verify_t(const VerifyArgs& a, hipStream_t st) {
  const int rows = a.B * (a.y ? 2 * a.T - 1 : a.T);
  launch(verify_stats_kernel<T>, dim3((unsigned)(rows * a.S)), dim3(kVfThreads), 0, st, a);
  if (a.T <= kVfShort && a.arrived) {
    launch(verify_rest_kernel<T>, dim3((unsigned)(a.B * a.groups)), dim3(kVfWide), 0, st, a);
  } else {
    launch(verify_walk_kernel<T>, dim3(a.B), dim3(kVfWide), 0, st, a);
    launch(verify_sums_kernel<T>, dim3((unsigned)(a.B * a.groups)), dim3(kVfWide), 0, st, a);
    launch(verify_token_kernel<T>, dim3(a.B), dim3(kVfWide), 0, st, a);
  }
  return hipGetLastError();
}

hipError_t launch_verify_drafts(const dropkv_verify_drafts_args& p, hipStream_t st) {
  const VerifyPlan pl = verify_plan(p.B, p.T, p.V, p.draft_logits != nullptr);
  VerifyArgs a{};
  a.x = p.logits;
  a.x_sb = p.x_s[0];
  a.x_st = p.x_s[1];
  a.y = p.T > 1 ? p.draft_logits : nullptr;
  a.y_sb = p.y_s[0];
  a.y_st = p.y_s[1];
  a.tokens = p.tokens;
  a.u = p.uniforms;
  a.B = (int)p.B;
  a.T = (int)p.T;
  a.V = (int)p.V;
  a.S = pl.S;
  a.seg = pl.seg;
  a.pieces = (int)((p.V + kVfPiece - 1) / kVfPiece);
  a.groups = (a.pieces + kVfWide / 64 - 1) / (kVfWide / 64);
  a.mul = 1.4426950408889634074 / p.temperature;
  a.deep = (float)(990. / a.mul);
  a.arrived = sync_counters(p.workspace, p.B, &a.arrived_s);
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p.workspace) + 15) & ~(uintptr_t)15) + kSyncBytes;
  a.part = reinterpret_cast<VfPart*>(ws);
  a.seq = reinterpret_cast<VfSeq*>(a.part + (size_t)p.B * (p.draft_logits ? 2 * p.T - 1 : p.T) * pl.S);
  a.sums = reinterpret_cast<double*>(a.seq + p.B);
  a.choice = p.choice;
  a.accepted = p.accepted;
  a.logprob = p.logprobs;
  if (p.dtype == kDtypeFp32) return launch_verify_t<float>(a, st);
  if (p.dtype == kDtypeBf16) return launch_verify_t<__bf16>(a, st);
  return launch_verify_t<_Float16>(a, st);
}

}  // namespace dkv
