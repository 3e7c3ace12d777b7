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
// difference of near values, so all weights and sums are in 64 bits: sums of two
// orders differ by 10^-15, which moves a border past a given u_0 about once in 10^10
// samples of a vocabulary of 150,000.  The exponential is 2^k times the Taylor sum
// of 2^f, |f| <= 1/2, to the 11th power (2^-52 of it is left).
//
// Four kernels: maximum and sum of every row in segments; the walk, a workgroup per
// sequence; sums of the weights that are sampled, in segments of the one row of each
// sequence; and the token.
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
  double mul;             // log2 e / temperature
  VfPart* part;           // [B, T, S], then [B, T - 1, S] of the drafts
  VfSeq* seq;             // [B]
  double* sums;           // [B, S, 2]: of the weights, and of p alone
  int64_t* choice;        // [B, T]
  int* accepted;          // [B]
  float* logprob;         // [B, T]
};

constexpr double kLn2 = 0.693147180559945309417232121458;
struct Exp2Taylor {
  double c[12];
  constexpr Exp2Taylor() : c() {
    c[0] = 1;
    for (int i = 1; i < 12; ++i) c[i] = c[i - 1] * kLn2 / i;
  }
};
__device__ __forceinline__ double exp2_64(double z) {  // z <= 0, or NaN
  constexpr Exp2Taylor t{};
  const double k = __builtin_rint(z), f = z - k;
  double p = t.c[11];
#pragma unroll
  for (int i = 10; i >= 0; --i) p = __builtin_fma(p, f, t.c[i]);
  return z < -1000. ? 0. : __builtin_ldexp(p, (int)k);
}

// Eight bytes from another lane.
__device__ __forceinline__ double shfl_xor_d(double x, int o) { return __shfl_xor(x, o); }
__device__ __forceinline__ double wave_sum_d(double x) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) x += shfl_xor_d(x, o);
  return x;
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

__device__ __forceinline__ double vf_weight(float v, float m, double mul) { return exp2_64(((double)v - (double)m) * mul); }

// Maximum and sum of a segment of a row.
template <typename T>
__global__ void __launch_bounds__(kVfThreads) verify_stats_kernel(VerifyArgs a) {
  constexpr int EPV = 16 / (int)sizeof(T), NV = kVfElems / EPV;
  __shared__ float wm[kVfThreads / 64];
  __shared__ double ws[kVfThreads / 64];
  const int tid = threadIdx.x, sg = blockIdx.x % a.S, row = blockIdx.x / a.S;
  const T* x;
  if (row < a.B * a.T) {
    x = static_cast<const T*>(a.x) + (row / a.T) * a.x_sb + (row % a.T) * a.x_st;
  } else {
    const int r = row - a.B * a.T;
    x = static_cast<const T*>(a.y) + (r / (a.T - 1)) * a.y_sb + (r % (a.T - 1)) * a.y_st;
  }
  const int lo = sg * a.seg, hi = min(a.V, lo + a.seg);
  float m = -__FLT_MAX__;  // (finite, so that -inf gets no weight)
  double s = 0.;
  for (int j0 = lo; j0 < hi; j0 += kVfTile) {
    float v[kVfElems];
#pragma unroll
    for (int q = 0; q < NV; ++q) vf_load<T>(x, j0 + (q * kVfThreads + tid) * EPV, hi, v + q * EPV);
    float top = v[0];
#pragma unroll
    for (int e = 1; e < kVfElems; ++e) top = fmaxf(top, v[e]);
    if (top > m) {
      s *= vf_weight(m, top, a.mul);
      m = top;
    }
#pragma unroll
    for (int e = 0; e < kVfElems; ++e) s += vf_weight(v[e], m, a.mul);
  }
  const float wave_m = wave_max_dpp(m);
  s = wave_sum_d(s * vf_weight(m, wave_m, a.mul));
  if ((tid & 63) == 0) {
    wm[tid >> 6] = wave_m;
    ws[tid >> 6] = s;
  }
  __syncthreads();
  if (tid == 0) {
    float all = wm[0];
    for (int w = 1; w < kVfThreads / 64; ++w) all = fmaxf(all, wm[w]);
    double sum = 0.;
    for (int w = 0; w < kVfThreads / 64; ++w) sum += ws[w] * vf_weight(wm[w], all, a.mul);
    a.part[(int64_t)row * a.S + sg] = VfPart{sum, all, 0};
  }
}

// A row's maximum and sum from its segments, lane s segment s.
__device__ __forceinline__ void vf_join(const VerifyArgs& a, int64_t row, int lane, float* m, double* s) {
  VfPart p{0., -__FLT_MAX__, 0};
  if (lane < a.S) p = a.part[row * a.S + lane];
  *m = wave_max_dpp(p.m);
  *s = wave_sum_d(p.s * vf_weight(p.m, *m, a.mul));
}

// One workgroup per sequence, a wave per node at a time: which nodes stand.
template <typename T>
__global__ void __launch_bounds__(512) verify_walk_kernel(VerifyArgs a) {
  __shared__ int first;  // the first node that does not stand
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t* tokens = a.tokens + (int64_t)b * a.T;
  if (tid == 0) first = a.T;
  __syncthreads();
  for (int i = 1 + wave; i < a.T; i += 8) {
    const int64_t token = tokens[i];
    bool stands = false;
    float lp = 0.f;
    if (token >= 0 && token < a.V) {
      float m, qm;
      double s, qs;
      vf_join(a, (int64_t)b * a.T + i - 1, lane, &m, &s);
      const float x = static_cast<float>(static_cast<const T*>(a.x)[b * a.x_sb + (i - 1) * a.x_st + token]);
      double q = 1.;
      if (a.y) {
        vf_join(a, (int64_t)a.B * a.T + (int64_t)b * (a.T - 1) + i - 1, lane, &qm, &qs);
        q = vf_weight(static_cast<float>(static_cast<const T*>(a.y)[b * a.y_sb + (i - 1) * a.y_st + token]), qm, a.mul) / qs;
      }
      stands = (double)a.u[(int64_t)b * a.T + i] * q < vf_weight(x, m, a.mul) / s;
      lp = (float)(((double)x - (double)m) * (a.mul * kLn2) - log(s));
    }
    if (lane == 0) {
      if (!stands) atomicMin(&first, i);
      // (Places past the node that is sampled are put right below.)
      a.choice[(int64_t)b * a.T + i - 1] = token;
      a.logprob[(int64_t)b * a.T + i - 1] = lp;
    }
  }
  __syncthreads();
  const int last = first - 1;
  for (int i = last + tid; i < a.T; i += 512) {
    a.choice[(int64_t)b * a.T + i] = -1;
    a.logprob[(int64_t)b * a.T + i] = 0.f;
  }
  if (wave != 0) return;
  float m, qm = 0.f;
  double s, qs = 1.;
  vf_join(a, (int64_t)b * a.T + last, lane, &m, &s);
  const int64_t failed = last + 1 < a.T ? tokens[last + 1] : -1;
  const bool real = failed >= 0 && failed < a.V;
  if (real && a.y) vf_join(a, (int64_t)a.B * a.T + (int64_t)b * (a.T - 1) + last, lane, &qm, &qs);
  if (lane == 0) {
    a.accepted[b] = last + 1;
    a.seq[b] = VfSeq{1. / s, 1. / qs, m, qm, last, real ? (int)failed : -1};
  }
}

// Weight of place j of the sampled row: of what is left of p, and of p.
template <typename T, int N>
__device__ __forceinline__ void vf_weights(const VerifyArgs& a, int b, const VfSeq& q, int j, int hi, double* w, double* p) {
  float v[N], z[N];
  const T* x = static_cast<const T*>(a.x) + b * a.x_sb + q.last * a.x_st;
  vf_load<T>(x, j, hi, v);
  const bool rest = q.token >= 0 && a.y;
  if (rest) vf_load<T>(static_cast<const T*>(a.y) + b * a.y_sb + q.last * a.y_st, j, hi, z);
#pragma unroll
  for (int e = 0; e < N; ++e) {
    p[e] = vf_weight(v[e], q.p_m, a.mul) * q.p_mul;
    // (A difference that is NaN counts for nothing: with a draft row that is not
    // finite p itself is sampled.)
    w[e] = rest ? fmax(p[e] - vf_weight(z[e], q.q_m, a.mul) * q.q_mul, 0.) : j + e == q.token ? 0. : p[e];
  }
}

template <typename T>
__global__ void __launch_bounds__(kVfThreads) verify_sums_kernel(VerifyArgs a) {
  constexpr int EPV = 16 / (int)sizeof(T);
  __shared__ double sum[2][kVfThreads / 64];
  const int tid = threadIdx.x, sg = blockIdx.x % a.S, b = blockIdx.x / a.S;
  const VfSeq q = a.seq[b];
  const int lo = sg * a.seg, hi = min(a.V, lo + a.seg);
  double sw = 0., sp = 0.;
  for (int j = lo + tid * EPV; j < hi; j += kVfThreads * EPV) {
    double w[EPV], p[EPV];
    vf_weights<T, EPV>(a, b, q, j, hi, w, p);
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      sw += w[e];
      sp += p[e];
    }
  }
  sw = wave_sum_d(sw);
  sp = wave_sum_d(sp);
  if ((tid & 63) == 0) {
    sum[0][tid >> 6] = sw;
    sum[1][tid >> 6] = sp;
  }
  __syncthreads();
  if (tid < 2) a.sums[((int64_t)b * a.S + sg) * 2 + tid] = (sum[tid][0] + sum[tid][1]) + (sum[tid][2] + sum[tid][3]);
}

// Inclusive sums along the lanes.
__device__ __forceinline__ double wave_scan_d(double x, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const double y = __shfl_up(x, o);
    if (lane >= o) x += y;
  }
  return x;
}

// The token: the segment whose running sum passes u_0 times the whole, and the
// place in it.
template <typename T>
__global__ void __launch_bounds__(kVfThreads) verify_token_kernel(VerifyArgs a) {
  constexpr int EPV = 16 / (int)sizeof(T), W = kVfThreads / 64;
  __shared__ double wsum[W];
  __shared__ int hit, any;
  const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const VfSeq q = a.seq[b];
  const double* sums = a.sums + (int64_t)b * a.S * 2;
  double sw = lane < a.S ? sums[2 * lane] : 0., sp = lane < a.S ? sums[2 * lane + 1] : 0.;
  // (Where nothing is left of p, all of p.)
  const bool left = wave_sum_d(sw) > 0.;
  const double mine = left ? sw : sp, upto = wave_scan_d(mine, lane), total = __shfl(upto, 63);
  if (tid == 0) {
    hit = a.V;
    any = -1;
  }
  __syncthreads();
  if (!(total > 0.) || !(total < __builtin_inf())) {  // (a row that is not finite; every wave alike)
    if (tid == 0) {
      a.choice[(int64_t)b * a.T + q.last] = -1;
      a.logprob[(int64_t)b * a.T + q.last] = __builtin_nanf("");
    }
    return;
  }
  const double target = (double)a.u[(int64_t)b * a.T] * total;
  // The first segment past the target, else the last one with any weight.
  const uint64_t past = __builtin_amdgcn_ballot_w64(mine > 0. && upto > target), some = __builtin_amdgcn_ballot_w64(mine > 0.);
  const int sg = past ? __builtin_ctzll(past) : 63 - __builtin_clzll(some);
  double base = __shfl(upto - mine, sg);
  const int lo = sg * a.seg, hi = min(a.V, lo + a.seg);
  for (int j0 = lo; j0 < hi; j0 += kVfThreads * EPV) {
    const int j = j0 + tid * EPV;
    double w[EPV], p[EPV], own = 0.;
    vf_weights<T, EPV>(a, b, q, j, hi, w, p);
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      w[e] = left ? w[e] : p[e];
      own += w[e];
    }
    const double incl = wave_scan_d(own, lane);
    if (lane == 63) wsum[wave] = incl;
    __syncthreads();
    double run = base + (incl - own);
    for (int k = 0; k < wave; ++k) run += wsum[k];
    int at = a.V, most = -1;
#pragma unroll
    for (int e = 0; e < EPV; ++e) {
      run += w[e];
      if (w[e] > 0.) {
        most = j + e;
        if (run > target && at == a.V) at = j + e;
      }
    }
    if (at < a.V) atomicMin(&hit, at);
    if (most >= 0) atomicMax(&any, most);
    for (int k = 0; k < W; ++k) base += wsum[k];
    __syncthreads();
    if (hit < a.V) break;
  }
  if (tid == 0) {
    const int token = hit < a.V ? hit : any;
    const float x = static_cast<float>(static_cast<const T*>(a.x)[b * a.x_sb + q.last * a.x_st + token]);
    a.choice[(int64_t)b * a.T + q.last] = token;
    a.logprob[(int64_t)b * a.T + q.last] = (float)(((double)x - (double)q.p_m) * (a.mul * kLn2) + log(q.p_mul));
  }
}

// Workgroups of a call: enough to fill the GPU where a row can be cut.
constexpr int64_t kVfGroups = 2048;

struct VerifyPlan {
  int S, seg;
  size_t bytes;
};
static VerifyPlan verify_plan(int64_t B, int64_t T, int64_t V, bool draft) {
  const int64_t rows = B * (draft ? 2 * T - 1 : T), tiles = (V + kVfTile - 1) / kVfTile;
  // (The sampled rows, one a sequence, are cut alike.)
  const int64_t want = std::min<int64_t>({tiles, kVfMaxSegs, std::max<int64_t>({1, kVfGroups / rows, 512 / B})});
  const int64_t per = (tiles + want - 1) / want;
  VerifyPlan p;
  p.S = (int)((tiles + per - 1) / per);
  p.seg = (int)std::min<int64_t>(per * kVfTile, INT32_MAX - kVfTile);
  p.bytes = kSyncBytes + 256 + (size_t)rows * p.S * sizeof(VfPart) + (size_t)B * (sizeof(VfSeq) + p.S * 16);
  return p;
}
size_t verify_workspace_bytes(int64_t B, int64_t T, int64_t V, bool draft) { return verify_plan(B, T, V, draft).bytes; }

template <typename T>
static hipError_t launch_verify_t(const VerifyArgs& a, hipStream_t st) {
  const int rows = a.B * (a.y ? 2 * a.T - 1 : a.T);
  launch(verify_stats_kernel<T>, dim3((unsigned)(rows * a.S)), dim3(kVfThreads), 0, st, a);
  launch(verify_walk_kernel<T>, dim3(a.B), dim3(512), 0, st, a);
  launch(verify_sums_kernel<T>, dim3((unsigned)(a.B * a.S)), dim3(kVfThreads), 0, st, a);
  launch(verify_token_kernel<T>, dim3(a.B), dim3(kVfThreads), 0, st, a);
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
  a.mul = 1.4426950408889634074 / p.temperature;
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
