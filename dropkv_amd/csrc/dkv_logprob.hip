// What a row of logits x[0..V) says: the log probability of a given token, the
// entropy, and the `top` most probable tokens.
//   m = max x,  s = sum e^(x-m),  u = sum e^(x-m) (x-m)
//   log p_i = x_i - m - ln s,  H = -sum p_i ln p_i = ln s - u / s
// in one pass over the row, with the running maximum; u is taken against the
// maximum and not against zero, so that H does not come from the difference of
// two large numbers.  Rows are cut into segments where there are few of them;
// they are joined by the workgroup that finishes a row last, or by a second
// kernel.  Bound by memory: 2047 rows of 151936 bf16 (622 MB) take 111 us (5.6
// TB/s), 115 with the best token and 144 with the 20 best, one call after the
// other; 216 rows 17, 20 and 26; one row 7, 9 and 12 in a graph, which is three
// dependent round trips or more.  The sums are fp32, and a thread adds its V / 256
// terms one after the other: 2047 rows come out within 1.9e-7 (relative) of 64 bits
// where PyTorch's sums, added in pairs, are within 7e-8.
//
// The `top` largest.  A value and its place make one 64-bit key (value above,
// the complement of the place below): keys are all different, larger means more
// probable, ties go to the lowest place.  The pass leaves the maximum of each
// block of 16 vectors (128 elements, or 64 of fp32).  The `top` best elements
// lie in the `top` best blocks by (maximum, lowest place): for any element of
// another block, each of those holds one that comes before it.  Then the
// blocks are picked, read again (1 to 2 in a hundred of the row), and the elements
// picked.  (Keeping a list of candidates within the pass took 263 us for 20 of
// 2047 x 151936.)  For the one largest the pass itself keeps each thread's
// maximum and its tile, and the threads that hold the workgroup's look into that
// tile again.
#include "dkv_common.h"
#include "dkv_internal.h"
#include "dkv_select_dev.h"

#include <algorithm>

namespace dkv {

constexpr int kLpThreads = 256;
constexpr int kLpElems = 16;                        // elements per thread and tile
constexpr int kLpTile = kLpThreads * kLpElems;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxSegs = 64;  // a lane each where they are joined
template <typename T>
constexpr int kLpBlock = 16 * 16 / (int)sizeof(T);  // elements: a row of 16 lanes' vectors
// The selection takes kLpItems items a thread at a time, and those kept so far.
constexpr int kLpItems = 8;
// Its list: what a threshold that `top` of 64 groups (of four threads) reach
// leaves at most, `top` whole groups.
constexpr int kLpCap = kLpMaxTop * 4 * (kLpItems + 1);
constexpr int kLpPer = (kLpCap + kLpThreads - 1) / kLpThreads;

struct LogprobArgs {
  const void* x;
  int64_t sx;  // elements between rows
  const int64_t* tokens;
  int64_t N;
  int V, top, S, seg;  // segments per row, elements per segment (whole tiles)
  int one;             // the row's last workgroup joins its segments (else a second kernel)
  float* part;         // [N, S, 3]: m, s, u
  uint32_t* blocks;    // [N, nb]: block maxima as ordered keys (top > 1)
  int nb;
  uint64_t* best;      // [N, S]: the segments' best keys (top 1)
  uint32_t* arrived;   // [N]: segments done (S > 1)
  float* logprob;
  float* entropy;
  float* top_lp;
  int64_t* top_id;
};

struct Stat {
  float m, s, u;
};
// (m, s, u) against the larger maximum M; a part without weight adds nothing.
__device__ __forceinline__ void stat_to(Stat& a, float M) {
  const float d = a.m - M, f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
  a.u = (f == 0.f || a.s == 0.f) ? 0.f * f : f * fmaf(d, a.s, a.u);
  a.s *= f;
  a.m = M;
}

// (-0 and 0 are equals: float_key sees to it.)
__device__ __forceinline__ uint32_t lp_order(float x) { return x != x ? 0xffffffffu : float_key(x); }
__device__ __forceinline__ uint64_t lp_key(uint32_t order, int i) {  // NaN above all, as in torch's topk
  return ((uint64_t)order << 32) | (0xffffffffu - (uint32_t)i);
}

__device__ __forceinline__ uint64_t shfl_xor64(uint64_t x, int o) {
  return ((uint64_t)(uint32_t)__shfl_xor((int)(x >> 32), o) << 32) | (uint32_t)__shfl_xor((int)x, o);
}

// The results of a row from its statistics and its top keys (one wave, key i on
// lane i).  x - lse is taken as (x - m) - ln s, which rounds less.
template <typename T>
__device__ __forceinline__ void lp_write(const LogprobArgs& a, int64_t row, Stat st, int lane, uint64_t key) {
  const float ln_s = logf(st.s);
  if (lane == 0) {
    a.entropy[row] = ln_s - st.u / st.s;
    if (a.tokens) {
      const int64_t t = a.tokens[row];
      a.logprob[row] = t < 0 ? 0.f : t >= a.V ? __builtin_nanf("") : (static_cast<float>(static_cast<const T*>(a.x)[row * a.sx + t]) - st.m) - ln_s;
    }
  }
  if (lane < a.top) {
    a.top_lp[row * a.top + lane] = (key_float((uint32_t)(key >> 32)) - st.m) - ln_s;
    a.top_id[row * a.top + lane] = 0xffffffffu - (uint32_t)key;
  }
}

struct LpList {
  uint64_t list[kLpCap];
  uint64_t group[64];
  int count;
};

// One less than the k-th largest of a wave's keys (all different, or 0: none), 0
// where there are fewer: its order two bits at a time, by counts of the lanes
// above, then among equals its place, unless all of them are among the k.  (The
// last 12 bits of a 2-byte type's order follow from the others.)
template <typename T>
__device__ __forceinline__ uint64_t lp_below_kth(uint64_t key, int k) {
  constexpr int kLow = sizeof(T) == 2 ? 12 : 0;
  const uint32_t hi = (uint32_t)(key >> 32);
  auto reach = [&](uint32_t x, uint32_t t) { return __builtin_popcountll(__builtin_amdgcn_ballot_w64(x >= t)) >= k; };
  uint32_t t = 0, u = 0;
#pragma unroll
  for (int b = 30; b >= kLow; b -= 2)
    t += (uint32_t)(reach(hi, t + (1u << b)) + reach(hi, t + (2u << b)) + reach(hi, t + (3u << b))) << b;
  if (t == 0) return 0;
  if (__builtin_popcountll(__builtin_amdgcn_ballot_w64(hi >= t)) > k) {
    const bool above = (hi >> kLow) > (t >> kLow), tie = (hi >> kLow) == (t >> kLow);
    t = (uint32_t)__builtin_amdgcn_readlane((int)hi, __builtin_ctzll(__builtin_amdgcn_ballot_w64(tie)));
    const uint32_t lo = above ? 0xffffffffu : tie ? (uint32_t)key : 0;
#pragma unroll 1
    for (int b = 30; b >= 0; b -= 2)
      u += (uint32_t)(reach(lo, u + (1u << b)) + reach(lo, u + (2u << b)) + reach(lo, u + (3u << b))) << b;
  }
  return (((uint64_t)t << 32) | u) - 1;
}

// The list's k largest of its `count` keys to list[0 .. k), falling (0: none);
// the whole workgroup, from a barrier to a barrier.
__device__ __forceinline__ void lp_rank(int k, LpList* s) {
  const int tid = threadIdx.x, c = s->count;
  uint64_t mykey[kLpPer];
  int place[kLpPer];
#pragma unroll
  for (int q = 0; q < kLpPer; ++q) {
    const int i = tid + q * kLpThreads;
    place[q] = k;
    mykey[q] = 0;
    if (q * kLpThreads < c && i < c) {
      mykey[q] = s->list[i];
      int r = 0;
      for (int j = 0; j < c; ++j) r += s->list[j] > mykey[q];
      place[q] = r;
    }
  }
  __syncthreads();
  if (tid >= c && tid < k) s->list[tid] = 0;
#pragma unroll
  for (int q = 0; q < kLpPer; ++q)
    if (place[q] < k) s->list[place[q]] = mykey[q];
  __syncthreads();
}

// The k largest of item(0) .. item(n - 1) (keys, or 0: none), in falling order in
// list[0 .. k); the whole workgroup.  kLpItems items a thread at a time: a
// threshold that k of them reach (the k-th largest of 64 groups' maxima), the few
// above it into the list, and the list in order by each item's rank in it.
template <typename T, typename F>
__device__ __forceinline__ void lp_select(F&& item, int n, int k, LpList* s) {
  const int tid = threadIdx.x, lane = tid & 63;
#pragma unroll 1
  for (int base = 0; base < n; base += kLpItems * kLpThreads) {
    uint64_t key[kLpItems + 1], most = 0;
#pragma unroll
    for (int q = 0; q < kLpItems; ++q) key[q] = item(base + q * kLpThreads + tid);
    key[kLpItems] = base > 0 && tid < k ? s->list[tid] : 0;
#pragma unroll
    for (int q = 0; q <= kLpItems; ++q) most = max(most, key[q]);
    most = max(most, shfl_xor64(most, 1));
    most = max(most, shfl_xor64(most, 2));
    if ((lane & 3) == 0) s->group[tid >> 2] = most;
    if (tid == 0) s->count = 0;
    __syncthreads();
    // (Where fewer than k groups hold anything, everything passes.)
    const uint64_t t = lp_below_kth<T>(s->group[lane], k);
#pragma unroll
    for (int q = 0; q <= kLpItems; ++q)
      if (key[q] > t) s->list[atomicAdd(&s->count, 1)] = key[q];
    __syncthreads();
    lp_rank(k, s);
  }
}

// Elements j .. j + 15 / sizeof(T) of x, -inf from `hi` on.
template <typename T>
__device__ __forceinline__ void lp_load(const T* x, int j, int hi, float* v) {
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

// A row's results: its segments joined, its best blocks and their best elements.
template <typename T, int kMode>
__device__ __forceinline__ void lp_finish(const LogprobArgs& a, int64_t row, LpList* s, int* chosen) {
  constexpr int kBlock = kLpBlock<T>, EPV = 16 / (int)sizeof(T);
  const int tid = threadIdx.x, lane = tid & 63;
  Stat st{-__FLT_MAX__, 0.f, 0.f};
  uint64_t key = 0;
  if (lane < a.S) {
    const int64_t p = row * a.S + lane;
    st = Stat{a.part[3 * p], a.part[3 * p + 1], a.part[3 * p + 2]};
    if (kMode == 1) key = a.best[p];
  }
  if (kMode == 2) {
    const int nb = a.nb, kb = min(a.top, nb);
    const uint32_t* blocks = a.blocks + row * nb;
    lp_select<T>(
        [&](int i) {
          const uint64_t k = lp_key(blocks[min(i, nb - 1)], i);
          return i < nb ? k : 0;
        },
        nb, kb, s);
    if (tid < kb) chosen[tid] = (int)(0xffffffffu - (uint32_t)s->list[tid]);
    const uint32_t least = kb < a.top ? 0 : (uint32_t)(s->list[kb - 1] >> 32);
    if (tid == 0) s->count = 0;
    __syncthreads();
    // Each of the `top` blocks holds a value of at least the last one's maximum: so
    // do the `top` values.
    const T* x = static_cast<const T*>(a.x) + row * a.sx;
    constexpr int kVecs = kLpMaxTop * 16 / kLpThreads;
    float v[kVecs][EPV];
    int at[kVecs];
#pragma unroll
    for (int q = 0; q < kVecs; ++q) {
      const int i = tid + q * kLpThreads;
      at[q] = chosen[min(i / 16, kb - 1)] * kBlock + i % 16 * EPV;
      lp_load<T>(x, at[q], i < 16 * kb ? a.V : 0, v[q]);
    }
#pragma unroll
    for (int q = 0; q < kVecs; ++q)
#pragma unroll
      for (int e = 0; e < EPV; ++e) {
        const uint32_t o = lp_order(v[q][e]);
        if (o >= least && at[q] + e < a.V && tid + q * kLpThreads < 16 * kb) {
          const int p = atomicAdd(&s->count, 1);
          if (p < kLpThreads) s->list[p] = lp_key(o, at[q] + e);
        }
      }
    __syncthreads();
    if (s->count <= kLpThreads) {
      lp_rank(a.top, s);
    } else {  // (many equals, or few blocks)
      __syncthreads();
      const int n = kb * kBlock;
      lp_select<T>(
          [&](int i) {
            const int j = chosen[min(i, n - 1) / kBlock] * kBlock + i % kBlock;
            const uint64_t k = lp_key(lp_order(static_cast<float>(x[min(j, a.V - 1)])), j);
            return i < n && j < a.V ? k : 0;
          },
          n, a.top, s);
    }
  }
  if (tid >= 64) return;
  stat_to(st, wave_max_dpp(st.m));
  st.s = wave_sum_dpp(st.s);
  st.u = wave_sum_dpp(st.u);
  if (kMode == 1) {
    const uint32_t order = wave_reduce_max((uint32_t)(key >> 32));
    const uint32_t low = wave_reduce_max((uint32_t)(key >> 32) == order ? (uint32_t)key : 0u);
    key = ((uint64_t)order << 32) | low;
  } else if (kMode == 2 && lane < a.top) {
    key = s->list[lane];
  }
  lp_write<T>(a, row, st, lane, key);
}

// The pass: statistics of a segment; kMode 1: and its best key; 2: and its blocks'
// maxima.
template <typename T, int kMode>
__global__ void __launch_bounds__(kLpThreads) logprob_kernel(LogprobArgs a) {
  constexpr int EPV = 16 / (int)sizeof(T), NV = kLpElems / EPV;
  __shared__ Stat wstat[kLpThreads / 64];
  __shared__ uint32_t worder[kLpThreads / 64];
  __shared__ int place, last;
  __shared__ char select_lds[kMode == 2 ? sizeof(LpList) : 1] __attribute__((aligned(8)));
  __shared__ int chosen[kMode == 2 ? kLpMaxTop : 1];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.S;
  const int sg = (int)(blockIdx.x - row * a.S);
  const T* x = static_cast<const T*>(a.x) + row * a.sx;
  const int lo = sg * a.seg, hi = min(a.V, lo + a.seg);

  Stat st{-__FLT_MAX__, 0.f, 0.f};
  uint32_t order = 0;  // kMode 1: the thread's largest value, and the first tile that holds it
  int tile = lo;
  const bool across = a.one && a.S > 1;  // (read by a workgroup of another XCD in this launch)
  for (int j0 = lo; j0 < hi; j0 += kLpTile) {
    float v[kLpElems], vmax[NV];
    // Element q EPV + e of the thread is at place j0 + (q 256 + tid) EPV + e.
#pragma unroll
    for (int q = 0; q < NV; ++q) lp_load<T>(x, j0 + (q * kLpThreads + tid) * EPV, hi, v + q * EPV);
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      vmax[q] = v[q * EPV];
#pragma unroll
      for (int e = 1; e < EPV; ++e) vmax[q] = __builtin_elementwise_maximum(vmax[q], v[q * EPV + e]);
    }
    float tmax = vmax[0];
#pragma unroll
    for (int q = 1; q < NV; ++q) tmax = __builtin_elementwise_maximum(tmax, vmax[q]);
    if (tmax > st.m) stat_to(st, tmax);
#pragma unroll
    for (int e = 0; e < kLpElems; ++e) {
      const float d = v[e] - st.m;
      const float f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      st.s += f;
      st.u = fmaf(f, fmaxf(d, -__FLT_MAX__), st.u);  // (0 * -inf is no NaN of ours; a NaN has made f NaN)
    }
    if (kMode == 1) {
      const uint32_t k = lp_order(tmax);
      tile = k > order ? j0 : tile;
      order = max(order, k);
    }
    if (kMode == 2) {
#pragma unroll
      for (int q = 0; q < NV; ++q) {
        uint32_t k = lp_order(vmax[q]);
        k = max(k, (uint32_t)dpp_i<kDppQuadSwap1>((int)k));
        k = max(k, (uint32_t)dpp_i<kDppQuadSwap2>((int)k));
        k = max(k, (uint32_t)dpp_i<kDppHalfMirror>((int)k));
        k = max(k, (uint32_t)dpp_i<kDppMirror>((int)k));
        const int j = j0 + (q * kLpThreads + tid) * EPV;
        if ((lane & 15) == 0 && j < hi) {
          uint32_t* to = a.blocks + row * a.nb + j / kLpBlock<T>;
          if (across) st_dev(to, k);
          else *to = k;
        }
      }
    }
  }

  // The workgroup's statistics.
  float M = wave_max_dpp(st.m);
  stat_to(st, M);
  st.s = wave_sum_dpp(st.s);
  st.u = wave_sum_dpp(st.u);
  if (lane == 0) wstat[wave] = st;
  uint64_t key = 0;
  if (kMode == 1) {
    const uint32_t wo = wave_reduce_max(order);
    if (lane == 0) worder[wave] = wo;
    if (tid == 0) place = 0x7fffffff;
    __syncthreads();
    uint32_t most = worder[0];
#pragma unroll
    for (int w = 1; w < kLpThreads / 64; ++w) most = max(most, worder[w]);
    if (order == most) {
      float v[kLpElems];
#pragma unroll
      for (int q = 0; q < NV; ++q) lp_load<T>(x, tile + (q * kLpThreads + tid) * EPV, hi, v + q * EPV);
      int at = 0x7fffffff;
#pragma unroll
      for (int e = kLpElems - 1; e >= 0; --e) {
        const int j = tile + ((e / EPV) * kLpThreads + tid) * EPV + e % EPV;
        at = j < hi && lp_order(v[e]) == most ? j : at;
      }
      atomicMin(&place, at);
    }
    key = most;  // (with the place below, once every thread has looked)
  }
  __syncthreads();
  if (wave == 0) {
    if (kMode == 1) key = lp_key((uint32_t)key, place);
#pragma unroll
    for (int w = 0; w < kLpThreads / 64; ++w) M = fmaxf(M, wstat[w].m);
    Stat all{M, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < kLpThreads / 64; ++w) {
      Stat p = wstat[w];
      stat_to(p, M);
      all.s += p.s;
      all.u += p.u;
    }
    if (kMode != 2 && a.S == 1) lp_write<T>(a, row, all, lane, key);
    if (lane == 0) {
      const int64_t p = row * a.S + sg;
      if (kMode == 2 || a.S > 1) {
        st_dev(a.part + 3 * p, all.m);
        st_dev(a.part + 3 * p + 1, all.s);
        st_dev(a.part + 3 * p + 2, all.u);
        if (kMode == 1) st_dev(a.best + p, key);
      }
    }
  }
  if (a.S == 1 ? kMode != 2 : !a.one) return;
  // The row's last workgroup goes on (a row's counter is zero before the call,
  // counts its segments and wraps to zero).  Every wave's stores are out first.
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (a.S > 1) {
    if (tid == 0) {
      last = atomicInc(a.arrived + row, (uint32_t)a.S - 1u) == (uint32_t)a.S - 1u;
      if (last) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
    }
    __syncthreads();
    if (!last) return;
  }
  lp_finish<T, kMode>(a, row, reinterpret_cast<LpList*>(select_lds), chosen);
}

template <typename T, int kMode>
__global__ void __launch_bounds__(kLpThreads) logprob_finish_kernel(LogprobArgs a) {
  __shared__ LpList sel;
  __shared__ int chosen[kLpMaxTop];
  lp_finish<T, kMode>(a, blockIdx.x, &sel, chosen);
}

// Workgroups of a call: enough to fill the GPU where a row can be cut.
constexpr int64_t kLpGroups = 2048;
// Up to so many, the row's last workgroup joins its segments: one launch (one row
// of 151936, 5 alternatives: 12 to 13 us in a graph either way, 11.2 us a call from
// the host against 14.0).  With more, its wait for the stores and the counter comes
// on top of every segment, and a second kernel is faster (20 rows 14.3 against 18.7
// us in a graph, 8 rows 13.7 against 14.1).
constexpr int64_t kLpOneLaunch = 128;
static_assert(kLpOneLaunch * sizeof(uint32_t) <= kSyncBytes, "a counter per row");

struct LogprobPlan {
  int S, seg;
  size_t bytes;
};
static LogprobPlan logprob_plan(int64_t N, int64_t V, int64_t top) {
  const int64_t tiles = (V + kLpTile - 1) / kLpTile;
  const int64_t want = std::min<int64_t>({tiles, kLpMaxSegs, std::max<int64_t>(1, kLpGroups / N)});
  const int64_t per = (tiles + want - 1) / want;
  LogprobPlan p;
  p.S = (int)((tiles + per - 1) / per);
  p.seg = (int)std::min<int64_t>(per * kLpTile, INT32_MAX - kLpTile);
  // (Bytes of a part and its best key; 64 elements to the smaller block.)
  p.bytes = p.S == 1 && top <= 1
                ? 0
                : kSyncBytes + 256 + (size_t)N * p.S * 24 + (top > 1 ? (size_t)N * ((V + 63) / 64) * 4 : 0);
  return p;
}
size_t logprob_workspace_bytes(int64_t N, int64_t V, int64_t top) { return logprob_plan(N, V, top).bytes; }
int64_t logprob_max_top() { return kLpMaxTop; }

// Rows of one launch: a grid holds fewer than 2^32 work-items.  (More than
// kLpGroups rows are not cut into segments.)
constexpr int64_t kLpLaunch = (int64_t)1 << 23;
static_assert(kLpLaunch > kLpGroups, "a workgroup a row");

template <typename T>
static hipError_t launch_logprob_t(LogprobArgs a, hipStream_t st) {
  a.nb = (a.V + kLpBlock<T> - 1) / kLpBlock<T>;
  const dim3 block(kLpThreads);
  const bool two = a.S > 1 && !a.one;
  for (int64_t left = a.N; left > 0; left -= kLpLaunch) {
    a.N = std::min(left, kLpLaunch);
    const dim3 grid((unsigned)(a.N * a.S)), rows((unsigned)a.N);
    if (a.top == 0) {
      launch((logprob_kernel<T, 0>), grid, block, 0, st, a);
      if (two) launch((logprob_finish_kernel<T, 0>), rows, block, 0, st, a);
    } else if (a.top == 1) {
      launch((logprob_kernel<T, 1>), grid, block, 0, st, a);
      if (two) launch((logprob_finish_kernel<T, 1>), rows, block, 0, st, a);
    } else {
      launch((logprob_kernel<T, 2>), grid, block, 0, st, a);
      if (two) launch((logprob_finish_kernel<T, 2>), rows, block, 0, st, a);
    }
    a.x = static_cast<const T*>(a.x) + kLpLaunch * a.sx;
    if (a.tokens) {
      a.tokens += kLpLaunch;
      a.logprob += kLpLaunch;
    }
    a.entropy += kLpLaunch;
    a.top_lp += kLpLaunch * a.top;
    a.top_id += kLpLaunch * a.top;
    a.part += kLpLaunch * 3;
    a.blocks += kLpLaunch * a.nb;
  }
  return hipGetLastError();
}

hipError_t launch_token_logprobs(const dropkv_token_logprobs_args& p, hipStream_t st) {
  const LogprobPlan pl = logprob_plan(p.N, p.V, p.top);
  LogprobArgs a{};
  a.x = p.logits;
  a.sx = p.row_stride;
  a.tokens = p.tokens;
  a.N = p.N;
  a.V = (int)p.V;
  a.top = (int)p.top;
  a.S = pl.S;
  a.one = p.N * pl.S <= kLpOneLaunch;
  a.seg = pl.seg;
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p.workspace) + 15) & ~(uintptr_t)15);
  a.arrived = reinterpret_cast<uint32_t*>(ws);
  a.best = reinterpret_cast<uint64_t*>(ws + kSyncBytes);
  a.part = reinterpret_cast<float*>(a.best + (size_t)p.N * pl.S);
  a.blocks = reinterpret_cast<uint32_t*>(a.part + (size_t)p.N * pl.S * 3);
  a.logprob = p.logprob;
  a.entropy = p.entropy;
  a.top_lp = p.top_logprobs;
  a.top_id = p.top_ids;
  if (p.dtype == kDtypeFp32) return launch_logprob_t<float>(a, st);
  if (p.dtype == kDtypeBf16) return launch_logprob_t<__bf16>(a, st);
  return launch_logprob_t<_Float16>(a, st);
}

}  // namespace dkv
