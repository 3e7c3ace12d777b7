// What a row of logits x[0..V) says: the log probability of a given token, the
// entropy, and the `top` most probable tokens.
//   m = max x,  s = sum e^(x-m),  u = sum e^(x-m) (x-m)
//   log p_i = x_i - m - ln s,  H = -sum p_i ln p_i = ln s - u / s
// in one pass over the row, with the running maximum; u is taken against the
// maximum and not against zero, so that H does not come from the difference of
// two large numbers.  Rows are cut into segments where there are few of them,
// and a second kernel joins the segments.
//
// The `top` largest come from the same pass.  A value and its place make one
// 64-bit key (value above, the complement of the place below): keys are all
// different, larger means more probable, ties go to the lowest place.  A
// workgroup keeps a threshold that at least `top` keys of its segment reach;
// only keys above it are appended to a list in LDS, whose `top` largest are
// kept, and their last one made the threshold, whenever it has grown long.  The
// threshold of the first tile is the top-th largest of 64 groups' maxima.
#include "dkv_common.h"
#include "dkv_internal.h"

#include <algorithm>

namespace dkv {

constexpr int kLpThreads = 256;
constexpr int kLpElems = 16;                        // elements per thread and tile
constexpr int kLpTile = kLpThreads * kLpElems;
constexpr int kLpMaxTop = 32;
constexpr int kLpMaxSegs = 64;                      // a lane of the merge each
// List: what is kept, and what one tile adds at most once its own threshold
// holds: (top - 1) whole groups of 64 elements, and one key.
constexpr int kLpCap = kLpMaxTop + (kLpMaxTop - 1) * (kLpTile / 64) + 1;
constexpr int kLpTrim = 96;                         // a longer list is cut back
constexpr int kLpPer = (kLpCap + kLpThreads - 1) / kLpThreads;

struct LogprobArgs {
  const void* x;
  int64_t sx;  // elements between rows
  const int64_t* tokens;
  int64_t N;
  int V, top, S, seg;  // segments per row, elements per segment (whole tiles)
  float* part;         // [N, S, 3]: m, s, u
  uint64_t* keys;      // [N, S, top]
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

__device__ __forceinline__ uint64_t lp_key(float x, int i) {
  const uint32_t k = x != x ? 0xffffffffu : float_key(x);  // NaN above all, as in torch's topk
  return ((uint64_t)k << 32) | (0xffffffffu - (uint32_t)i);
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

// Keys of the list in order of rank: those of rank < top stay, at their rank.
__device__ __forceinline__ void lp_trim(uint64_t* list, int c, int top) {
  uint64_t key[kLpPer];
  int rank[kLpPer];
#pragma unroll
  for (int q = 0; q < kLpPer; ++q) {
    const int i = threadIdx.x + q * kLpThreads;
    rank[q] = top;
    if (i < c) {
      key[q] = list[i];
      int r = 0;
      for (int j = 0; j < c; ++j) r += list[j] > key[q];
      rank[q] = r;
    }
  }
  __syncthreads();
#pragma unroll
  for (int q = 0; q < kLpPer; ++q)
    if (rank[q] < top) list[rank[q]] = key[q];
  __syncthreads();
}

// kTop 0: none; 1: the largest; 2: more.
template <typename T, int kTop>
__global__ void __launch_bounds__(kLpThreads) logprob_kernel(LogprobArgs a) {
  constexpr int EPV = 16 / (int)sizeof(T), NV = kLpElems / EPV;
  struct __attribute__((packed, aligned(sizeof(T)))) Raw {
    T e[EPV];
  };
  __shared__ Stat wstat[kLpThreads / 64];
  __shared__ uint64_t wkey[kLpThreads / 64];
  __shared__ uint64_t list[kTop == 2 ? kLpCap : 1];
  __shared__ uint64_t group[kTop == 2 ? 64 : 1];
  // Keys listed by a tile.  Tile i counts in word i mod 3 and clears the next
  // one: its last readers (tile i - 2) have passed tile i - 1's barrier.
  __shared__ int added[3];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int64_t row = blockIdx.x / a.S;
  const int sg = (int)(blockIdx.x - row * a.S);
  const T* x = static_cast<const T*>(a.x) + row * a.sx;
  const int lo = sg * a.seg, hi = min(a.V, lo + a.seg);

  Stat st{-__FLT_MAX__, 0.f, 0.f};
  float best = -INFINITY;  // kTop 1: the thread's largest value and its place
  int best_i = -1;
  uint64_t T0 = 0;         // kTop 2: keys above it are listed
  float T0f = -INFINITY;
  int listed = 0;
  int turn = 0;
  if (kTop == 2) {
    if (tid == 0) added[0] = 0;
    __syncthreads();
  }

  for (int j0 = lo; j0 < hi; j0 += kLpTile) {
    float v[kLpElems];
    // Element q EPV + e of the thread is at place j0 + (q 256 + tid) EPV + e.
#pragma unroll
    for (int q = 0; q < NV; ++q) {
      const int j = j0 + (q * kLpThreads + tid) * EPV;
      if (j + EPV <= hi) {
        const Raw r = *reinterpret_cast<const Raw*>(x + j);
#pragma unroll
        for (int e = 0; e < EPV; ++e) v[q * EPV + e] = static_cast<float>(r.e[e]);
      } else {
#pragma unroll
        for (int e = 0; e < EPV; ++e) v[q * EPV + e] = j + e < hi ? static_cast<float>(x[j + e]) : -INFINITY;
      }
    }
    float tmax = v[0];
#pragma unroll
    for (int e = 1; e < kLpElems; ++e) tmax = __builtin_elementwise_maximum(tmax, v[e]);
    if (tmax > st.m) stat_to(st, tmax);
#pragma unroll
    for (int e = 0; e < kLpElems; ++e) {
      const float d = v[e] - st.m;
      const float f = __builtin_amdgcn_exp2f(d * 1.4426950408889634f);
      st.s += f;
      st.u = fmaf(f, fmaxf(d, -__FLT_MAX__), st.u);  // (0 * -inf is no NaN of ours; a NaN has made f NaN)
    }
    auto place = [&](int e) { return j0 + ((e / EPV) * kLpThreads + tid) * EPV + e % EPV; };
    if (kTop == 1) {
      if (best_i < 0 ? place(0) < hi : (tmax > best || (tmax != tmax && best == best))) {
        best = tmax;
        best_i = 0x7fffffff;
#pragma unroll
        for (int e = kLpElems - 1; e >= 0; --e)
          if (place(e) < hi && (v[e] == tmax || v[e] != v[e])) best_i = place(e);
      }
    }
    if (kTop == 2) {
      auto threshold = [&]() {  // the top-th largest of the tile's 64 group maxima, and every key above
        uint64_t k = 0;
#pragma unroll
        for (int e = 0; e < kLpElems; ++e)
          if (place(e) < hi) k = max(k, lp_key(v[e], place(e)));
        k = max(k, shfl_xor64(k, 1));
        k = max(k, shfl_xor64(k, 2));
        if ((lane & 3) == 0) group[tid >> 2] = k;
        __syncthreads();
        const uint64_t mine = group[lane];
        int r = 0;
        for (int j = 0; j < 64; ++j) r += group[j] > mine;
        const uint64_t at = __builtin_amdgcn_ballot_w64(r == a.top - 1 && mine != 0);
        // (Fewer groups than `top` hold anything: all keys pass.)
        const uint64_t t = at ? group[__builtin_ctzll(at)] - 1 : 0;
        __syncthreads();
        return t;
      };
      auto append = [&]() {
        if (!wave_any(!(tmax < T0f))) return;
#pragma unroll
        for (int e = 0; e < kLpElems; ++e) {
          const uint64_t k = place(e) < hi ? lp_key(v[e], place(e)) : 0;
          if (k > T0) {
            const int at = listed + atomicAdd(&added[turn], 1);
            if (at < kLpCap) list[at] = k;
          }
        }
      };
      auto set = [&](uint64_t t) {
        if (t <= T0) return;
        T0 = t;
        const uint32_t hk = (uint32_t)(t >> 32);
        T0f = hk == 0xffffffffu ? INFINITY : key_float(hk);
      };
      const int next = turn == 2 ? 0 : turn + 1;
      if (tid == 0) added[next] = 0;
      if (j0 == lo) set(threshold());
      append();
      __syncthreads();
      int c = listed + added[turn];
      if (c > kLpCap) {
        // More than fits: the list as it was before this tile is cut back, and
        // the tile goes in again above a threshold of its own.
        lp_trim(list, listed, a.top);
        if (listed >= a.top) set(list[a.top - 1]);
        listed = min(listed, a.top);
        if (tid == 0) added[turn] = 0;
        set(threshold());
        append();
        __syncthreads();
        c = listed + added[turn];
      }
      if (c > kLpTrim) {
        lp_trim(list, c, a.top);
        set(list[a.top - 1]);
        c = a.top;
      }
      listed = c;
      turn = next;
    }
  }

  // The workgroup's statistics.
  const float wm = wave_max(st.m);
  float M = wm;
  stat_to(st, wm);
  st.s = wave_sum(st.s);
  st.u = wave_sum(st.u);
  if (lane == 0) wstat[wave] = st;
  if (kTop == 1) {
    uint64_t k = best_i < 0 ? 0 : lp_key(best, best_i);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) k = max(k, shfl_xor64(k, o));
    if (lane == 0) wkey[wave] = k;
  }
  __syncthreads();
  if (kTop == 2) lp_trim(list, listed, a.top);
  if (wave != 0) return;
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
  uint64_t key = 0;
  if (kTop == 1) {
#pragma unroll
    for (int w = 0; w < kLpThreads / 64; ++w) key = max(key, wkey[w]);
  }
  if (kTop == 2 && lane < min(listed, a.top)) key = list[lane];
  if (a.S == 1) {
    lp_write<T>(a, row, all, lane, key);
    return;
  }
  const int64_t p = row * a.S + sg;
  if (lane == 0) {
    a.part[3 * p] = all.m;
    a.part[3 * p + 1] = all.s;
    a.part[3 * p + 2] = all.u;
  }
  if (lane < a.top) a.keys[p * a.top + lane] = key;
}

// One wave per row: a lane per segment, whose keys are in falling order.
template <typename T>
__global__ void __launch_bounds__(64) logprob_merge_kernel(LogprobArgs a) {
  const int64_t row = blockIdx.x;
  const int lane = threadIdx.x;
  const bool on = lane < a.S;
  const int64_t p = row * a.S + lane;
  Stat st{-__FLT_MAX__, 0.f, 0.f};
  if (on) st = Stat{a.part[3 * p], a.part[3 * p + 1], a.part[3 * p + 2]};
  stat_to(st, wave_max(st.m));
  st.s = wave_sum(st.s);
  st.u = wave_sum(st.u);
  const uint64_t* mine = a.keys + p * a.top;
  uint64_t head = on && a.top > 0 ? mine[0] : 0, key = 0;
  int at = 0;
  for (int i = 0; i < a.top; ++i) {
    uint64_t k = head;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) k = max(k, shfl_xor64(k, o));
    if (lane == i) key = k;
    if (head == k && k != 0) {
      ++at;
      head = at < a.top ? mine[at] : 0;
    }
  }
  lp_write<T>(a, row, st, lane, key);
}

// Workgroups of a call: enough to fill the GPU where a row can be cut.
constexpr int64_t kLpGroups = 2048;

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
  p.bytes = p.S == 1 ? 0 : kSyncBytes + (size_t)N * p.S * (3 * sizeof(float) + (size_t)top * sizeof(uint64_t)) + 256;
  return p;
}
size_t logprob_workspace_bytes(int64_t N, int64_t V, int64_t top) { return logprob_plan(N, V, top).bytes; }
int64_t logprob_max_top() { return kLpMaxTop; }

template <typename T>
static hipError_t launch_logprob_t(const LogprobArgs& a, hipStream_t st) {
  const dim3 grid((unsigned)(a.N * a.S));
  if (a.top == 0)
    launch((logprob_kernel<T, 0>), grid, dim3(kLpThreads), 0, st, a);
  else if (a.top == 1)
    launch((logprob_kernel<T, 1>), grid, dim3(kLpThreads), 0, st, a);
  else
    launch((logprob_kernel<T, 2>), grid, dim3(kLpThreads), 0, st, a);
  if (a.S > 1) launch((logprob_merge_kernel<T>), dim3((unsigned)a.N), dim3(64), 0, st, a);
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
  a.seg = pl.seg;
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p.workspace) + 15) & ~(uintptr_t)15);
  a.keys = reinterpret_cast<uint64_t*>(ws + kSyncBytes);
  a.part = reinterpret_cast<float*>(a.keys + (size_t)p.N * pl.S * p.top);
  a.logprob = p.logprob;
  a.entropy = p.entropy;
  a.top_lp = p.top_logprobs;
  a.top_id = p.top_ids;
  if (p.dtype == kDtypeFp32) return launch_logprob_t<float>(a, st);
  if (p.dtype == kDtypeBf16) return launch_logprob_t<__bf16>(a, st);
  return launch_logprob_t<_Float16>(a, st);
}

}  // namespace dkv
