// What the attention kernels of drafted tokens share (dkv_tree.hip, over a
// cache in 16 bits; dkv_quant_attn.hip, in 8): how the cache is cut into
// parts, the mask of the drafted keys, and the kernel that joins the parts.
#pragma once

#include "dkv_common.h"
#include "dkv_internal.h"
#include "dkv_select_dev.h"

#include <type_traits>

namespace dkv {

constexpr int kTreeTile = 32;       // keys per tile
constexpr int kTreeMaxSplits = 63;  // of the cache: one lane of the merge each, with the drafted keys'

struct TreeArgs {
  const void* q;  // [B, Hq, T, D], D contiguous
  int64_t q_sb, q_sh, q_st;
  const void* kn;  // drafted K and V [B, Hkv, T, D], D contiguous
  const void* vn;
  int64_t kn_sb, kn_sh, kn_st, vn_sb, vn_sh, vn_st;
  const void* kbuf;  // [B, Hkv, C, D] contiguous
  const void* vbuf;
  const int* n_rows;
  int n_sb;             // 0: one count for every sequence
  const uint8_t* mask;  // [T, T] bytes at m_sb, m_st, m_sj; null: a chain (j <= t)
  int64_t m_sb, m_st, m_sj;
  int B, Hq, Hkv, D, T, C, M, S, MC;
  int P;       // parts of a KV head: S per sequence, and one more each where the drafted keys are a part of their own
  int apart;   // they are
  int tail_tiles;
  int ragged;  // the B * S parts are dealt out by the sequences' lengths
  int direct;  // one part: the output is written by it
  Div div_t;
  float scale_log2;
  int* deal;      // [B, 2]: first part and number of parts (ragged), for the joining kernel
  float* part_m;  // [Hkv, P, M]
  float* part_l;
  float* part_o;  // [Hkv, P, M, D]
  void* out;      // [B, T, Hq, D], D contiguous
  int64_t o_sb, o_st, o_sh;
};

template <typename T>
__device__ __forceinline__ bool not_finite(T x) {
  constexpr uint16_t kExp = std::is_same<T, _Float16>::value ? 0x7c00 : 0x7f80;
  return (__builtin_bit_cast(uint16_t, x) & kExp) == kExp;
}

// Eight elements of a row that may start anywhere (the hardware's 16-byte loads
// take any address).
template <typename T>
__device__ __forceinline__ typename Elem<T>::v8 tree_load8(const T* p) {
  struct __attribute__((packed, aligned(sizeof(T)))) Raw {
    T e[8];
  };
  return __builtin_bit_cast(typename Elem<T>::v8, *reinterpret_cast<const Raw*>(p));
}

// Lane i's value and lane i ^ 16's (32's), the larger; NaN where either is.
__device__ __forceinline__ float maximum_xor16(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float maximum_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __builtin_elementwise_maximum(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// Sequence b's stored rows.  The host keeps 0 <= n <= C; the clamp keeps every
// access in bounds.
__device__ __forceinline__ int tree_rows(const TreeArgs& a, int b) {
  return min(max(a.n_rows[b * a.n_sb], 0), a.C);
}

// Sequence b's parts of the cache: `count` of them from `first` on, `per` tiles
// each.  With one count for all, or one sequence, S parts each.  Otherwise the
// B * S parts go by length, so that no workgroup has much more than the mean (8
// sequences of 940 to 8003 rows at equal parts: the longest took twice the
// mean's time): ceil(tiles / per) parts each, at least one, with about the least
// `per` whose parts fit; sum ceil(t_b / per) <= sum t_b / per + B always does at
// sum / (B (S - 1)).  Every lane of the wave calls this; lane i looks at
// sequence i.  Drafted keys that go with a sequence's last part count as
// `tail_tiles` tiles of it.  Cut::tiles(n): the tiles that n rows make.
struct TreeCut {
  static __device__ __forceinline__ int tiles(int n) { return (n + kTreeTile - 1) / kTreeTile; }
};
constexpr int kTreeRaggedB = 64;
constexpr size_t kTreeDealBytes = kTreeRaggedB * 2 * sizeof(int);
struct TreeParts {
  int first, count, per;
};
__device__ __forceinline__ int ceil_div(int a, int b) { return (a + b - 1) / b; }
__device__ __forceinline__ int wave_sum_int(int x) { return (int)wave_reduce_add((uint32_t)x); }
template <class Cut>
__device__ __forceinline__ TreeParts tree_parts_ragged(const TreeArgs& a, int lane) {
  const int t = lane < a.B ? Cut::tiles(tree_rows(a, lane)) + a.tail_tiles : 0;
  const int sum = wave_sum_int(t), most = (int)wave_reduce_max((uint32_t)t);
  TreeParts p;
  p.per = max(max(1, ceil_div(most, kTreeMaxSplits)), ceil_div(sum, a.B * a.S));
  for (;;) {
    p.count = lane < a.B ? max(1, ceil_div(t, p.per)) : 0;
    if (wave_sum_int(p.count) <= a.B * a.S) break;
    p.per += max(1, p.per / 32);  // (ends where per >= sum / (B (S - 1)) at the latest)
  }
  p.first = (int)wave_incl_scan((uint32_t)p.count) - p.count;
  return p;
}
// Part `slot` of a KV head: tiles t_lo .. t_hi of sequence b, whose stored rows
// are n, and with `tail` the drafted keys; b < 0: none.  The sequence's parts are
// `count` from `first` on.
struct TreePart {
  int b, n, t_lo, t_hi;
  bool tail;
  int first, count;
};
template <class Cut = TreeCut>
__device__ __forceinline__ TreePart tree_part(const TreeArgs& a, int hkv, int slot, int lane) {
  TreePart p;
  if (slot >= a.B * a.S) return TreePart{slot - a.B * a.S, 0, 0, 0, true, 0, 0};
  int first, count, per;
  if (a.ragged) {
    const TreeParts all = tree_parts_ragged<Cut>(a, lane);
    if (slot == 0 && hkv == 0 && lane < a.B) {  // (by each workgroup of the slot's rows alike)
      a.deal[2 * lane] = all.first;
      a.deal[2 * lane + 1] = all.count;
    }
    const uint64_t hit = __builtin_amdgcn_ballot_w64(all.first <= slot && slot < all.first + all.count);
    if (!hit) return TreePart{-1, 0, 0, 0, false, 0, 0};
    p.b = __builtin_ctzll(hit);
    first = __builtin_amdgcn_readlane(all.first, p.b);
    count = __builtin_amdgcn_readlane(all.count, p.b);
    per = __builtin_amdgcn_readfirstlane(all.per);
    p.n = tree_rows(a, p.b);
  } else {
    p.b = slot / a.S;
    p.n = tree_rows(a, p.b);
    first = p.b * a.S;
    count = a.S;
    per = ceil_div(Cut::tiles(p.n) + a.tail_tiles, a.S);
  }
  const int tiles = Cut::tiles(p.n);
  p.t_lo = min((slot - first) * per, tiles);
  p.t_hi = min(p.t_lo + per, tiles);
  p.tail = !a.apart && slot - first == count - 1;
  p.first = first;
  p.count = count;
  return p;
}

// The mask of drafted keys j0 .. j0 + 63, a word per token: a wave takes every
// NW-th token, a lane a key (a lane's own bytes one by one, a row each, took
// longer than the tile's products).
// The loads are unconditional (the last token's row and key again past the
// ends): behind branches they went out one after the other.
template <int NW>
__device__ __forceinline__ void tree_mask_words(const TreeArgs& a, int b, int j0, int wave, int lane, uint64_t* words) {
  const int j = j0 + lane;
  if (!a.mask) {  // a chain
    for (int t = 64 * wave + lane; t < a.T; t += 64 * NW)
      words[t] = t < j0 ? 0 : t - j0 >= 63 ? ~uint64_t(0) : (uint64_t(2) << (t - j0)) - 1;
    return;
  }
  const uint8_t* m = a.mask + (int64_t)b * a.m_sb + (int64_t)min(j, a.T - 1) * a.m_sj;
  for (int t0 = wave; t0 < a.T; t0 += 8 * NW) {
    uint8_t x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = m[(int64_t)min(t0 + i * NW, a.T - 1) * a.m_st];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint64_t w = __builtin_amdgcn_ballot_w64(j < a.T && x[i] != 0);
      if (lane == 0 && t0 + i * NW < a.T) words[t0 + i * NW] = w;
    }
  }
}
// Bits 0 .. 3 and 16 .. 19 of a tile's word (shifted by 4 lg): the lane's keys.
__device__ __forceinline__ uint32_t tree_key_bits(uint32_t w) { return (w & 0xf) | ((w >> 12) & 0xf0); }
// The same of a word whose first `keys` bits are set.
__device__ __forceinline__ uint32_t tree_first_bits(int keys, int lg) {
  return tree_key_bits(keys >= 32 ? 0xffffffffu : ((1u << max(keys, 0)) - 1u) >> (4 * lg));
}

// A drafted value that is not finite reaches only the rows that see its key: the
// products take it as zero (0 * inf is NaN), and here, once the part's rows are
// stored, it is added where it is seen.  Rare: one element at a time.
template <typename T, int D, int NT>
__device__ __forceinline__ void tree_add_odd(const TreeArgs& a, int b, int hkv, int slot, int row0, int rows) {
  const T* vn = static_cast<const T*>(a.vn) + (int64_t)b * a.vn_sb + (int64_t)hkv * a.vn_sh;
  for (int i = threadIdx.x; i < rows * D; i += NT) {
    const int row = row0 + i / D, d = i % D;
    if (row >= a.M) break;
    const int h = a.div_t.div(row), t = row - h * a.T;
    float sum = 0.f;
    for (int j = 0; j < a.T; ++j) {
      const bool see =
          a.mask ? a.mask[(int64_t)b * a.m_sb + (int64_t)t * a.m_st + (int64_t)j * a.m_sj] != 0 : j <= t;
      const T x = vn[(int64_t)j * a.vn_st + d];
      if (see && not_finite<T>(x)) sum += static_cast<float>(x);
    }
    if (sum == 0.f) continue;
    if (a.direct) {
      T* o = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)t * a.o_st +
             (int64_t)(hkv * (a.Hq / a.Hkv) + h) * a.o_sh + d;
      *o = static_cast<T>(static_cast<float>(*o) + sum);
    } else {
      float* o = a.part_o + (((int64_t)hkv * a.P + slot) * a.M + row) * D + d;
      st_dev(o, *o + sum);
    }
  }
}

// One wave per row: lane s holds part s's maximum and sum, D / 4 lanes a
// partial output row.  The first eight loads of partial outputs are issued with
// the statistics, before the reductions: one round trip for up to 16 (D = 128)
// or 32 parts.  4 to 5 us for a few hundred rows, all latency; 16384 rows of 4 parts
// 12 us.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeArgs a) {
  constexpr int LPR = D / 4, SPL = 64 / LPR, NL = 8;
  const int wid = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x & 63;
  if (wid >= a.B * a.Hkv * a.M) return;
  const int bh = wid / a.M, row = wid - bh * a.M;
  const int b = bh / a.Hkv, hkv = bh % a.Hkv;
  const int h = a.div_t.div(row), t = row - h * a.T;
  const int sub = lane / LPR, d0 = 4 * (lane % LPR);
  const int first = a.ragged ? a.deal[2 * b] : b * a.S, count = a.ragged ? a.deal[2 * b + 1] : a.S;
  const int S1 = count + a.apart;
  // Row of part s: those of the cache, then the drafted keys'.
  auto at = [&](int s) { return ((int64_t)hkv * a.P + (s < count ? first + s : a.B * a.S + b)) * a.M + row; };
  const float ml = lane < S1 ? a.part_m[at(lane)] : -__FLT_MAX__;
  const float ll = lane < S1 ? a.part_l[at(lane)] : 0.f;
  f32x4 x[NL];
  auto fetch = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int s = s0 + SPL * i + sub;
      x[i] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (s < S1) x[i] = *reinterpret_cast<const f32x4*>(a.part_o + at(s) * D + d0);
    }
  };
  fetch(0);
  const float mx = wave_max_dpp(ml);
  const float f = __builtin_amdgcn_exp2f(ml - mx);
  const float l = wave_sum_dpp(ll * f);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s0 = 0; s0 < S1; s0 += SPL * NL) {
    if (s0 > 0) fetch(s0);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const float fs = __shfl(f, (s0 + SPL * i + sub) & 63);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(fs, x[i][e], acc[e]);
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)t * a.o_st +
           (int64_t)(hkv * (a.Hq / a.Hkv) + h) * a.o_sh;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float y = add_xor32(acc[e]);
    if (SPL == 4) y = add_xor16(y);
    if (sub == 0) out[d0 + e] = static_cast<T>(l == 0.f ? 0.f : y * inv);
  }
}

}  // namespace dkv
