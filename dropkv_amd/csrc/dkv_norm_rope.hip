// Queries and keys of new tokens made ready for the cache and the attention:
// an RMS norm over each head (optional), the rotation by position, and K and V
// stored where the caller keeps them, in one pass.  (The reference takes
// rotated queries and keys from the model; patches/dropkv_transformers.patch:
// 329-343.)
//
// For a head's row x of D values and the token's rows c, s of R values:
//   y = x rsqrt(mean(x^2) + eps) w          (y = x without a weight)
//   z_i       = y_i c_i - y_{i+R/2} s_i               i < R/2
//   z_{i+R/2} = y_{i+R/2} c_{i+R/2} + y_i s_{i+R/2}
//   z_i       = y_i                                   i >= R
// in fp32, rounded once, at the store.
//
// Bound by memory: every row is read and written once (4 x 7001 tokens of 32 query
// and 8 KV heads of 128, fp16, norms and V: 688 MB in 148 to 151 us, 4.6 TB/s, where a
// large copy reaches 4.9; 8 tokens 3.7 us, one round trip).  A lane holds 8 values
// of the first half and their partners of the second, so that a pair never
// leaves the lane and the norm is a reduction over the row's 4, 8 or 16 lanes, of
// which D / 16 hold values.  A
// wave takes several heads of one token, since c and s (as long as a row, and
// in fp32 twice its bytes) are then loaded once for all of them.
#include "dkv_common.h"
#include "dkv_internal.h"

#include <algorithm>

namespace dkv {

struct RopeSide {  // of q, k or v: row (b, h, l) at element b sb + h sh + l sl
  const void* src;
  void* dst;
  int64_t s_sb, s_sh, s_sl, d_sb, d_sh, d_sl;
  const void* w;  // norm weight, or null
};
struct RopeArgs {
  RopeSide q, k, v;
  int w_f32;
  const void* cos;  // row l of sequence b at element b c_sb + l c_sl; with positions, row `position` at position * c_sl
  const void* sin;
  int64_t c_sb, c_sl;
  const int64_t* pos;
  int64_t p_sb, P;
  int L, Hq, Hk, Hv, D, R, tokens;
  int per, chunks;  // heads (q, k and v, in that order) per wave; waves per token
  int64_t first;    // the launch's first wave
  float eps;
};

// Eight values from or to a 16-byte aligned place.
template <typename T>
__device__ __forceinline__ void load_vec8(const T* p, float* f) {
  if constexpr (sizeof(T) == 4) {
    const f32x4 x0 = reinterpret_cast<const f32x4*>(p)[0], x1 = reinterpret_cast<const f32x4*>(p)[1];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = e < 4 ? x0[e % 4] : x1[e % 4];
  } else {
    const typename Elem<T>::v8 x = *reinterpret_cast<const typename Elem<T>::v8*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(x[e]);
  }
}
template <typename T>
__device__ __forceinline__ void store_vec8(T* p, const float* f) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<f32x4*>(p)[0] = f32x4{f[0], f[1], f[2], f[3]};
    reinterpret_cast<f32x4*>(p)[1] = f32x4{f[4], f[5], f[6], f[7]};
  } else {
    typename Elem<T>::v8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = static_cast<T>(f[e]);
    *reinterpret_cast<typename Elem<T>::v8*>(p) = x;
  }
}

// The side that head hh of the list (q's, k's, v's heads) belongs to, and its head
// there.  (Member by member: an array indexed by the lane is kept in LDS.)
__device__ __forceinline__ RopeSide rope_side(const RopeArgs& a, int hh, int* h, bool* copy) {
  const bool q = hh < a.Hq, k = hh < a.Hq + a.Hk;
  *h = hh - (q ? 0 : k ? a.Hq : a.Hq + a.Hk);
  *copy = !k;
  RopeSide s;
  s.src = q ? a.q.src : k ? a.k.src : a.v.src;
  s.dst = q ? a.q.dst : k ? a.k.dst : a.v.dst;
  s.s_sb = q ? a.q.s_sb : k ? a.k.s_sb : a.v.s_sb;
  s.s_sh = q ? a.q.s_sh : k ? a.k.s_sh : a.v.s_sh;
  s.s_sl = q ? a.q.s_sl : k ? a.k.s_sl : a.v.s_sl;
  s.d_sb = q ? a.q.d_sb : k ? a.k.d_sb : a.v.d_sb;
  s.d_sh = q ? a.q.d_sh : k ? a.k.d_sh : a.v.d_sh;
  s.d_sl = q ? a.q.d_sl : k ? a.k.d_sl : a.v.d_sl;
  s.w = q ? a.q.w : a.k.w;
  return s;
}

// The token's row of the tables; false where its position is not in them.
template <typename TC>
__device__ __forceinline__ bool rope_row(const RopeArgs& a, int b, int l, const TC** c, const TC** s) {
  int64_t off = (int64_t)b * a.c_sb + (int64_t)l * a.c_sl;
  if (a.pos) {
    const int64_t p = a.pos[(int64_t)b * a.p_sb + l];
    if (p < 0 || p >= a.P) return false;
    off = p * a.c_sl;
  }
  *c = static_cast<const TC*>(a.cos) + off;
  *s = static_cast<const TC*>(a.sin) + off;
  return true;
}

// LPR lanes a row, D / 16 of them at work (D a multiple of 16).
template <typename T, typename TC, int LPR>
__global__ void __launch_bounds__(256) norm_rope_kernel(RopeArgs a) {
  constexpr int HPW = 64 / LPR;
  const int wid = (int)a.first + blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x & 63;
  const int token = wid / a.chunks, h0 = (wid - token * a.chunks) * a.per;
  if (token >= a.tokens) return;
  const int b = token / a.L, l = token - b * a.L;
  const int c = lane % LPR;
  const int R = a.R, pairs = R / 16;
  const bool live = 16 * c < a.D;
  // The lane's two runs of 8 values.
  const bool turned = c < pairs;
  const int i0 = turned ? 8 * c : R + 16 * (c - pairs), i1 = turned ? i0 + R / 2 : i0 + 8;
  float c0[8], c1[8], s0[8], s1[8];
  if (turned) {
    const TC *cr, *sr;
    if (rope_row(a, b, l, &cr, &sr)) {
      load_vec8(cr + i0, c0);
      load_vec8(cr + i1, c1);
      load_vec8(sr + i0, s0);
      load_vec8(sr + i1, s1);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) c0[e] = c1[e] = s0[e] = s1[e] = __builtin_nanf("");
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      c0[e] = c1[e] = 1.f;
      s0[e] = s1[e] = 0.f;
    }
  }
  const int heads = a.Hq + a.Hk + a.Hv, h_end = min(heads, h0 + a.per);
  for (int hh = h0 + lane / LPR; hh < h_end; hh += HPW) {
    int h;
    bool copy;
    const RopeSide side = rope_side(a, hh, &h, &copy);
    const T* src = static_cast<const T*>(side.src) + b * side.s_sb + h * side.s_sh + l * side.s_sl;
    T* dst = static_cast<T*>(side.dst) + b * side.d_sb + h * side.d_sh + l * side.d_sl;
    if (copy) {
      if (!live) continue;
#pragma unroll
      for (int u = 0; u < (int)sizeof(T) / 2; ++u) {  // 16 bytes each
        const u32x4 x0 = reinterpret_cast<const u32x4*>(src + i0)[u], x1 = reinterpret_cast<const u32x4*>(src + i1)[u];
        reinterpret_cast<u32x4*>(dst + i0)[u] = x0;
        reinterpret_cast<u32x4*>(dst + i1)[u] = x1;
      }
      continue;
    }
    float x0[8] = {}, x1[8] = {};
    if (live) {
      load_vec8(src + i0, x0);
      load_vec8(src + i1, x1);
    }
    const void* w = side.w;
    if (w) {
      float ss = 0.f, w0[8] = {}, w1[8] = {};
      if (!live) {
      } else if (a.w_f32) {
        load_vec8(static_cast<const float*>(w) + i0, w0);
        load_vec8(static_cast<const float*>(w) + i1, w1);
      } else {
        load_vec8(static_cast<const T*>(w) + i0, w0);
        load_vec8(static_cast<const T*>(w) + i1, w1);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(x0[e], x0[e], fmaf(x1[e], x1[e], ss));
#pragma unroll
      for (int o = 1; o < LPR; o <<= 1) ss += __shfl_xor(ss, o);
      const float inv = 1.f / sqrtf(ss / (float)a.D + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x0[e] = x0[e] * inv * w0[e];
        x1[e] = x1[e] * inv * w1[e];
      }
    }
    if (turned) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float y0 = fmaf(x0[e], c0[e], -(x1[e] * s0[e]));
        x1[e] = fmaf(x1[e], c1[e], x0[e] * s1[e]);
        x0[e] = y0;
      }
    }
    if (live) {
      store_vec8(dst + i0, x0);
      store_vec8(dst + i1, x1);
    }
  }
}

// Any head dimension, alignment and rotated width: a wave per head's row, a
// pair per lane at a time (4096 tokens of 32 + 8 heads of 96: 112 us where the
// kernel above takes 19).
template <typename T, typename TC>
__global__ void __launch_bounds__(256) norm_rope_any_kernel(RopeArgs a) {
  const int heads = a.Hq + a.Hk + a.Hv;
  const int64_t wid = a.first + (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
  const int lane = threadIdx.x & 63;
  if (wid >= (int64_t)a.tokens * heads) return;
  const int token = (int)(wid / heads), hh = (int)(wid - (int64_t)token * heads);
  const int b = token / a.L, l = token - b * a.L;
  int h;
  bool copy;
  const RopeSide side = rope_side(a, hh, &h, &copy);
  const T* src = static_cast<const T*>(side.src) + b * side.s_sb + h * side.s_sh + l * side.s_sl;
  T* dst = static_cast<T*>(side.dst) + b * side.d_sb + h * side.d_sh + l * side.d_sl;
  if (copy) {
    for (int i = lane; i < a.D; i += 64) dst[i] = src[i];
    return;
  }
  const void* w = side.w;
  float inv = 1.f;
  if (w) {
    float ss = 0.f;
    for (int i = lane; i < a.D; i += 64) {
      const float x = static_cast<float>(src[i]);
      ss = fmaf(x, x, ss);
    }
    inv = 1.f / sqrtf(wave_sum(ss) / (float)a.D + a.eps);
  }
  auto get = [&](int i) {
    const float x = static_cast<float>(src[i]);
    if (!w) return x;
    return x * inv * (a.w_f32 ? static_cast<const float*>(w)[i] : static_cast<float>(static_cast<const T*>(w)[i]));
  };
  const TC *cr = nullptr, *sr = nullptr;
  const bool known = rope_row(a, b, l, &cr, &sr);
  const int half = a.R / 2;
  for (int i = lane; i < half; i += 64) {
    const float x0 = get(i), x1 = get(i + half);
    const float c0 = known ? static_cast<float>(cr[i]) : __builtin_nanf("");
    const float c1 = known ? static_cast<float>(cr[i + half]) : __builtin_nanf("");
    const float s0 = known ? static_cast<float>(sr[i]) : 0.f, s1 = known ? static_cast<float>(sr[i + half]) : 0.f;
    dst[i] = static_cast<T>(fmaf(x0, c0, -(x1 * s0)));
    dst[i + half] = static_cast<T>(fmaf(x1, c1, x0 * s1));
  }
  for (int i = a.R + lane; i < a.D; i += 64) dst[i] = static_cast<T>(get(i));
}

// Waves that a call is spread over, where its tokens allow.
constexpr int64_t kRopeWaves = 4096;
// Waves of one launch: a grid holds fewer than 2^32 work-items.
constexpr int64_t kRopeLaunch = (int64_t)1 << 25;

template <typename F>
static void launch_waves(F kernel, RopeArgs& a, int64_t waves, hipStream_t st) {
  for (a.first = 0; a.first < waves; a.first += kRopeLaunch)
    launch(kernel, dim3((unsigned)((std::min(waves - a.first, kRopeLaunch) + 3) / 4)), dim3(256), 0, st, a);
}

template <typename T, typename TC>
static hipError_t launch_rope_t(RopeArgs a, bool vec, hipStream_t st) {
  const int64_t heads = (int64_t)a.Hq + a.Hk + a.Hv;
  if (vec && a.D % 16 == 0 && a.D <= 256) {
    const int lanes = a.D <= 64 ? 4 : a.D <= 128 ? 8 : 16, hpw = 64 / lanes;
    const int64_t its = (heads + hpw - 1) / hpw;
    const int64_t want = std::min<int64_t>(its, std::max<int64_t>(1, kRopeWaves / a.tokens));  // waves per token
    const int64_t its_w = (its + want - 1) / want;
    a.per = (int)(its_w * hpw);
    a.chunks = (int)((its + its_w - 1) / its_w);
    const int64_t waves = (int64_t)a.tokens * a.chunks;
    if (lanes == 4)
      launch_waves(norm_rope_kernel<T, TC, 4>, a, waves, st);
    else if (lanes == 8)
      launch_waves(norm_rope_kernel<T, TC, 8>, a, waves, st);
    else
      launch_waves(norm_rope_kernel<T, TC, 16>, a, waves, st);
  } else {
    launch_waves(norm_rope_any_kernel<T, TC>, a, (int64_t)a.tokens * heads, st);
  }
  return hipGetLastError();
}

hipError_t launch_norm_rope(const dropkv_norm_rope_args& p, hipStream_t st) {
  RopeArgs a{};
  const int64_t eb = p.dtype == kDtypeFp32 ? 4 : 2, cb = p.c_dtype == kDtypeFp32 ? 4 : eb;
  uint64_t all = 0;
  auto tensor = [&](const void* src, const int64_t* s, void* dst, const int64_t* d, const void* w) {
    all |= reinterpret_cast<uintptr_t>(src) | reinterpret_cast<uintptr_t>(dst) | reinterpret_cast<uintptr_t>(w) |
           (uint64_t)((s[0] | s[1] | s[2] | d[0] | d[1] | d[2]) * eb);
    return RopeSide{src, dst, s[0], s[1], s[2], d[0], d[1], d[2], w};
  };
  a.q = tensor(p.q, p.q_s, p.q_out, p.qo_s, p.q_w);
  a.k = tensor(p.k, p.k_s, p.k_out, p.ko_s, p.k_w);
  if (p.v) a.v = tensor(p.v, p.v_s, p.v_out, p.vo_s, nullptr);
  a.w_f32 = p.w_dtype == kDtypeFp32;
  a.cos = p.cos;
  a.sin = p.sin;
  a.c_sb = p.positions ? 0 : p.c_sb;
  a.c_sl = p.c_sl;
  a.pos = p.positions;
  a.p_sb = p.p_sb;
  a.P = p.c_rows;
  a.L = (int)p.L;
  a.tokens = (int)(p.B * p.L);
  a.Hq = (int)p.Hq;
  a.Hk = (int)p.Hkv;
  a.Hv = p.v ? (int)p.Hkv : 0;
  a.D = (int)p.D;
  a.R = (int)p.R;
  a.eps = (float)p.eps;
  all |= reinterpret_cast<uintptr_t>(p.cos) | reinterpret_cast<uintptr_t>(p.sin) | (uint64_t)((a.c_sb | a.c_sl) * cb);
  const bool vec = all % 16 == 0 && p.R % 16 == 0;
  if (p.dtype == kDtypeFp32) return launch_rope_t<float, float>(a, vec, st);
  if (p.dtype == kDtypeBf16)
    return cb == 4 ? launch_rope_t<__bf16, float>(a, vec, st) : launch_rope_t<__bf16, __bf16>(a, vec, st);
  return cb == 4 ? launch_rope_t<_Float16, float>(a, vec, st) : launch_rope_t<_Float16, _Float16>(a, vec, st);
}

}  // namespace dkv
