// Attention of a tree (or chain) of drafted tokens over the compressed cache,
// and the accepted path's rows appended to it: one verification step of
// speculative decoding.  (The reference decodes one token per step and appends
// its row with torch.cat, dropkv_cache.py:609-617.)
//
// Attention: T drafted tokens per sequence, whose K and V rows are not in the
// cache yet.  Token t sees the n rows that the cache holds, and drafted token j
// where mask[t][j].  The g query heads of a KV head and the T tokens are its
// M = g T rows, row h T + t, 16 to a matrix-core tile:
//   out_r = sum_j e^(s_rj - m_r) v_j / sum_j e^(s_rj - m_r),  s_rj = scale q_r . k_j
// over the cache in splits of whole 32-key tiles and the drafted keys as one
// split more (the only one with a mask), joined by a second kernel.  The call
// writes only its output.
//
// Commit: node 0 of each tree is accepted (it is the token that the step was
// fed); from an accepted node the walk goes to its lowest child whose token is
// the one chosen after it.  The path's K and V rows go to rows n, n + 1, ... of
// every layer's cache.
#include "dkv_common.h"
#include "dkv_internal.h"

#include <algorithm>
#include <cmath>

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
  int qvec, nvec;
  Div div_t;
  float scale_log2;
  float* part_m;  // [B*Hkv, S + 1, M]
  float* part_l;
  float* part_o;  // [B*Hkv, S + 1, M, D]
  void* out;      // [B, T, Hq, D], D contiguous
  int64_t o_sb, o_st, o_sh;
};

// P in the element type.  fp16 keeps it 2^14 times larger: its smallest number
// is 2^-24, and a long cache holds many keys whose weight against the running
// maximum is below that (the factor goes into the reference of the exponent and
// cancels in the quotient).
template <typename T>
constexpr float kPBias = 0.f;
template <>
constexpr float kPBias<_Float16> = 14.f;

template <typename T>
__device__ __forceinline__ bool not_finite(T x) {
  constexpr uint16_t kExp = std::is_same<T, _Float16>::value ? 0x7c00 : 0x7f80;
  return (__builtin_bit_cast(uint16_t, x) & kExp) == kExp;
}

template <typename T>
__device__ __forceinline__ typename Elem<T>::v8 tree_load8(const T* p, bool vec) {
  typename Elem<T>::v8 x;
  if (vec) {
    x = *reinterpret_cast<const typename Elem<T>::v8*>(p);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[e];
  }
  return x;
}

// Sequence b's stored rows.  The host keeps 0 <= n <= C; the clamp keeps every
// access in bounds.
__device__ __forceinline__ int tree_rows(const TreeArgs& a, int b) {
  return min(max(a.n_rows[b * a.n_sb], 0), a.C);
}

template <typename T, int D>
__global__ void __launch_bounds__(64) tree_partial_kernel(TreeArgs a) {
  typedef typename Elem<T>::v8 v8;
  constexpr int KK = D / 32, DT = D / 16, CPR = D / 8, GRP = 64 / CPR, NVC = kTreeTile / GRP;
  constexpr int kVPitch = D + 16;  // transposing reads without bank conflicts
  constexpr uint32_t kRowBytes = D * (uint32_t)sizeof(T);
  const int split = blockIdx.x % (a.S + 1);
  const int mc = (blockIdx.x / (a.S + 1)) % a.MC, bh = blockIdx.x / ((a.S + 1) * a.MC);
  const int b = bh / a.Hkv, hkv = bh % a.Hkv, g = a.Hq / a.Hkv;
  const int lane = threadIdx.x, li = lane & 15, lg = lane >> 4;
  __shared__ __attribute__((aligned(16))) T vt[kTreeTile * kVPitch];

  // Row 16 mc + li of the KV head: query head hkv g + h, token t.
  const int row = 16 * mc + li;
  const bool valid = row < a.M;
  const int h = valid ? a.div_t.div(row) : 0, t = valid ? row - h * a.T : 0;
  v8 qop[KK];
  const T* qr = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)(hkv * g + h) * a.q_sh + (int64_t)t * a.q_st;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qop[kk] = tree_load8(qr + 32 * kk + 8 * lg, a.qvec);

  const bool drafted = split == a.S;
  const int n = drafted ? a.T : tree_rows(a, b);
  const int tiles = (n + kTreeTile - 1) / kTreeTile;
  const int per = drafted ? tiles : (tiles + a.S - 1) / a.S;
  const int j_lo = drafted ? 0 : split * per * kTreeTile, j_hi = drafted ? n : min(n, j_lo + per * kTreeTile);
  // Rows past n read as zeros.
  const rsrc_t krs = make_rsrc(static_cast<const T*>(a.kbuf) + (int64_t)bh * a.C * D, (uint32_t)n * kRowBytes);
  const rsrc_t vrs = make_rsrc(static_cast<const T*>(a.vbuf) + (int64_t)bh * a.C * D, (uint32_t)n * kRowBytes);
  const T* kn = static_cast<const T*>(a.kn) + (int64_t)b * a.kn_sb + (int64_t)hkv * a.kn_sh;
  const T* vn = static_cast<const T*>(a.vn) + (int64_t)b * a.vn_sb + (int64_t)hkv * a.vn_sh;
  const uint8_t* mrow = a.mask ? a.mask + (int64_t)b * a.m_sb + (int64_t)t * a.m_st : nullptr;

  const int v_row = lane / CPR, v_col = 8 * (lane % CPR);
  const int tr_row = 4 * lg + li / 4, tr_col = 4 * (li % 4);
  float m = -__FLT_MAX__, lsum = 0.f;  // (finite, so that logits of -inf get no weight)
  f32x4 o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  for (int j0 = j_lo; j0 < j_hi; j0 += kTreeTile) {
    v8 kop[2][KK];
    bool odd = false;  // drafted values that are not finite
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const int j = j0 + 16 * hf + li;
        if (!drafted)
          kop[hf][kk] = bitcast_u4<v8>(buf_load16(krs, (uint32_t)j * kRowBytes + 64u * kk + 16u * lg));
        else if (j < n)
          kop[hf][kk] = tree_load8(kn + (int64_t)j * a.kn_st + 32 * kk + 8 * lg, a.nvec);
        else
          kop[hf][kk] = v8{};
      }
#pragma unroll
    for (int i = 0; i < NVC; ++i) {
      const int j = j0 + v_row + i * GRP;
      v8 x = v8{};
      if (!drafted) {
        x = bitcast_u4<v8>(buf_load16(vrs, (uint32_t)j * kRowBytes + v_col * (uint32_t)sizeof(T)));
      } else if (j < n) {
        x = tree_load8(vn + (int64_t)j * a.vn_st + v_col, a.nvec);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (not_finite<T>(x[e])) {
            odd = true;
            x[e] = static_cast<T>(0.f);
          }
      }
      *reinterpret_cast<v8*>(vt + (v_row + i * GRP) * kVPitch + v_col) = x;
    }
    f32x4 s[2];
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) acc = Elem<T>::mfma(kop[hf][kk], qop[kk], acc);
      s[hf] = acc;
    }
    uint32_t seen = 0;  // bit e: the lane's key e is visible
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int j = j0 + 16 * (e / 4) + 4 * lg + e % 4;
      bool see = j < j_hi;
      if (drafted && see) see = mrow ? mrow[(int64_t)j * a.m_sj] != 0 : j <= t;
      seen |= (uint32_t)see << e;
    }
    float tmax = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (seen >> e) & 1 ? s[e / 4][e % 4] * a.scale_log2 : -INFINITY;
      s[e / 4][e % 4] = x;
      tmax = __builtin_elementwise_maximum(tmax, x);
    }
    const float mnew = fmaxf(m, max_xor32(max_xor16(tmax)));
    const float alpha = __builtin_amdgcn_exp2f(m - mnew);
    float psum = 0.f, pf[8];
    v8 phi, plo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = __builtin_amdgcn_exp2f(s[e / 4][e % 4] - (mnew - kPBias<T>));
      pf[e] = x;
      psum += x;
      phi[e] = static_cast<T>(x);
      plo[e] = static_cast<T>(x - static_cast<float>(phi[e]));
    }
    lsum = lsum * alpha + psum;
    m = mnew;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
    __syncthreads();
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      typedef short s4 __attribute__((ext_vector_type(4)));
      typedef __attribute__((address_space(3))) s4 lds_s4;
      const s4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(vt + tr_row * kVPitch + 16 * dt + tr_col));
      const s4 x1 =
          __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(vt + (16 + tr_row) * kVPitch + 16 * dt + tr_col));
      const v8 aop = __builtin_bit_cast(v8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
      o[dt] = Elem<T>::mfma(aop, phi, o[dt]);
      o[dt] = Elem<T>::mfma(aop, plo, o[dt]);
    }
    __syncthreads();
    if (wave_any(odd)) {
      // A drafted value that is not finite reaches only the rows that see its
      // key: the product above took it as zero (0 * inf is NaN), and here it
      // is added where it is seen.
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll 1
        for (int lgp = 0; lgp < 4; ++lgp) {
          const int j = j0 + 16 * (e / 4) + 4 * lgp + e % 4;
          const float p = __shfl((seen >> e) & 1 ? pf[e] : -1.f, li + 16 * lgp);
          if (j < n && !(p < 0.f))
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                const T x = vn[(int64_t)j * a.vn_st + 16 * dt + 4 * lg + r];
                if (not_finite<T>(x)) o[dt][r] = fmaf(p, static_cast<float>(x), o[dt][r]);
              }
        }
    }
  }

  lsum = add_xor32(add_xor16(lsum));
  const int64_t base = ((int64_t)bh * (a.S + 1) + split) * a.M + row;
  if (valid) {
    float* po = a.part_o + base * D + 4 * lg;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(po + 16 * dt) = o[dt];
    if (lg == 0) {
      a.part_m[base] = m - kPBias<T>;
      a.part_l[base] = lsum;
    }
  }
}

// One wave per row: lane s holds split s's maximum and sum, D / 4 lanes a
// partial output row.
template <typename T, int D>
__global__ void __launch_bounds__(256) tree_merge_kernel(TreeArgs a) {
  constexpr int LPR = D / 4, SPL = 64 / LPR;
  const int S1 = a.S + 1;
  const int wid = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x & 63;
  if (wid >= a.B * a.Hkv * a.M) return;
  const int bh = wid / a.M, row = wid - bh * a.M;
  const int b = bh / a.Hkv, hkv = bh % a.Hkv;
  const int h = a.div_t.div(row), t = row - h * a.T;
  const int sub = lane / LPR, d0 = 4 * (lane % LPR);
  const int64_t base = (int64_t)bh * S1 * a.M + row;
  const float ml = lane < S1 ? a.part_m[base + (int64_t)lane * a.M] : -__FLT_MAX__;
  const float ll = lane < S1 ? a.part_l[base + (int64_t)lane * a.M] : 0.f;
  const float mx = wave_max(ml);
  const float f = __builtin_amdgcn_exp2f(ml - mx);
  const float l = wave_sum(ll * f);
  f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < S1; s += SPL) {
    const float fs = __shfl(f, (s + sub) & 63);
    if (s + sub < S1) {
      const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + (base + (int64_t)(s + sub) * a.M) * D + d0);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = fmaf(fs, x[e], acc[e]);
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

// Splits of the cache for so many (b, KV head, row chunk) pairs.
constexpr int kTreeWaves = 2048;
static int tree_splits(int64_t chunks, int C) {
  const int tiles = (C + kTreeTile - 1) / kTreeTile;
  const int64_t want = std::max<int64_t>(1, kTreeWaves / chunks);
  return (int)std::max<int64_t>(1, std::min<int64_t>({want, kTreeMaxSplits, (tiles + 1) / 2}));
}

struct TreePlan {
  int M, MC, S;
  size_t rows, bytes;
};
static TreePlan tree_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t T, int64_t C) {
  TreePlan p;
  p.M = (int)(Hq / Hkv * T);
  p.MC = (p.M + 15) / 16;
  p.S = tree_splits(B * Hkv * p.MC, (int)C);
  p.rows = (size_t)B * Hkv * (p.S + 1) * p.M;
  p.bytes = p.rows * sizeof(float) * (2 + (size_t)D) + 256;
  return p;
}
size_t tree_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t T, int64_t C) {
  return tree_plan(B, Hq, Hkv, D, T, C).bytes;
}

template <typename T, int D>
static hipError_t launch_tree_t(const TreeArgs& a, hipStream_t st) {
  launch((tree_partial_kernel<T, D>), dim3(a.B * a.Hkv * a.MC * (a.S + 1)), dim3(64), 0, st, a);
  launch((tree_merge_kernel<T, D>), dim3((a.B * a.Hkv * a.M + 3) / 4), dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_tree_attention(const TreeParams& p, hipStream_t st) {
  const TreePlan pl = tree_plan(p.B, p.Hq, p.Hkv, p.D, p.T, p.C);
  TreeArgs a{};
  a.q = p.q;
  a.q_sb = p.q_sb;
  a.q_sh = p.q_sh;
  a.q_st = p.q_st;
  a.kn = p.k_new;
  a.vn = p.v_new;
  a.kn_sb = p.kn_sb;
  a.kn_sh = p.kn_sh;
  a.kn_st = p.kn_st;
  a.vn_sb = p.vn_sb;
  a.vn_sh = p.vn_sh;
  a.vn_st = p.vn_st;
  a.kbuf = p.k_cache;
  a.vbuf = p.v_cache;
  a.n_rows = p.n_rows;
  a.n_sb = p.n_sb;
  a.mask = p.mask;
  a.m_sb = p.m_sb;
  a.m_st = p.m_st;
  a.m_sj = p.m_sj;
  a.B = p.B;
  a.Hq = p.Hq;
  a.Hkv = p.Hkv;
  a.D = p.D;
  a.T = p.T;
  a.C = p.C;
  a.M = pl.M;
  a.MC = pl.MC;
  a.S = pl.S;
  a.div_t = Div::of(p.T);
  a.scale_log2 = p.scale * 1.4426950408889634f;
  auto vec = [](const void* x, int64_t s0, int64_t s1, int64_t s2) {
    return (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && s0 % 8 == 0 && s1 % 8 == 0 && s2 % 8 == 0;
  };
  a.qvec = vec(p.q, p.q_sb, p.q_sh, p.q_st);
  a.nvec = vec(p.k_new, p.kn_sb, p.kn_sh, p.kn_st) && vec(p.v_new, p.vn_sb, p.vn_sh, p.vn_st);
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p.workspace) + 15) & ~(uintptr_t)15);
  a.part_m = reinterpret_cast<float*>(ws);
  a.part_l = a.part_m + pl.rows;
  a.part_o = a.part_m + ((2 * pl.rows + 3) & ~(size_t)3);
  a.out = p.out;
  a.o_sb = p.o_sb;
  a.o_st = p.o_st;
  a.o_sh = p.o_sh;
  if (p.dtype == kDtypeBf16) {
    if (p.D == 64) return launch_tree_t<__bf16, 64>(a, st);
    return launch_tree_t<__bf16, 128>(a, st);
  }
  if (p.D == 64) return launch_tree_t<_Float16, 64>(a, st);
  return launch_tree_t<_Float16, 128>(a, st);
}

// The walk, by one wave per sequence (lane i looks at nodes i, i + 64, ...).
// Nodes are taken in ascending order, so that the walk ends and no node is
// taken twice whatever the parents say.

struct CommitArgs {
  const int64_t* tokens;  // [B, T]
  const int64_t* choice;
  const int* parents;
  int p_sb;  // 0: one tree for every sequence
  int T;
  int* path;  // [B, T]
  int* accepted;
  const uint8_t* kn;  // drafted rows [N, B, H, T, row]: byte strides, units contiguous
  const uint8_t* vn;
  int64_t kn_sn, kn_sb, kn_sh, kn_st, vn_sn, vn_sb, vn_sh, vn_st;
  uint8_t* kbuf;  // [N, B, H, C, row] contiguous
  uint8_t* vbuf;
  const int* n_rows;
  int n_sn, n_sb;
  int B, H, C, units;  // units per row
};

__global__ void __launch_bounds__(64) tree_walk_kernel(CommitArgs a) {
  constexpr int NL = (int)kTreeMaxT / 64;
  const int b = blockIdx.x, lane = threadIdx.x;
  const int64_t* tok = a.tokens + (int64_t)b * a.T;
  const int64_t* cho = a.choice + (int64_t)b * a.T;
  const int* par = a.parents + (int64_t)b * a.p_sb;
  int parent[NL];  // of nodes whose token is their parent's choice; -1 otherwise
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int c = lane + 64 * i;
    parent[i] = -1;
    if (c > 0 && c < a.T) {
      const int p = par[c];
      if (p >= 0 && p < c && tok[c] == cho[p]) parent[i] = p;
    }
  }
  int* path = a.path + (int64_t)b * a.T;
  int cur = 0, len = 0;
  while (cur >= 0) {
    if (lane == 0) path[len] = cur;
    ++len;
    int next = -1;
#pragma unroll
    for (int i = NL - 1; i >= 0; --i) {
      const uint64_t hit = __builtin_amdgcn_ballot_w64(parent[i] == cur);  // (children only: parents lie below)
      if (hit) next = 64 * i + __builtin_ctzll(hit);
    }
    cur = next;
  }
  for (int i = len + lane; i < a.T; i += 64) path[i] = -1;
  if (lane == 0) a.accepted[b] = len;
}

// One workgroup per (layer, sequence, head): the path's rows, K then V.
template <typename U>
__global__ void __launch_bounds__(256) tree_commit_kernel(CommitArgs a) {
  const int h = blockIdx.x % a.H, b = (blockIdx.x / a.H) % a.B, l = blockIdx.x / (a.H * a.B);
  const int n = a.n_rows[(int64_t)l * a.n_sn + (int64_t)b * a.n_sb];
  const int len = a.accepted[b];
  if (n < 0) return;
  const int fit = min(len, a.C - n);  // (rows past the capacity are not stored)
  const int64_t dst = (((int64_t)l * a.B + b) * a.H + h) * a.C * a.units;
  const int* path = a.path + (int64_t)b * a.T;
  for (int x = threadIdx.x; x < 2 * fit * a.units; x += 256) {
    const int v = x >= fit * a.units, y = x - v * fit * a.units;
    const int i = y / a.units, u = y - i * a.units, node = path[i];
    const uint8_t* src = v ? a.vn + (int64_t)l * a.vn_sn + (int64_t)b * a.vn_sb + (int64_t)h * a.vn_sh + (int64_t)node * a.vn_st
                           : a.kn + (int64_t)l * a.kn_sn + (int64_t)b * a.kn_sb + (int64_t)h * a.kn_sh + (int64_t)node * a.kn_st;
    reinterpret_cast<U*>(v ? a.vbuf : a.kbuf)[dst + (int64_t)(n + i) * a.units + u] = reinterpret_cast<const U*>(src)[u];
  }
}

hipError_t launch_tree_commit(const CommitParams& p, hipStream_t st) {
  CommitArgs a{};
  a.tokens = p.tokens;
  a.choice = p.choice;
  a.parents = p.parents;
  a.p_sb = p.p_sb;
  a.T = p.T;
  a.path = p.path;
  a.accepted = p.accepted;
  const int64_t eb = p.elem_bytes;
  a.kn = static_cast<const uint8_t*>(p.k_new);
  a.vn = static_cast<const uint8_t*>(p.v_new);
  a.kn_sn = p.kn_sn * eb;
  a.kn_sb = p.kn_sb * eb;
  a.kn_sh = p.kn_sh * eb;
  a.kn_st = p.kn_st * eb;
  a.vn_sn = p.vn_sn * eb;
  a.vn_sb = p.vn_sb * eb;
  a.vn_sh = p.vn_sh * eb;
  a.vn_st = p.vn_st * eb;
  a.kbuf = static_cast<uint8_t*>(p.k_cache);
  a.vbuf = static_cast<uint8_t*>(p.v_cache);
  a.n_rows = p.n_rows;
  a.n_sn = p.n_sn;
  a.n_sb = p.n_sb;
  a.B = p.B;
  a.H = p.H;
  a.C = p.C;
  launch(tree_walk_kernel, dim3(p.B), dim3(64), 0, st, a);
  const int64_t all = (int64_t)reinterpret_cast<uintptr_t>(a.kn) | (int64_t)reinterpret_cast<uintptr_t>(a.vn) |
                      (int64_t)reinterpret_cast<uintptr_t>(a.kbuf) | (int64_t)reinterpret_cast<uintptr_t>(a.vbuf) |
                      a.kn_sn | a.kn_sb | a.kn_sh | a.kn_st | a.vn_sn | a.vn_sb | a.vn_sh | a.vn_st | (p.D * eb);
  const dim3 grid((unsigned)(p.N * p.B * p.H));
  if (all % 16 == 0) {
    a.units = (int)(p.D * eb / 16);
    launch(tree_commit_kernel<u32x4>, grid, dim3(256), 0, st, a);
  } else if (eb == 4) {
    a.units = p.D;
    launch(tree_commit_kernel<uint32_t>, grid, dim3(256), 0, st, a);
  } else {
    a.units = p.D;
    launch(tree_commit_kernel<uint16_t>, grid, dim3(256), 0, st, a);
  }
  return hipGetLastError();
}

}  // namespace dkv
