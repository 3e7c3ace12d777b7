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
#include "dkv_tree_dev.h"

#include <algorithm>
#include <cmath>

namespace dkv {

// P in the element type.  fp16 keeps it 2^14 times larger: its smallest number
// is 2^-24, and a long cache holds many keys whose weight against the running
// maximum is below that (the factor goes into the reference of the exponent and
// cancels in the quotient).
template <typename T>
constexpr float kPBias = 0.f;
template <>
constexpr float kPBias<_Float16> = 14.f;

// The wide kernel lets a row's maximum rise so far above the reference that its
// weights are taken against (powers of two) before it moves the reference and
// turns what it has summed: P is at most 2^8 in bf16, and 2^15 with the bias in
// fp16, whose largest number is just below 2^16.  (Moving it at every new maximum
// turned two stages of three over 26214 keys in 4 parts, one vector
// instruction in six: 255 and 248 us where this takes 248 and 243.  The largest
// weight is then no exact 1 and is rounded like the others, in the sum as in the
// product: there the error against 64 bits is 0.0023, not 0.0021, of the output.)
template <typename T>
constexpr float kPRise = 8.f;
template <>
constexpr float kPRise<_Float16> = 1.f;

// Beyond 2^22 (in powers of two) a scaled logit's fraction is lost, and the scaled
// maximum, rounded, may lie below the logit it stands for by more than P has room
// for: the weights are then taken from differences of the logits themselves
// (exact where they are near) and scaled after.  Below, by one fma.
constexpr float kTreeFar = 4194304.f;

// Up to 16 rows per KV head: one wave per part, its own tiles.  K comes in
// registers as the matrix operand, V through LDS for the transposing reads; the
// next tile's loads are issued as soon as a tile's registers are consumed.
// Bound by memory: 4 x 16 heads of 6553 rows, D = 64 (107 MB) take 19 to 20 us (5.4
// TB/s) and 25 with the join.  P goes into the product in two parts, rounded and
// remainder (the matrix cores have room here), so that the result is off by its
// own rounding alone.
template <typename T, int D>
__global__ void __launch_bounds__(64) tree_partial_kernel(TreeArgs a) {
  typedef typename Elem<T>::v8 v8;
  constexpr int KK = D / 32, DT = D / 16, CPR = D / 8, GRP = 64 / CPR, NVC = kTreeTile / GRP;
  constexpr int kVPitch = D + 16;  // transposing reads without bank conflicts
  constexpr uint32_t kRowBytes = D * (uint32_t)sizeof(T);
  const int slot = blockIdx.x % a.P, hkv = blockIdx.x / a.P, g = a.Hq / a.Hkv;
  const int lane = threadIdx.x, li = lane & 15, lg = lane >> 4;
  __shared__ __attribute__((aligned(16))) T vt[kTreeTile * kVPitch];
  __shared__ uint64_t mask_words[16];  // (T <= 16 rows)

  const TreePart part = tree_part(a, hkv, slot, lane);
  const int b = part.b, n = part.n;
  if (b < 0) return;
  const int bh = b * a.Hkv + hkv;
  // Rows past n read as zeros.
  const rsrc_t krs = make_rsrc(static_cast<const T*>(a.kbuf) + (int64_t)bh * a.C * D, (uint32_t)n * kRowBytes);
  const rsrc_t vrs = make_rsrc(static_cast<const T*>(a.vbuf) + (int64_t)bh * a.C * D, (uint32_t)n * kRowBytes);
  const int v_row = lane / CPR, v_col = 8 * (lane % CPR);
  const int tr_row = 4 * lg + li / 4, tr_col = 4 * (li % 4);
  v8 kop[2][KK], vch[NVC];
  auto load_k = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf)
#pragma unroll
      for (int kk = 0; kk < KK; ++kk)
        kop[hf][kk] = bitcast_u4<v8>(buf_load16(krs, (uint32_t)(j0 + 16 * hf + li) * kRowBytes + 64u * kk + 16u * lg));
  };
  auto load_v = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NVC; ++i)
      vch[i] = bitcast_u4<v8>(
          buf_load16(vrs, (uint32_t)(j0 + v_row + i * GRP) * kRowBytes + v_col * (uint32_t)sizeof(T)));
  };
  int j0 = part.t_lo * kTreeTile;
  const int j_hi = min(n, part.t_hi * kTreeTile);
  if (j0 < j_hi) {
    load_k(j0);
    load_v(j0);
  }

  // Row li of the KV head: query head hkv g + h, token t.
  const int row = li;
  const bool valid = row < a.M;
  const int h = valid ? a.div_t.div(row) : 0, t = valid ? row - h * a.T : 0;
  v8 qop[KK];
  const T* qr = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)(hkv * g + h) * a.q_sh + (int64_t)t * a.q_st;
#pragma unroll
  for (int kk = 0; kk < KK; ++kk) qop[kk] = tree_load8(qr + 32 * kk + 8 * lg);

  // The running maximum of the logits, and times the scale (that one finite, so
  // that logits of -inf get no weight).
  float raw = -INFINITY, m = -__FLT_MAX__, lsum = 0.f;
  bool far = false;  // (of any of the wave's rows)
  f32x4 s[2], o[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};

  auto logits = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) acc = Elem<T>::mfma(kop[hf][kk], qop[kk], acc);
      s[hf] = acc;
    }
  };
  auto put_v = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NVC; ++i) *reinterpret_cast<v8*>(vt + (v_row + i * GRP) * kVPitch + v_col) = vch[i];
  };
  // Softmax step and O^T += V^T P^T; bit e of `seen`: the lane's key e counts.
  auto attend = [&](uint32_t seen) __attribute__((always_inline)) {
    float tmax = -INFINITY;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = (seen >> e) & 1 ? s[e / 4][e % 4] : -INFINITY;
      s[e / 4][e % 4] = x;
      tmax = __builtin_elementwise_maximum(tmax, x);
    }
    tmax = max_xor32(max_xor16(tmax));
    const bool turn = tmax > raw;
    float ref = m - kPBias<T>;
    if (wave_any(turn) || far) {
      const float mnew = turn ? fmaxf(tmax * a.scale_log2, -__FLT_MAX__) : m;
      const float by = fabsf(mnew) < kTreeFar ? m - mnew : (raw - tmax) * a.scale_log2;
      const float alpha = turn ? __builtin_amdgcn_exp2f(by) : 1.f;
      lsum *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
      m = mnew;
      raw = turn ? tmax : raw;
      ref = m - kPBias<T>;
      far = wave_any(fabsf(m) >= kTreeFar);
      if (far) {
        ref = -kPBias<T>;
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e / 4][e % 4] -= fmaxf(raw, -__FLT_MAX__);
      }
    }
    float psum = 0.f;
    v8 phi, plo;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float x = __builtin_amdgcn_exp2f(fmaf(s[e / 4][e % 4], a.scale_log2, -ref));
      psum += x;
      phi[e] = static_cast<T>(x);
      plo[e] = static_cast<T>(x - static_cast<float>(phi[e]));
    }
    lsum += psum;
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
  };

  // (One wave: its own LDS operations stay in order.)
  for (; j0 + kTreeTile <= j_hi; j0 += kTreeTile) {
    logits();
    load_k(j0 + kTreeTile);
    put_v();
    load_v(j0 + kTreeTile);
    attend(0xff);
  }
  // A last tile of the cache, and the drafted keys (T <= 16: one tile), through
  // the same code: what a short call fetches of it counts.
  bool stored = j0 < j_hi, drafted = part.tail, odd = false;
#pragma unroll 1
  while (stored || drafted) {
    uint32_t seen;
    if (stored) {
      seen = tree_first_bits(j_hi - j0, lg);
    } else {
      const T* kn = static_cast<const T*>(a.kn) + (int64_t)b * a.kn_sb + (int64_t)hkv * a.kn_sh;
      const T* vn = static_cast<const T*>(a.vn) + (int64_t)b * a.vn_sb + (int64_t)hkv * a.vn_sh;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        kop[0][kk] = tree_load8(kn + (int64_t)min(li, a.T - 1) * a.kn_st + 32 * kk + 8 * lg);
        kop[1][kk] = v8{};
      }
#pragma unroll
      for (int i = 0; i < NVC; ++i) {
        vch[i] = tree_load8(vn + (int64_t)min(v_row + i * GRP, a.T - 1) * a.vn_st + v_col);
      }
      tree_mask_words<1>(a, b, 0, 0, lane, mask_words);
#pragma unroll
      for (int i = 0; i < NVC; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (v_row + i * GRP >= a.T) {
            vch[i][e] = static_cast<T>(0.f);
          } else if (not_finite<T>(vch[i][e])) {
            odd = true;
            vch[i][e] = static_cast<T>(0.f);
          }
      seen = tree_key_bits((uint32_t)(mask_words[t] >> (4 * lg)));
      drafted = false;
    }
    stored = false;
    logits();
    put_v();
    attend(seen);
  }

  lsum = add_xor32(add_xor16(lsum));
  const int64_t base = ((int64_t)hkv * a.P + slot) * a.M + row;
  if (valid) {
    float* po = a.part_o + base * D + 4 * lg;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(po + 16 * dt) = o[dt];
    if (lg == 0) {
      a.part_m[base] = m - kPBias<T>;
      a.part_l[base] = lsum;
    }
  }
  if (__builtin_expect(wave_any(odd), 0)) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    tree_add_odd<T, D, 64>(a, b, hkv, slot, 0, 16);
  }
}

// With LO, P goes into the product in two parts, rounded and remainder (about 16
// significant bits).  In workgroups of 128 rows and more a call is bound by the
// matrix cores and the ALUs and not by memory, and P is rounded once: each weight
// is off by at most half a step of the element type, as the output is by its own
// rounding (4 x 64 heads of 26214 rows, 64 tokens: 333 us in two parts, 246 in
// one, 890 TFLOP/s; 8 x 32 heads of up to 8003 rows, 27 tokens: 58 and 48.5, of
// which 42 are this kernel's, 3.6 TB/s).  What bounds the one: matrix cores busy 49%
// of the time and vector units 46%, hardly ever together, with two waves on a
// SIMD; wave priorities, waves of 64 rows (388 us), and the next stage's products
// with K beside a stage's softmax (248) did not help.
//
// More than 16 rows: NW waves of QB blocks of 16 rows (4 of one or two, 8 of two)
// take the same keys, so
// that a tile of K and V is read once for all of them, into LDS.  The next tile
// is on its way in registers while the waves compute on this one, and goes to
// the other of two buffers: one barrier per tile.  A K operand (a V operand)
// read from LDS serves QB products.  LDS pitches leave every 16 lanes of a
// K read, and every 32 of a transposing V read, on banks of their own.
template <typename T, int D, int QB, int NW, bool LO>
__global__ void __launch_bounds__(64 * NW, 2) tree_wide_kernel(TreeArgs a) {
  typedef typename Elem<T>::v8 v8;
  constexpr int KK = D / 32, DT = D / 16, CPR = D / 8, NT = 64 * NW;
  constexpr int kSub = 2, kStage = kSub * kTreeTile;
  constexpr int kChunks = kStage * CPR;         // 16-byte pieces of a stage's K (or V)
  constexpr int NC = 2 * kChunks / NT;          // pieces per thread
  constexpr int kKP = D + 8, kVP = D + 16, kBuf = kStage * (kKP + kVP);
  constexpr uint32_t kRowBytes = D * (uint32_t)sizeof(T);
  static_assert(NC * NT == 2 * kChunks, "whole pieces per thread");
  __shared__ __attribute__((aligned(16))) T lds[2 * kBuf];
  __shared__ int odd_flag;

  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int mc = id % a.MC, slot = (id / a.MC) % a.P, hkv = id / (a.MC * a.P), g = a.Hq / a.Hkv;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const TreePart part = tree_part(a, hkv, slot, lane);
  const int b = part.b, n = part.n;
  if (b < 0) return;
  const int bh = b * a.Hkv + hkv;
  const int row0 = (mc * NW + wave) * (16 * QB) + li;  // the lane's row of block 0

  v8 qop[QB][KK];
  int tq[QB];
#pragma unroll
  for (int x = 0; x < QB; ++x) {
    const int row = min(row0 + 16 * x, a.M - 1);  // (rows past the last repeat it and are not stored)
    const int h = a.div_t.div(row), t = row - h * a.T;
    tq[x] = t;
    const T* qr =
        static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)(hkv * g + h) * a.q_sh + (int64_t)t * a.q_st;
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) qop[x][kk] = tree_load8(qr + 32 * kk + 8 * lg);
  }

  // Rows past n read as zeros.
  const rsrc_t krs = make_rsrc(static_cast<const T*>(a.kbuf) + (int64_t)bh * a.C * D, (uint32_t)n * kRowBytes);
  const rsrc_t vrs = make_rsrc(static_cast<const T*>(a.vbuf) + (int64_t)bh * a.C * D, (uint32_t)n * kRowBytes);
  const T* kn = static_cast<const T*>(a.kn) + (int64_t)b * a.kn_sb + (int64_t)hkv * a.kn_sh;
  const T* vn = static_cast<const T*>(a.vn) + (int64_t)b * a.vn_sb + (int64_t)hkv * a.vn_sh;

  u32x4 piece[NC];
  auto place = [&](int i, int* row, int* col) __attribute__((always_inline)) {  // piece i: K or V, its row and column
    const int c = tid + i * NT, v = c >= kChunks;
    *row = (c - v * kChunks) / CPR;
    *col = 8 * (c % CPR);
    return v != 0;
  };
  auto fetch = [&](int j0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      int r, col;
      const bool v = place(i, &r, &col);
      piece[i] = buf_load16(v ? vrs : krs, (uint32_t)(j0 + r) * kRowBytes + col * (uint32_t)sizeof(T));
    }
  };
  auto put = [&](int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      int r, col;
      const bool v = place(i, &r, &col);
      *reinterpret_cast<u32x4*>(lds + buf * kBuf + (v ? kStage * kKP + r * kVP : r * kKP) + col) = piece[i];
    }
  };

  v8 ones;
#pragma unroll
  for (int e = 0; e < 8; ++e) ones[e] = static_cast<T>(1.f);
  // The reference of the weights, and times the scale (that one finite, so that
  // logits of -inf get no weight).
  float raw[QB], m[QB];
  bool far = false;           // (of any of the wave's rows)
  f32x4 lsum[QB], o[QB][DT];  // (each of lsum's values is the whole sum of row li)
#pragma unroll
  for (int x = 0; x < QB; ++x) {
    raw[x] = -INFINITY;
    m[x] = -__FLT_MAX__;
    lsum[x] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[x][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const int tr_row = 4 * lg + li / 4, tr_col = 4 * (li % 4);

  uint32_t see_bits[QB];  // bit 8 sub + e: the lane's key e of the stage's tile sub counts
  __shared__ uint64_t mask_words[kTreeMaxT];
  // The stage in buffer `buf`; with `masked` the keys of see_bits.
  auto compute = [&](int buf, auto masked) __attribute__((always_inline)) {
    constexpr bool kMasked = decltype(masked)::value;
    const T* kt = lds + buf * kBuf;
    const T* vt = kt + kStage * kKP;
    f32x4 s[QB][2 * kSub];  // keys 16 i + 4 lg + r
#pragma unroll
    for (int i = 0; i < 2 * kSub; ++i) {
#pragma unroll
      for (int x = 0; x < QB; ++x) s[x][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) {
        const v8 kop = *reinterpret_cast<const v8*>(kt + (16 * i + li) * kKP + 32 * kk + 8 * lg);
#pragma unroll
        for (int x = 0; x < QB; ++x) s[x][i] = Elem<T>::mfma(kop, qop[x][kk], s[x][i]);
      }
    }
    float top[QB], ref[QB];
    bool turn = false;
#pragma unroll
    for (int x = 0; x < QB; ++x) {
      if (kMasked) {
#pragma unroll
        for (int e = 0; e < 8 * kSub; ++e)
          s[x][e / 4][e % 4] = (see_bits[x] >> e) & 1 ? s[x][e / 4][e % 4] : -INFINITY;
      }
      float tmax = s[x][0][0];
#pragma unroll
      for (int e = 1; e < 8 * kSub; ++e) tmax = __builtin_elementwise_maximum(tmax, s[x][e / 4][e % 4]);
      top[x] = maximum_xor32(maximum_xor16(tmax));
      turn |= (top[x] - raw[x]) * a.scale_log2 > kPRise<T>;
      ref[x] = m[x] - kPBias<T>;
    }
    if (wave_any(turn) || far) {
      bool beyond = false;
#pragma unroll
      for (int x = 0; x < QB; ++x) {
        const float rise = (top[x] - raw[x]) * a.scale_log2;
        const bool up = rise > kPRise<T>;
        const float mnew = up ? fmaxf(top[x] * a.scale_log2, -__FLT_MAX__) : m[x];
        const float alpha = up ? __builtin_amdgcn_exp2f(fabsf(mnew) < kTreeFar ? m[x] - mnew : -rise) : 1.f;
        lsum[x] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= alpha;
        m[x] = mnew;
        raw[x] = up ? top[x] : raw[x];
        ref[x] = m[x] - kPBias<T>;
        beyond |= fabsf(m[x]) >= kTreeFar;
      }
      far = wave_any(beyond);
      if (far) {
#pragma unroll
        for (int x = 0; x < QB; ++x) {
          ref[x] = -kPBias<T>;
#pragma unroll
          for (int e = 0; e < 8 * kSub; ++e) s[x][e / 4][e % 4] -= fmaxf(raw[x], -__FLT_MAX__);
        }
      }
    }
#pragma unroll
    for (int sub = 0; sub < kSub; ++sub) {
      v8 phi[QB], plo[LO ? QB : 1];
#pragma unroll
      for (int x = 0; x < QB; ++x)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[x][2 * sub + e / 4][e % 4], a.scale_log2, -ref[x]));
          phi[x][e] = static_cast<T>(p);
          if (LO) plo[x][e] = static_cast<T>(p - static_cast<float>(phi[x][e]));
        }
      // The weights' sum as one more product, with ones.
#pragma unroll
      for (int x = 0; x < QB; ++x) {
        lsum[x] = Elem<T>::mfma(ones, phi[x], lsum[x]);
        if (LO) lsum[x] = Elem<T>::mfma(ones, plo[x], lsum[x]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        typedef short s4 __attribute__((ext_vector_type(4)));
        typedef __attribute__((address_space(3))) s4 lds_s4;
        const T* vs = vt + (kTreeTile * sub + tr_row) * kVP + 16 * dt + tr_col;
        const s4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)vs);
        const s4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(vs + 16 * kVP));
        const v8 aop = __builtin_bit_cast(v8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
        for (int x = 0; x < QB; ++x) {
          o[x][dt] = Elem<T>::mfma(aop, phi[x], o[x][dt]);
          if (LO) o[x][dt] = Elem<T>::mfma(aop, plo[x], o[x][dt]);
        }
      }
    }
  };

  if (tid == 0) odd_flag = 0;
  int buf = 0;
  const int j_hi = min(n, part.t_hi * kTreeTile);
  int j0 = part.t_lo * kTreeTile;
  bool stored = j0 < j_hi;
  if (stored) {
    fetch(j0);
    put(0);
    for (; j0 + kStage < j_hi; j0 += kStage) {
      fetch(j0 + kStage);
      __syncthreads();
      compute(buf, std::false_type{});
      buf ^= 1;
      put(buf);
    }
  }
  // The cache's last stage, and the drafted keys, through the same code: what a
  // short call fetches of it counts (with three copies of the stage and the
  // drafted keys' rare cases in line the drafted keys of 8 tokens took 6.0 us, not
  // 4.5).
#pragma unroll 1
  for (int jd = part.tail ? 0 : a.T; stored || jd < a.T;) {
    if (stored) {
      __syncthreads();
#pragma unroll
      for (int x = 0; x < QB; ++x)
        see_bits[x] = tree_first_bits(j_hi - j0, lg) | tree_first_bits(j_hi - j0 - kTreeTile, lg) << 8;
      stored = false;
    } else {
      __syncthreads();  // (the words' and the buffer's last readers are done)
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        int r, col;
        const bool v = place(i, &r, &col);
        const int j = min(jd + r, a.T - 1);
        piece[i] = __builtin_bit_cast(u32x4, tree_load8((v ? vn + (int64_t)j * a.vn_st : kn + (int64_t)j * a.kn_st) + col));
      }
      tree_mask_words<NW>(a, b, jd, wave, lane, mask_words);
      bool odd = false;
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        int r, col;
        const bool v = place(i, &r, &col);
        if (jd + r >= a.T) piece[i] = u32x4{0u, 0u, 0u, 0u};
        if (v) {
          v8 x = bitcast_u4<v8>(piece[i]);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (not_finite<T>(x[e])) {
              odd = true;
              x[e] = static_cast<T>(0.f);
            }
          piece[i] = __builtin_bit_cast(u32x4, x);
        }
      }
      put(buf);
      if (odd) odd_flag = 1;
      __syncthreads();
#pragma unroll
      for (int x = 0; x < QB; ++x) {
        const uint64_t w = mask_words[tq[x]] >> (4 * lg);
        see_bits[x] = tree_key_bits((uint32_t)w) | tree_key_bits((uint32_t)(w >> 32)) << 8;
      }
      jd += kStage;
    }
    compute(buf, std::true_type{});
    buf ^= 1;
  }

#pragma unroll
  for (int x = 0; x < QB; ++x) {
    const int row = row0 + 16 * x;
    const float l = lsum[x][0];
    if (row >= a.M) continue;
    if (a.direct) {
      const int h = a.div_t.div(row), t = row - h * a.T;
      T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)t * a.o_st + (int64_t)(hkv * g + h) * a.o_sh;
      const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          out[16 * dt + 4 * lg + r] = static_cast<T>(l == 0.f ? 0.f : o[x][dt][r] * inv);
      continue;
    }
    const int64_t base = ((int64_t)hkv * a.P + slot) * a.M + row;
    const rsrc_t prs = make_rsrc(a.part_o + (base - 16 * x - li) * D, (16 * x + 16) * D * 4u);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) st_dev16(prs, ((16 * x + li) * D + 16 * dt + 4 * lg) * 4u, o[x][dt]);
    if (lg == 0) {
      st_dev(a.part_m + base, m[x] - kPBias<T>);
      st_dev(a.part_l + base, l);
    }
  }
  if (part.tail && __builtin_expect(odd_flag != 0, 0)) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    tree_add_odd<T, D, NT>(a, b, hkv, slot, mc * NW * 16 * QB, NW * 16 * QB);
  }
}

// How a call is cut: rows per workgroup (16: one wave), parts of the cache per
// sequence, and whether the drafted keys are parts of their own.
struct TreePlan {
  int M, rows_wg, MC, S, P, apart;
  size_t rows, bytes;
};

// An estimate of a call's time in us, from sweeps of both over calls of 1 to 1024
// rows per KV head, 900 to 100,000 keys and 2 to 256 heads (the plan chosen by it
// took up to a tenth longer than the best one there).  The sum of
// - the longest workgroup's tiles, a tile's time by the rows, 0.65 of it at D =
//   64, and longer where two workgroups share a CU or take turns;
//   or, if longer, K and V at 5.2 TB/s, where 8 MB or a quarter of them are in
//   flight;
// - the partial rows, written and read at 4 TB/s, and a round trip of the joining
//   kernel for every 16 (D = 128) or 32 parts;
// - the two kernels' fixed part.
struct TreeShape {
  int rows;
  double tile_us, fixed_us, shared;  // shared: two workgroups on a CU, against one
  int per_cu;
};
constexpr TreeShape kTreeShapes[] = {
    {16, 0.50, 6.5, 1.0, 8}, {64, 0.60, 7.0, 1.45, 2}, {128, 0.72, 7.2, 1.7, 2}, {256, 1.10, 8.5, 1.0, 1}};

static double tree_cost(const TreeShape& w, double heads, double M, double D, double tiles, int64_t S) {
  const double wgs = heads * std::ceil(M / w.rows) * S, wide = D / 128;
  const double per = std::ceil(tiles / S), load = wgs / (256.0 * w.per_cu);
  double tile = w.tile_us * (wide < 1 ? 0.65 : 1);
  if (load > 1)
    tile *= std::ceil(load) * w.shared;
  else if (w.per_cu == 2 && load > 0.5)
    tile *= w.shared;
  const double flight = std::min(wgs, 256.0 * w.per_cu) * (w.rows == 16 ? 16384 : 32768) * wide;
  const double bytes = heads * tiles * kTreeTile * D * 4;
  const double stream = bytes / 5.2e6 / std::min(1.0, flight / std::max(1.0, std::min(8e6, bytes / 4)));
  return std::max(per * tile, stream) + S * heads * M * D * 8 / 4e6 + 0.6 * std::ceil((S + 1) * wide / 16) + w.fixed_us;
}

static TreePlan tree_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t T, int64_t C) {
  TreePlan p;
  p.M = (int)(Hq / Hkv * T);
  const int64_t heads = B * Hkv, tiles = (C + kTreeTile - 1) / kTreeTile;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kTreeMaxSplits, (tiles + 1) / 2));
  double best = 0;
  p.S = 0;
  for (const TreeShape& w : kTreeShapes) {
    // One wave for up to 16 rows; no shape that the rows would leave half empty.
    if ((w.rows == 16) != (p.M <= 16) || (w.rows > 64 && p.M <= w.rows / 2)) continue;
    const int64_t chunks = heads * ((p.M + w.rows - 1) / w.rows);
    const int64_t tries[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, kTreeMaxSplits, 256 / chunks, 512 / chunks};
    for (int64_t S : tries) {
      S = std::max<int64_t>(1, std::min(S, most));
      const double cost = tree_cost(w, (double)heads, p.M, (double)D, (double)tiles, S);
      if (p.S == 0 || cost < best) {
        best = cost;
        p.S = (int)S;
        p.rows_wg = w.rows;
      }
    }
  }
  p.MC = (p.M + p.rows_wg - 1) / p.rows_wg;
  p.apart = p.rows_wg <= 64 || heads * p.MC * p.S < 192;
  p.P = (int)(B * (p.S + p.apart));
  p.rows = (size_t)Hkv * p.P * p.M;
  p.bytes = kSyncBytes + kTreeDealBytes + p.rows * sizeof(float) * (2 + (size_t)D) + 256;
  return p;
}
size_t tree_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t T, int64_t C) {
  return tree_plan(B, Hq, Hkv, D, T, C).bytes;
}

template <typename T, int D>
static hipError_t launch_tree_t(const TreeArgs& a, int rows_wg, hipStream_t st) {
  const dim3 grid(a.Hkv * a.P * a.MC);
  if (rows_wg == 16)
    launch((tree_partial_kernel<T, D>), grid, dim3(64), 0, st, a);
  else if (rows_wg == 64)
    launch((tree_wide_kernel<T, D, 1, 4, true>), grid, dim3(256), 0, st, a);
  else if (rows_wg == 128)
    launch((tree_wide_kernel<T, D, 2, 4, false>), grid, dim3(256), 0, st, a);
  else
    launch((tree_wide_kernel<T, D, 2, 8, false>), grid, dim3(512), 0, st, a);
  if (!a.direct) launch((tree_merge_kernel<T, D>), dim3((a.B * a.Hkv * a.M + 3) / 4), dim3(256), 0, st, a);
  return hipGetLastError();
}

hipError_t launch_tree_attention(const dropkv_tree_attention_args& p, size_t* need, hipStream_t st) {
  const TreePlan pl = tree_plan(p.B, p.Hq, p.Hkv, p.D, p.T, p.capacity);
  *need = pl.bytes;
  if (p.workspace_bytes < 0 || (size_t)p.workspace_bytes < pl.bytes) return hipSuccess;  // (the caller says so)
  TreeArgs a{};
  a.q = p.q;
  a.q_sb = p.q_s[0];
  a.q_sh = p.q_s[1];
  a.q_st = p.q_s[2];
  a.kn = p.k_new;
  a.vn = p.v_new;
  a.kn_sb = p.kn_s[0];
  a.kn_sh = p.kn_s[1];
  a.kn_st = p.kn_s[2];
  a.vn_sb = p.vn_s[0];
  a.vn_sh = p.vn_s[1];
  a.vn_st = p.vn_s[2];
  a.kbuf = p.k_cache;
  a.vbuf = p.v_cache;
  a.n_rows = p.n_rows;
  a.n_sb = (int)p.n_sb;
  a.mask = static_cast<const uint8_t*>(p.mask);
  a.m_sb = p.m_s[0];
  a.m_st = p.m_s[1];
  a.m_sj = p.m_s[2];
  a.B = (int)p.B;
  a.Hq = (int)p.Hq;
  a.Hkv = (int)p.Hkv;
  a.D = (int)p.D;
  a.T = (int)p.T;
  a.C = (int)p.capacity;
  a.M = pl.M;
  a.MC = pl.MC;
  a.S = pl.S;
  a.P = pl.P;
  a.apart = pl.apart;
  a.tail_tiles = pl.apart ? 0 : 3 + 2 * ((a.T + kTreeTile - 1) / kTreeTile);
  a.ragged = p.n_sb != 0 && p.B > 1 && p.B <= kTreeRaggedB && pl.S > 1;
  a.direct = pl.S == 1 && !pl.apart;
  a.div_t = Div::of(a.T);
  a.scale_log2 = (float)p.scale * 1.4426950408889634f;
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p.workspace) + 15) & ~(uintptr_t)15);
  a.deal = reinterpret_cast<int*>(ws + kSyncBytes);
  a.part_m = reinterpret_cast<float*>(ws + kSyncBytes + kTreeDealBytes);
  a.part_l = a.part_m + pl.rows;
  a.part_o = a.part_m + ((2 * pl.rows + 3) & ~(size_t)3);
  a.out = p.out;
  a.o_sb = p.o_s[0];
  a.o_st = p.o_s[1];
  a.o_sh = p.o_s[2];
  if (p.dtype == kDtypeBf16) {
    if (p.D == 64) return launch_tree_t<__bf16, 64>(a, pl.rows_wg, st);
    return launch_tree_t<__bf16, 128>(a, pl.rows_wg, st);
  }
  if (p.D == 64) return launch_tree_t<_Float16, 64>(a, pl.rows_wg, st);
  return launch_tree_t<_Float16, 128>(a, pl.rows_wg, st);
}

// Accepted rows: one workgroup per (layer, sequence, head).  Each walks its tree
// by itself, a few hundred cycles for usual depths, so that one launch does (two
// took 13 us of host and GPU time a call, this one 10; its kernel takes 3.5 us for
// 24 layers' 2 heads and 6.3 for 32 x 8 x 8 heads of 64 tokens).
struct CommitArgs {
  const int64_t* tokens;  // [B, T]
  const int64_t* choice;
  const int* parents;
  int64_t p_sb;  // 0: one tree for every sequence
  int T;
  int* path;  // [B, T]
  int* accepted;
  const uint8_t* kn;  // drafted rows [N, B, H, T, row]: byte strides, units contiguous
  const uint8_t* vn;
  int64_t kn_sn, kn_sb, kn_sh, kn_st, vn_sn, vn_sb, vn_sh, vn_st;
  uint8_t* kbuf;  // [N, B, H, C, row] contiguous
  uint8_t* vbuf;
  const int* n_rows;
  int64_t n_sn, n_sb;
  int B, H, C, units;  // units per row
};

// The walk, by one wave (lane i looks at nodes i, i + 64, ...); the number of
// nodes.  Nodes are taken in ascending order, so that the walk ends and no node
// is taken twice whatever the parents say.
__device__ __forceinline__ int tree_walk(const CommitArgs& a, int b, int lane, int* path) {
  constexpr int NL = (int)kTreeMaxT / 64;
  const int64_t* tok = a.tokens + (int64_t)b * a.T;
  const int64_t* cho = a.choice + (int64_t)b * a.T;
  const int* par = a.parents + b * a.p_sb;
  int parent[NL];  // of nodes whose token is their parent's choice; -1 otherwise
  int64_t token[NL];
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int c = min(lane + 64 * i, a.T - 1);
    parent[i] = par[c];
    token[i] = tok[c];
  }
#pragma unroll
  for (int i = 0; i < NL; ++i) {
    const int c = lane + 64 * i, p = parent[i];
    const bool child = c > 0 && c < a.T && p >= 0 && p < c;
    if (!child || token[i] != cho[child ? p : 0]) parent[i] = -1;
  }
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
  return len;
}

// The path's rows, K then V.
template <typename U>
__global__ void __launch_bounds__(256) tree_commit_kernel(CommitArgs a) {
  __shared__ int path[kTreeMaxT];
  __shared__ int length;
  const int h = blockIdx.x % a.H, b = (blockIdx.x / a.H) % a.B, l = blockIdx.x / (a.H * a.B);
  const int n = a.n_rows[l * a.n_sn + b * a.n_sb];
  if (threadIdx.x < 64) {
    const int len = tree_walk(a, b, threadIdx.x, path);
    if (threadIdx.x == 0) length = len;
  }
  __syncthreads();
  const int len = length;
  if (l == 0 && h == 0) {
    for (int i = threadIdx.x; i < a.T; i += 256) a.path[(int64_t)b * a.T + i] = i < len ? path[i] : -1;
    if (threadIdx.x == 0) a.accepted[b] = len;
  }
  if (n < 0) return;
  const int fit = min(len, a.C - n);  // (rows past the capacity are not stored)
  const int64_t dst = (((int64_t)l * a.B + b) * a.H + h) * a.C * a.units;
  const uint8_t* kn = a.kn + l * a.kn_sn + b * a.kn_sb + h * a.kn_sh;
  const uint8_t* vn = a.vn + l * a.vn_sn + b * a.vn_sb + h * a.vn_sh;
  for (int x = threadIdx.x; x < 2 * fit * a.units; x += 256) {
    const int v = x >= fit * a.units, y = x - v * fit * a.units;
    const int i = y / a.units, u = y - i * a.units;
    const uint8_t* src = v ? vn + path[i] * a.vn_st : kn + path[i] * a.kn_st;
    reinterpret_cast<U*>(v ? a.vbuf : a.kbuf)[dst + (int64_t)(n + i) * a.units + u] = reinterpret_cast<const U*>(src)[u];
  }
}

hipError_t launch_tree_commit(const dropkv_tree_commit_args& p, hipStream_t st) {
  CommitArgs a{};
  a.tokens = p.tokens;
  a.choice = p.choice;
  a.parents = p.parents;
  a.p_sb = p.p_sb;
  a.T = (int)p.T;
  a.path = p.path;
  a.accepted = p.accepted;
  const int64_t eb = p.elem_bytes;
  a.kn = static_cast<const uint8_t*>(p.k_new);
  a.vn = static_cast<const uint8_t*>(p.v_new);
  a.kn_sn = p.kn_s[0] * eb;
  a.kn_sb = p.kn_s[1] * eb;
  a.kn_sh = p.kn_s[2] * eb;
  a.kn_st = p.kn_s[3] * eb;
  a.vn_sn = p.vn_s[0] * eb;
  a.vn_sb = p.vn_s[1] * eb;
  a.vn_sh = p.vn_s[2] * eb;
  a.vn_st = p.vn_s[3] * eb;
  a.kbuf = static_cast<uint8_t*>(p.k_cache);
  a.vbuf = static_cast<uint8_t*>(p.v_cache);
  a.n_rows = p.n_rows;
  a.n_sn = p.n_s[0];
  a.n_sb = p.n_s[1];
  a.B = (int)p.B;
  a.H = (int)p.H;
  a.C = (int)p.capacity;
  const int64_t all = (int64_t)reinterpret_cast<uintptr_t>(a.kn) | (int64_t)reinterpret_cast<uintptr_t>(a.vn) |
                      (int64_t)reinterpret_cast<uintptr_t>(a.kbuf) | (int64_t)reinterpret_cast<uintptr_t>(a.vbuf) |
                      a.kn_sn | a.kn_sb | a.kn_sh | a.kn_st | a.vn_sn | a.vn_sb | a.vn_sh | a.vn_st | (p.D * eb);
  const dim3 grid((unsigned)(p.N * p.B * p.H));
  if (all % 16 == 0) {
    a.units = (int)(p.D * eb / 16);
    launch(tree_commit_kernel<u32x4>, grid, dim3(256), 0, st, a);
  } else if (eb == 4) {
    a.units = (int)p.D;
    launch(tree_commit_kernel<uint32_t>, grid, dim3(256), 0, st, a);
  } else {
    a.units = (int)p.D;
    launch(tree_commit_kernel<uint16_t>, grid, dim3(256), 0, st, a);
  }
  return hipGetLastError();
}

}  // namespace dkv
