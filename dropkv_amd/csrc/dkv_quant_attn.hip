// Attention over a cache in 8 bits (its layout: dkv_quant_dev.h): T new tokens per
// sequence over the stored rows and over one another under a mask, one token of a
// decode step or a tree or chain of drafted ones.  (The reference decodes one
// token per step over a cache in the model's type, dropkv_cache.py:609-617.)
//
// The g query heads of a KV head and the T tokens are its M = g T rows, as in
// dkv_tree.hip.  A block's scales are numbers of their own, so that the stored
// values themselves enter the products (exactly: they fit the element type):
//   x_rj = (scale ks_b log2 e) (q_r . k8_j),  out_r = sum_b vs_b sum_j 2^(x_rj - m_r) v8_j / sum_j 2^(x_rj - m_r)
// with j in block b, and ks, vs = 1 for the keys in 16 bits: the rows of the block
// that is not full, and the new tokens' own.  The blocks are cut into parts,
// dealt by the sequences' lengths; the 16-bit keys are one part more, or the last
// one's end; a second kernel, or the last workgroup to arrive, joins the parts.
//
// S = K Q^T and O += V^T P^T with 64 keys a step.  Row rho = 4 lg + r of key block kb
// is key 16 lg + 4 kb + r, so that lane (li, lg) holds row li's weights of keys 16 lg
// .. 16 lg + 15, which are those of the 16 bytes it holds of a column of V.  The
// depth of a product is permuted alike for K and Q (bytes 16 lg + 8 h .. + 7 of 64
// are step h's).
#include "dkv_quant_dev.h"
#include "dkv_tree_dev.h"

#include <algorithm>
#include <cmath>

namespace dkv {

struct QuantAttnArgs : TreeArgs {  // (kbuf, vbuf: the 8-bit blocks)
  const float* ks;    // [B, Hkv, C / 64]
  const float* vs;
  const void* ktail;  // [B, Hkv, 128, D]
  const void* vtail;
  uint32_t* arrived;  // [B, Hkv] at arrived_s: parts done, where the last one to arrive joins them; else null
  int arrived_s;
};

struct QuantCut {
  static __device__ __forceinline__ int tiles(int n) { return n / kQBlock; }
};

// The wide kernel lets a row's maximum rise so far (powers of two) above the
// reference that its weights are taken against before it turns what it has summed.
constexpr float kQRise = 8.f;

// Weights of 16-bit keys enter their products in the element type, and fp16 ends at 2^-24:
// there they are 2^14 times as large, so that weights from 2^-22 on hold 16 bits in two
// parts, and the outputs' sums are for as long.  (The wide kernel's maximum may then rise
// by no more than 1: the largest weight is 2^15.  Without it a value of 1000 at a weight
// of 2^-19 came out up to 1% off.)
template <typename T>
constexpr int kNearLift = std::is_same<T, _Float16>::value ? 14 : 0;
template <typename T>
constexpr float kNearRise = std::is_same<T, _Float16>::value ? 1.f : kQRise;

// Weights are 2^(x mul - m + log2 vs) by one fma, vs the scale of the block's values.
// From here on (in powers of two) m's own rounding would lift them far above 1, or lose
// them: there the difference of the two rounded logits is taken first, the larger one
// itself among them.  (Both rounded: `weigh` is compiled without contraction, which would
// make one fma of a logit's product and the difference, and at 2^29 the largest weight
// anything from 2^-32 to 2^32.)
constexpr float kQFar = 4194304.f;

// A step of 16-bit keys: the `held` rows of the tail (rows first ..), then `fresh`
// new ones from j0 on.
struct Near {
  int first, held, j0, fresh;
};
// Key e of it.  (Past the last: its row again, whose weight there is 0; 0 times a value
// that is not finite is NaN, which only a tail row leaves there, and it reaches every
// token anyway.)
template <typename T, int D>
__device__ __forceinline__ const T* near_row(const Near& s, int e, const T* tail, const T* kn, int64_t st) {
  const int i = min(e, s.held + s.fresh - 1);
  return i < s.held ? tail + ((s.first + i) % kQTail) * D : kn + (int64_t)(s.j0 + i - s.held) * st;
}
// The steps of n % 64 tail rows and T new ones: one step if they fit, else the
// tail's first.
__device__ __forceinline__ Near near_begin(int n, int T) {
  const int held = n % kQBlock;
  return Near{n - held, held, 0, held + T <= kQBlock ? T : held ? 0 : min(T, kQBlock)};
}
__device__ __forceinline__ bool near_next(Near* s, int T) {
  s->j0 += s->fresh;
  s->held = 0;
  s->fresh = min(T - s->j0, kQBlock);
  return s->fresh > 0;
}
// The keys of it that a token sees, whose word of the new ones is w.
__device__ __forceinline__ uint64_t near_bits(const Near& s, uint64_t w) {
  return s.held ? ((uint64_t(1) << s.held) - 1) | (s.fresh ? w << s.held : 0) : w;
}

// The V operand of eight 16-bit keys (k0 .. k0 + 7 for this lane's group) at columns
// d0 .. d0 + 15, by two transposing reads of four keys each.
template <typename T, int D>
__device__ __forceinline__ typename Elem<T>::v8 near_v(const T* vt, int k0, int d0, int li, int pitch) {
  typedef short s4 __attribute__((ext_vector_type(4)));
  typedef __attribute__((address_space(3))) s4 lds_s4;
  const T* p = vt + (k0 + li / 4) * pitch + d0 + 4 * (li % 4);
  const s4 x0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)p);
  const s4 x1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4*)(p + 4 * pitch));
  return __builtin_bit_cast(typename Elem<T>::v8, __builtin_shufflevector(x0, x1, 0, 1, 2, 3, 4, 5, 6, 7));
}

// Whether an element of `n` 16-byte pieces is not finite, by the largest magnitude as
// a whole number; and, where some lane has one, those of new rows taken out of the
// rows in LDS (`at(i)`: piece i's row and column).  (One by one in line they were
// 20 KB of code, fetched by every call: the 16-bit step took 7 us, 2 without.)
template <typename T, int N>
__device__ __forceinline__ bool near_any_odd(const typename Elem<T>::v8 (&x)[N]) {
  typedef uint16_t us2 __attribute__((ext_vector_type(2)));
  us2 m = {0, 0};
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const u32x4 w = __builtin_bit_cast(u32x4, x[i]) & 0x7fff7fffu;
#pragma unroll
    for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(us2, (uint32_t)w[e]));
  }
  return wave_any(max(m[0], m[1]) >= (std::is_same<T, _Float16>::value ? 0x7c00 : 0x7f80));
}
template <typename T, typename F>
__device__ __forceinline__ bool near_take_out(T* rows, int pitch, const Near& s, int n, F&& at) {
  bool odd = false;
#pragma unroll 1
  for (int i = 0; i < 8 * n; ++i) {
    int e, col;
    at(i / 8, &e, &col);
    T* x = rows + e * pitch + col + i % 8;
    if (e >= s.held && not_finite<T>(*x)) {
      odd = true;
      *x = static_cast<T>(0.f);
    }
  }
  return odd;
}

// Up to 32 rows per KV head (RT tiles of 16): workgroups of four waves, which take the
// blocks of a part in turn, and the step of 16-bit keys as one block more.  K and V come as
// matrix operands straight into registers, the next block's loads issued as soon as
// a block's registers are consumed.  P goes into the product in two parts, rounded
// and remainder.  The waves' results are joined in LDS; the only part's workgroup
// writes the output.  Of several parts the last workgroup to arrive joins them, where
// they are few bytes; more are joined by a second kernel.
// Bound by memory or by latency: 8 x 8 heads of 19151 to 26214 rows, D = 128 (372 MB), one
// token: 71.6 us (5.2 TB/s); 2 heads of 1638 rows, D = 64: 7.1 (4.1 of them a kernel that
// loads nothing); 8 heads of 3276 rows, D = 128: 9.6.
constexpr int kNarrowWaves = 4;
template <typename T, typename S, int D, int RT>
__global__ void __launch_bounds__(64 * kNarrowWaves, RT == 1 ? 2 : 1) quant_narrow_kernel(QuantAttnArgs a) {
  typedef typename Elem<T>::v8 v8;
  typedef Elem<__bf16>::v8 b8;
  constexpr int KC = D / 64, DT = D / 16, CPR = D / 8, GRP = 64 / CPR, NW = kNarrowWaves, ROWS = 16 * RT;
  constexpr int kVPitch = D + 16;  // transposing reads without bank conflicts
  constexpr int kOPitch = D + 4;   // floats
  constexpr int kLds = std::max(kQBlock * kVPitch * (int)sizeof(T), NW * ROWS * kOPitch * 4);
  const int slot = blockIdx.x % a.P, hkv = blockIdx.x / a.P, g = a.Hq / a.Hkv;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, li = lane & 15, lg = lane >> 4;
  __shared__ __attribute__((aligned(16))) char lds[kLds];
  __shared__ uint64_t mask_words[ROWS];  // (T <= the rows)
  __shared__ float part_m[NW][ROWS], part_l[NW][ROWS];
  __shared__ int odd_flag, last;

  const TreePart part = tree_part<QuantCut>(a, hkv, slot, lane);
  const int b = part.b;
  if (b < 0) return;
  const int64_t bh = (int64_t)b * a.Hkv + hkv;
  const int blocks = a.C / kQBlock;
  const uint8_t* kb = static_cast<const uint8_t*>(a.kbuf) + bh * a.C * D;
  const uint8_t* vb = static_cast<const uint8_t*>(a.vbuf) + bh * a.C * D;
  // Loads at and past the part's end read zeros.
  const rsrc_t krs = make_rsrc(kb, (uint32_t)part.t_hi * kQBlock * D), vrs = make_rsrc(vb, (uint32_t)part.t_hi * kQBlock * D);
  const float *ksc = a.ks + bh * blocks, *vsc = a.vs + bh * blocks;
  u32x4 kx[4][KC], vx[DT];
  float ks, vs;
  auto load_k = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int c = 0; c < KC; ++c)
        kx[i][c] = buf_load16(krs, (uint32_t)(j * kQBlock + 16 * (li / 4) + 4 * i + li % 4) * D + 64u * c + 16u * lg);
    ks = ksc[min(j, blocks - 1)];
  };
  auto load_v = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) vx[dt] = buf_load16(vrs, (uint32_t)j * kQBlock * D + (16 * dt + li) * kQBlock + 16u * lg);
    vs = vsc[min(j, blocks - 1)];
  };
  int j = part.t_lo + wave;
  if (j < part.t_hi) {
    load_k(j);
    load_v(j);
  }

  // Row 16 x + li: query head hkv g + h, token t.
  int tq[RT];
  v8 qop[RT][KC][2];
  float m[RT], lsum[RT];
  f32x4 s[RT][4], o[RT][DT];
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int row = min(16 * x + li, a.M - 1);  // (rows past the last repeat it and are not stored)
    const int h = a.div_t.div(row), t = row - h * a.T;
    tq[x] = t;
    const T* qr = static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)(hkv * g + h) * a.q_sh + (int64_t)t * a.q_st;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) qop[x][c][hf] = tree_load8(qr + 64 * c + 16 * lg + 8 * hf);
    m[x] = -__FLT_MAX__;  // (finite, so that logits of -inf get no weight)
    lsum[x] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[x][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // From products (times `mul`: logits) to weights times the values' scale, 2^up = 1 /
  // down; `seen`: a bit for each of the lane's keys.
  auto weigh = [&](int x, float mul, float up, float down, uint32_t seen) __attribute__((always_inline)) {
#pragma clang fp contract(off)
    float tmax = -INFINITY;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      s[x][e / 4][e % 4] = (seen >> e) & 1 ? s[x][e / 4][e % 4] : -INFINITY;
      tmax = __builtin_elementwise_maximum(tmax, s[x][e / 4][e % 4]);
    }
    tmax = maximum_xor32(maximum_xor16(tmax)) * mul;
    if (wave_any(tmax > m[x])) {
      const float mnew = fmaxf(m[x], tmax), alpha = __builtin_amdgcn_exp2f(m[x] - mnew);
      lsum[x] *= alpha;
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) o[x][dt] *= alpha;
      m[x] = mnew;
    }
    float by = mul, less = up - m[x];
    if (wave_any(fabsf(m[x]) >= kQFar)) {
#pragma unroll
      for (int e = 0; e < 16; ++e) s[x][e / 4][e % 4] = s[x][e / 4][e % 4] * mul - m[x];
      by = 1.f;
      less = up;
    }
    float sum = 0.f;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      const float p = __builtin_amdgcn_exp2f(fmaf(s[x][e / 4][e % 4], by, less));
      s[x][e / 4][e % 4] = p;
      sum += p;
    }
    lsum[x] = fmaf(sum, down, lsum[x]);
  };

  for (; j < part.t_hi; j += NW) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int x = 0; x < RT; ++x) s[x][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < KC; ++c)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const v8 kop = unpack8<S, T>(kx[i][c], hf);
#pragma unroll
          for (int x = 0; x < RT; ++x) s[x][i] = Elem<T>::mfma(kop, qop[x][c][hf], s[x][i]);
        }
    }
    // (A block of zeros has no scale: any will do.)
    const float mul = ks * a.scale_log2, fold = vs == 0.f ? 1.f : vs, up = __builtin_amdgcn_logf(fold), down = __builtin_amdgcn_rcpf(fold);
    load_k(j + NW);
#pragma unroll
    for (int x = 0; x < RT; ++x) weigh(x, mul, up, down, 0xffffu);
    b8 phi[RT][2], plo[RT][2];
#pragma unroll
    for (int x = 0; x < RT; ++x)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = s[x][2 * hf + e / 4][e % 4];
          phi[x][hf][e] = static_cast<__bf16>(p);
          plo[x][hf][e] = static_cast<__bf16>(p - static_cast<float>(phi[x][hf][e]));
        }
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const b8 vop = unpack8<S, __bf16>(vx[dt], hf);
#pragma unroll
        for (int x = 0; x < RT; ++x) {
          o[x][dt] = Elem<__bf16>::mfma(vop, phi[x][hf], o[x][dt]);
          o[x][dt] = Elem<__bf16>::mfma(vop, plo[x][hf], o[x][dt]);
        }
      }
    load_v(j + NW);
  }

  // The 16-bit keys: by the wave whose turn it is.
  bool odd = false;
  if (part.tail && (part.t_hi - part.t_lo) % NW == wave) {
    const T* kt = static_cast<const T*>(a.ktail) + bh * kQTail * D;
    const T* vtl = static_cast<const T*>(a.vtail) + bh * kQTail * D;
    const T* kn = static_cast<const T*>(a.kn) + (int64_t)b * a.kn_sb + (int64_t)hkv * a.kn_sh;
    const T* vn = static_cast<const T*>(a.vn) + (int64_t)b * a.vn_sb + (int64_t)hkv * a.vn_sh;
    const int v_row = lane / CPR, v_col = 8 * (lane % CPR);
    T* vt = reinterpret_cast<T*>(lds);
    Near step = near_begin(part.n, a.T);
    constexpr float kLift = 1 << kNearLift<T>;
    if (kLift != 1.f)
#pragma unroll
      for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= kLift;
#pragma unroll 1
    do {  // (one wave: its own LDS operations stay in order)
      v8 kop[4][KC][2], vch[kQBlock / GRP];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const T* row = near_row<T, D>(step, 16 * (li / 4) + 4 * i + li % 4, kt, kn, a.kn_st);
#pragma unroll
        for (int c = 0; c < KC; ++c)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) kop[i][c][hf] = tree_load8(row + 64 * c + 16 * lg + 8 * hf);
      }
#pragma unroll
      for (int i = 0; i < kQBlock / GRP; ++i)
        vch[i] = tree_load8(near_row<T, D>(step, v_row + i * GRP, vtl, vn, a.vn_st) + v_col);
      tree_mask_words<1>(a, b, step.j0, 0, lane, mask_words);
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int x = 0; x < RT; ++x) {
          s[x][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int c = 0; c < KC; ++c)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) s[x][i] = Elem<T>::mfma(kop[i][c][hf], qop[x][c][hf], s[x][i]);
        }
#pragma unroll
      for (int i = 0; i < kQBlock / GRP; ++i) *reinterpret_cast<v8*>(vt + (v_row + i * GRP) * kVPitch + v_col) = vch[i];
      if (__builtin_expect(near_any_odd<T>(vch), 0))
        odd |= near_take_out(vt, kVPitch, step, kQBlock / GRP, [&](int i, int* e, int* col) {
          *e = v_row + i * GRP;
          *col = v_col;
        });
      v8 phi[RT][2], plo[RT][2];
#pragma unroll
      for (int x = 0; x < RT; ++x) {
        const uint64_t bits = near_bits(step, mask_words[tq[x]]);
        weigh(x, a.scale_log2, kNearLift<T>, 1.f / kLift, (uint32_t)(bits >> (16 * lg)) & 0xffffu);
#pragma unroll
        for (int hf = 0; hf < 2; ++hf)
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float p = s[x][2 * hf + e / 4][e % 4];
            phi[x][hf][e] = static_cast<T>(p);
            plo[x][hf][e] = static_cast<T>(p - static_cast<float>(phi[x][hf][e]));
          }
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {
          const v8 vop = near_v<T, D>(vt, 16 * lg + 8 * hf, 16 * dt, li, kVPitch);
#pragma unroll
          for (int x = 0; x < RT; ++x) {
            o[x][dt] = Elem<T>::mfma(vop, phi[x][hf], o[x][dt]);
            o[x][dt] = Elem<T>::mfma(vop, plo[x][hf], o[x][dt]);
          }
        }
    } while (near_next(&step, a.T));
    if (kLift != 1.f)
#pragma unroll
      for (int x = 0; x < RT; ++x)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= 1.f / kLift;
  }

  // The waves' results joined: 16 threads a row.
  if (threadIdx.x == 0) odd_flag = 0;
  __syncthreads();  // (V's rows have been read)
#pragma unroll
  for (int x = 0; x < RT; ++x) {
    const int at = 16 * x + li;
    const float l = add_xor32(add_xor16(lsum[x]));
    float* ol = reinterpret_cast<float*>(lds) + (wave * ROWS + at) * kOPitch + 4 * lg;
    if (at < a.M) {
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) *reinterpret_cast<f32x4*>(ol + 16 * dt) = o[x][dt];
    }
    if (lg == 0) {
      part_m[wave][at] = m[x];
      part_l[wave][at] = l;
    }
  }
  if (wave_any(odd) && lane == 0) odd_flag = 1;
  __syncthreads();
#pragma unroll 1
  for (int row = threadIdx.x >> 4; row < a.M; row += 16) {
    float mx = part_m[0][row], l = 0.f, f[NW];
#pragma unroll
    for (int w = 1; w < NW; ++w) mx = fmaxf(mx, part_m[w][row]);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      f[w] = __builtin_amdgcn_exp2f(part_m[w][row] - mx);
      l += part_l[w][row] * f[w];
    }
    const int hr = a.div_t.div(row), tr = row - hr * a.T;
    T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)tr * a.o_st + (int64_t)(hkv * g + hr) * a.o_sh;
    const int64_t base = ((int64_t)hkv * a.P + slot) * a.M + row;
    // (The wave's four rows.)
    const rsrc_t prs = make_rsrc(
        a.part_o + (((int64_t)hkv * a.P + slot) * a.M + __builtin_amdgcn_readfirstlane(row & ~3)) * D, 4 * D * 4u);
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const int d0 = 4 * (threadIdx.x & 15) + 64 * i;
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        const f32x4 y = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds) + (w * ROWS + row) * kOPitch + d0);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = fmaf(f[w], y[e], acc[e]);
      }
      if (a.direct) {
#pragma unroll
        for (int e = 0; e < 4; ++e) out[d0 + e] = static_cast<T>(l == 0.f ? 0.f : acc[e] * inv);
      } else {
        st_dev16(prs, ((row & 3) * D + d0) * 4u, acc);
      }
    }
    if (!a.direct && (threadIdx.x & 15) == 0) {
      st_dev(a.part_m + base, mx);
      st_dev(a.part_l + base, l);
    }
  }
  if (__builtin_expect(odd_flag, 0)) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    tree_add_odd<T, D, 64 * NW>(a, b, hkv, slot, 0, ROWS);
  }
  if (!a.arrived) return;
  // (Every wave's stores are out first.  The counter is zero before the call and wraps
  // to zero.)
  __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    last = atomicInc(a.arrived + bh * a.arrived_s, (uint32_t)part.count - 1u) == (uint32_t)part.count - 1u;
    if (last) __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "agent");
  }
  __syncthreads();
  if (!last) return;
  // 16 threads a row: 16 parts' maxima and sums a thread each, and the partial rows, in
  // one round trip.
  const int sub = threadIdx.x & 15;
#pragma unroll 1
  for (int row = threadIdx.x >> 4; row < a.M; row += 16) {
    const int64_t at0 = ((int64_t)hkv * a.P + part.first) * a.M + row;
    // (Ragged sequences may have more than 16.)
    f32x4 acc[D / 64];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) acc[c] = f32x4{0.f, 0.f, 0.f, 0.f};
    float mx = -__FLT_MAX__, l = 0.f;
#pragma unroll 1
    for (int s0 = 0; s0 < part.count; s0 += 16) {
      const int s = s0 + sub;
      const float pm = s < part.count ? a.part_m[at0 + (int64_t)s * a.M] : -__FLT_MAX__;
      const float pl = s < part.count ? a.part_l[at0 + (int64_t)s * a.M] : 0.f;
      f32x4 x[16][D / 64];
#pragma unroll
      for (int k = 0; k < 16; ++k)
#pragma unroll
        for (int c = 0; c < D / 64; ++c)
          x[k][c] = *reinterpret_cast<const f32x4*>(a.part_o + (at0 + (int64_t)min(s0 + k, part.count - 1) * a.M) * D +
                                                    4 * sub + 64 * c);
      float top = pm;
      top = fmaxf(top, dpp_f<kDppQuadSwap1>(top));
      top = fmaxf(top, dpp_f<kDppQuadSwap2>(top));
      top = fmaxf(top, dpp_f<kDppHalfMirror>(top));
      top = fmaxf(top, dpp_f<kDppMirror>(top));
      top = fmaxf(mx, top);
      const float turn = __builtin_amdgcn_exp2f(mx - top), f = s < part.count ? __builtin_amdgcn_exp2f(pm - top) : 0.f;
      mx = top;
      float sum = pl * f;
      sum += dpp_f<kDppQuadSwap1>(sum);
      sum += dpp_f<kDppQuadSwap2>(sum);
      sum += dpp_f<kDppHalfMirror>(sum);
      sum += dpp_f<kDppMirror>(sum);
      l = l * turn + sum;
#pragma unroll
      for (int c = 0; c < D / 64; ++c) acc[c] *= turn;
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float fk = __shfl(f, (lane & 48) | k);
        if (s0 + k < part.count)
#pragma unroll
          for (int c = 0; c < D / 64; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[c][e] = fmaf(fk, x[k][c][e], acc[c][e]);
      }
    }
    const int hr = a.div_t.div(row), tr = row - hr * a.T;
    T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)tr * a.o_st + (int64_t)(hkv * g + hr) * a.o_sh;
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int c = 0; c < D / 64; ++c)
#pragma unroll
      for (int e = 0; e < 4; ++e) out[4 * sub + 64 * c + e] = static_cast<T>(l == 0.f ? 0.f : acc[c][e] * inv);
  }
}

// More than 32 rows: NW waves of QB blocks of 16 rows take the same keys, so that a
// block of K and V is read, and turned into operands, once for all of them.  LDS holds
// the operands of a stage of 64 keys as the lanes read them, 16 bytes a lane, 1 KB a
// product; the next stage's bytes are on their way in registers while the waves
// compute, and go to another buffer.  V's scale goes into the reference of the exponent
// (P is 2^(x - m + log2 vs)), and is taken out of the weights' sum.  P is rounded once
// for bf16 in workgroups of 128 rows and more, in two parts otherwise.
// 64 or 128 rows: one barrier a stage, and the two workgroups of a CU overlap.  256 rows
// (PAIR): two groups of four waves, half a stage apart.
// Bound by the matrix cores and the ALUs, which share the issue of a SIMD and the clock
// that the power leaves: 4 x 64 heads of 26214 rows, 64 tokens, 204 to 222 us by the box
// (1080 to 990 TFLOP/s; 231 with all waves in step), of which 11 are the join; the
// matrix cores are busy 55% of the time, the ALUs 62%.  16 tokens of 32/8 heads over 3276
// rows: 13 us, two kernels' latencies (9 and 4).
template <typename T, typename S, int D, int QB, int NW, bool LO, bool PAIR>
__global__ void __launch_bounds__(64 * NW, 2) quant_wide_kernel(QuantAttnArgs a) {
  typedef typename Elem<T>::v8 v8;
  constexpr int KC = D / 64, DT = D / 16, NT = 64 * NW;
  constexpr int kPieces = 64 * (4 * KC), NC = 2 * kPieces / NT;  // 16-byte pieces of a block's K (or V); per thread
  constexpr int kOps = 4 * KC * 2;                               // operands of a stage's K (or V)
  constexpr int kBuf = kOps * 64;                                // 16-byte places per buffer of K (or V)
  constexpr int kVBufs = PAIR ? 3 : 2;                           // (of K: 2)
  static_assert(DT == 4 * KC && NC * NT == 2 * kPieces && (!PAIR || NW == 8), "whole pieces per thread");
  __shared__ u32x4 lds[(2 + kVBufs) * kBuf];
  __shared__ uint64_t mask_words[kTreeMaxT];
  __shared__ int odd_flag;

  const int id = xcd_remap(blockIdx.x, gridDim.x);
  const int mc = id % a.MC, slot = (id / a.MC) % a.P, hkv = id / (a.MC * a.P), g = a.Hq / a.Hkv;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63, li = lane & 15, lg = lane >> 4;
  const TreePart part = tree_part<QuantCut>(a, hkv, slot, lane);
  const int b = part.b;
  if (b < 0) return;
  const int64_t bh = (int64_t)b * a.Hkv + hkv;
  const int row0 = (mc * NW + wave) * (16 * QB) + li;  // the lane's row of block 0

  v8 qop[QB][KC][2];
  int tq[QB];
#pragma unroll
  for (int x = 0; x < QB; ++x) {
    const int row = min(row0 + 16 * x, a.M - 1);  // (rows past the last repeat it and are not stored)
    const int h = a.div_t.div(row), t = row - h * a.T;
    tq[x] = t;
    const T* qr =
        static_cast<const T*>(a.q) + (int64_t)b * a.q_sb + (int64_t)(hkv * g + h) * a.q_sh + (int64_t)t * a.q_st;
#pragma unroll
    for (int c = 0; c < KC; ++c)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) qop[x][c][hf] = tree_load8(qr + 64 * c + 16 * lg + 8 * hf);
  }

  const uint8_t* kb = static_cast<const uint8_t*>(a.kbuf) + bh * a.C * D;
  const uint8_t* vb = static_cast<const uint8_t*>(a.vbuf) + bh * a.C * D;
  const rsrc_t krs = make_rsrc(kb, (uint32_t)part.t_hi * kQBlock * D), vrs = make_rsrc(vb, (uint32_t)part.t_hi * kQBlock * D);
  const int blocks = a.C / kQBlock;
  const float *ksc = a.ks + bh * blocks, *vsc = a.vs + bh * blocks;

  // Piece i of the thread: operand pair `op` of K (key block op / KC, 64 columns op %
  // KC) or V (16 columns), for lane `lane`.
  u32x4 piece[NC];
  float ks, vs;
  auto place = [&](int i, int* op) __attribute__((always_inline)) {
    const int f = (tid + i * NT) / 64;
    *op = f % (4 * KC);
    return f >= 4 * KC;
  };
  auto fetch = [&](int j) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      int op;
      if (place(i, &op))
        piece[i] = buf_load16(vrs, (uint32_t)j * kQBlock * D + (16 * op + li) * kQBlock + 16u * lg);
      else
        piece[i] = buf_load16(krs, (uint32_t)(j * kQBlock + 16 * (li / 4) + 4 * (op / KC) + li % 4) * D + 64u * (op % KC) + 16u * lg);
    }
    ks = ksc[min(j, blocks - 1)];
    vs = vsc[min(j, blocks - 1)];
  };
  auto put = [&](int kbuf, int vbuf) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      int op;
      const bool v = place(i, &op);
      u32x4* to = lds + (v ? 2 + vbuf : kbuf) * kBuf + 2 * op * 64 + lane;
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        to[64 * hf] = v ? __builtin_bit_cast(u32x4, unpack8<S, __bf16>(piece[i], hf))
                        : __builtin_bit_cast(u32x4, unpack8<S, T>(piece[i], hf));
    }
  };

  // The reference of the weights (finite, so that logits of -inf get no weight), and
  // the whole sum of row li.
  float m[QB], lsum[QB];
  f32x4 o[QB][DT];
#pragma unroll
  for (int x = 0; x < QB; ++x) {
    m[x] = -__FLT_MAX__;
    lsum[x] = 0.f;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[x][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
  }

  // A stage in three steps: products with K, weights, products with V.  Of `near` stages,
  // 16-bit keys of see_bits, K's operands are at the start of LDS and V's rows behind.
  uint32_t see_bits[QB];
  constexpr int kVPitch = D + 16;  // transposing reads without bank conflicts
  static_assert(kOps * 64 * 16 + kQBlock * kVPitch * 2 <= (int)sizeof(lds), "a step of 16-bit keys fits");
  f32x4 s[QB][4];
  u32x4 phi[QB][2], plo[LO ? QB : 1][2];
  float down = 1.f;
  auto with_k = [&](int buf) __attribute__((always_inline)) {
    const u32x4* kt = lds + buf * kBuf + lane;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
#pragma unroll
      for (int x = 0; x < QB; ++x) s[x][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2 * KC; ++c) {
        const v8 kop = bitcast_u4<v8>(kt[(2 * KC * i + c) * 64]);
#pragma unroll
        for (int x = 0; x < QB; ++x) s[x][i] = Elem<T>::mfma(kop, qop[x][c / 2][c % 2], s[x][i]);
      }
    }
  };
  // The logits are the products times `mul`; the weights come times vscale.
  auto weigh = [&](float mul, float vscale, auto near) __attribute__((always_inline)) {
#pragma clang fp contract(off)
    constexpr bool kNear = decltype(near)::value;
    constexpr float kRise = kNear ? kNearRise<T> : kQRise;
    typedef std::conditional_t<kNear, T, __bf16> VT;
    typedef typename Elem<VT>::v8 vv8;
    float top[QB];
    bool turn = false;
#pragma unroll
    for (int x = 0; x < QB; ++x) {
      if (kNear)
#pragma unroll
        for (int e = 0; e < 16; ++e) s[x][e / 4][e % 4] = (see_bits[x] >> e) & 1 ? s[x][e / 4][e % 4] : -INFINITY;
      float tmax = s[x][0][0];
#pragma unroll
      for (int e = 1; e < 16; ++e) tmax = __builtin_elementwise_maximum(tmax, s[x][e / 4][e % 4]);
      top[x] = maximum_xor32(maximum_xor16(tmax)) * mul;
      turn |= top[x] - m[x] > kRise;
    }
    if (wave_any(turn)) {
#pragma unroll
      for (int x = 0; x < QB; ++x) {
        const float mnew = top[x] - m[x] > kRise ? top[x] : m[x], alpha = __builtin_amdgcn_exp2f(m[x] - mnew);
        lsum[x] *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= alpha;
        m[x] = mnew;
      }
    }
    // (A block of zeros has no scale: any will do.)
    const float fold = vscale == 0.f ? 1.f : vscale, up = kNear ? (float)kNearLift<T> : __builtin_amdgcn_logf(fold);
    down = kNear ? 1.f / (1 << kNearLift<T>) : __builtin_amdgcn_rcpf(fold);
    float by = mul, less[QB];
    bool far = false;
#pragma unroll
    for (int x = 0; x < QB; ++x) {
      less[x] = up - m[x];
      far |= fabsf(m[x]) >= kQFar;
    }
    if (wave_any(far)) {
#pragma unroll
      for (int x = 0; x < QB; ++x) {
#pragma unroll
        for (int e = 0; e < 16; ++e) s[x][e / 4][e % 4] = s[x][e / 4][e % 4] * mul - m[x];
        less[x] = up;
      }
      by = 1.f;
    }
#pragma unroll
    for (int x = 0; x < QB; ++x)
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        vv8 hi, lo;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(s[x][2 * hf + e / 4][e % 4], by, less[x]));
          hi[e] = static_cast<VT>(p);
          if (LO) lo[e] = static_cast<VT>(p - static_cast<float>(hi[e]));
        }
        phi[x][hf] = __builtin_bit_cast(u32x4, hi);
        if (LO) plo[x][hf] = __builtin_bit_cast(u32x4, lo);
      }
  };
  auto with_v = [&](int buf, auto near) __attribute__((always_inline)) {
    constexpr bool kNear = decltype(near)::value;
    typedef std::conditional_t<kNear, T, __bf16> VT;
    typedef typename Elem<VT>::v8 vv8;
    const u32x4* vt = lds + (2 + buf) * kBuf + lane;
    f32x4 sum[QB];
#pragma unroll
    for (int x = 0; x < QB; ++x) sum[x] = f32x4{0.f, 0.f, 0.f, 0.f};
    vv8 ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = static_cast<VT>(1.f);
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
#pragma unroll
      for (int x = 0; x < QB; ++x) {
        sum[x] = Elem<VT>::mfma(ones, bitcast_u4<vv8>(phi[x][hf]), sum[x]);
        if (LO) sum[x] = Elem<VT>::mfma(ones, bitcast_u4<vv8>(plo[x][hf]), sum[x]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        vv8 vop;
        if constexpr (kNear)
          vop = near_v<T, D>(reinterpret_cast<const T*>(lds + kOps * 64), 16 * lg + 8 * hf, 16 * dt, li, kVPitch);
        else
          vop = bitcast_u4<vv8>(vt[(2 * dt + hf) * 64]);
#pragma unroll
        for (int x = 0; x < QB; ++x) {
          o[x][dt] = Elem<VT>::mfma(vop, bitcast_u4<vv8>(phi[x][hf]), o[x][dt]);
          if (LO) o[x][dt] = Elem<VT>::mfma(vop, bitcast_u4<vv8>(plo[x][hf]), o[x][dt]);
        }
      }
    }
#pragma unroll
    for (int x = 0; x < QB; ++x) lsum[x] = fmaf(sum[x][0], down, lsum[x]);
  };

  // Keeps kAhead operands on their way from LDS before the products that take them: left
  // alone, the compiler has two (64 cycles of products under a latency of 130, which was
  // 1000 of a stage's 4400 cycles).
  auto ahead = [&](auto reads, auto products) __attribute__((always_inline)) {
    constexpr int R = decltype(reads)::value, M = decltype(products)::value, kAhead = R < 16 ? 4 : 8, kEach = M / R;
    __builtin_amdgcn_sched_group_barrier(0x100, kAhead, 0);
#pragma unroll
    for (int i = 0; i < R - kAhead; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x8, kEach, 0);
      __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, M - (R - kAhead) * kEach, 0);
  };

  if (tid == 0) odd_flag = 0;
  if constexpr (PAIR) {
    // Two groups of four waves, one on each SIMD, half a stage apart: while one works with
    // the matrix cores (V of its last stage, K of this one), the other makes weights and
    // puts operands, a barrier between the halves.  The second group is ahead by a stage
    // with its pieces: those of stage j + 1 must lie there when the first one begins it.
    // V is read a stage after K, so it has three buffers.
    const int group = wave >> 2, n = part.t_hi - part.t_lo;
    if (n > 0) {
      auto turn_over = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_sched_barrier(0);
        __syncthreads();
        __builtin_amdgcn_sched_barrier(0);
      };
      fetch(part.t_lo);
      float mul = ks * a.scale_log2, vscale = vs;
      put(0, 0);
      if (group) {
        fetch(part.t_lo + 1);
        put(1, 1);
      }
      fetch(part.t_lo + 1 + group);
      turn_over();
      if (group) turn_over();
      int vput = 1 + group, vget = 0;  // buffers of V: of the stage put next, and of the last one
#pragma unroll
      for (int x = 0; x < QB; ++x)
#pragma unroll
        for (int hf = 0; hf < 2; ++hf) {  // (before the first stage there are no weights)
          phi[x][hf] = u32x4{0u, 0u, 0u, 0u};
          if (LO) plo[x][hf] = u32x4{0u, 0u, 0u, 0u};
        }
      for (int j = 0; j < n; ++j) {
        with_v(vget, std::false_type{});
        with_k(j & 1);
        ahead(std::integral_constant<int, 2 * kOps>{}, std::integral_constant<int, (2 * DT + 2) * QB * (LO ? 2 : 1) + 8 * KC * QB>{});
        vget = j == 0 ? 0 : vget == 2 ? 0 : vget + 1;
        turn_over();
        weigh(mul, vscale, std::false_type{});
        put((j + 1 + group) & 1, vput);
        vput = vput == 2 ? 0 : vput + 1;
        fetch(part.t_lo + j + 2 + group);
        mul = ksc[min(part.t_lo + j + 1, blocks - 1)] * a.scale_log2;
        vscale = vsc[min(part.t_lo + j + 1, blocks - 1)];
        turn_over();
      }
      with_v(vget, std::false_type{});
      ahead(std::integral_constant<int, kOps>{}, std::integral_constant<int, (2 * DT + 2) * QB * (LO ? 2 : 1)>{});
      if (!group) turn_over();
    }
  } else {
    int buf = 0, j = part.t_lo;
    if (j < part.t_hi) {
      fetch(j);
      float mul = ks * a.scale_log2, vscale = vs;
      put(0, 0);
      for (; j < part.t_hi; ++j) {
        fetch(j + 1);
        __syncthreads();
        with_k(buf);
        ahead(std::integral_constant<int, kOps>{}, std::integral_constant<int, 8 * KC * QB>{});
        weigh(mul, vscale, std::false_type{});
        with_v(buf, std::false_type{});
        ahead(std::integral_constant<int, kOps>{}, std::integral_constant<int, (2 * DT + 2) * QB * (LO ? 2 : 1)>{});
        buf ^= 1;
        mul = ks * a.scale_log2;
        vscale = vs;
        put(buf, buf);
      }
    }
  }
  if (part.tail) {
    const T* kt = static_cast<const T*>(a.ktail) + bh * kQTail * D;
    const T* vtl = static_cast<const T*>(a.vtail) + bh * kQTail * D;
    const T* kn = static_cast<const T*>(a.kn) + (int64_t)b * a.kn_sb + (int64_t)hkv * a.kn_sh;
    const T* vn = static_cast<const T*>(a.vn) + (int64_t)b * a.vn_sb + (int64_t)hkv * a.vn_sh;
    Near step = near_begin(tree_rows(a, b), a.T);
    constexpr float kLift = 1 << kNearLift<T>;
    if (kLift != 1.f)
#pragma unroll
      for (int x = 0; x < QB; ++x)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= kLift;
    constexpr int NK = kOps * 64 / NT, CPR = D / 8, NV = kQBlock * CPR / NT;
#pragma unroll 1
    do {
      u32x4 kpc[NK];
      v8 vch[NV];
#pragma unroll
      for (int i = 0; i < NK; ++i) {
        const int f = (tid + i * NT) / 64, op = f / 2, hf = f % 2;
        const T* row = near_row<T, D>(step, 16 * (li / 4) + 4 * (op / KC) + li % 4, kt, kn, a.kn_st);
        kpc[i] = __builtin_bit_cast(u32x4, tree_load8(row + 64 * (op % KC) + 16 * lg + 8 * hf));
      }
#pragma unroll
      for (int i = 0; i < NV; ++i)
        vch[i] = tree_load8(near_row<T, D>(step, (tid + i * NT) / CPR, vtl, vn, a.vn_st) + 8 * (tid % CPR));
      __syncthreads();  // (the words' and the buffers' last readers are done)
      tree_mask_words<NW>(a, b, step.j0, wave, lane, mask_words);
      bool odd = false;
#pragma unroll
      for (int i = 0; i < NK; ++i) lds[tid + i * NT] = kpc[i];
      T* vrows = reinterpret_cast<T*>(lds + kOps * 64);
#pragma unroll
      for (int i = 0; i < NV; ++i)
        *reinterpret_cast<v8*>(vrows + (tid + i * NT) / CPR * kVPitch + 8 * (tid % CPR)) = vch[i];
      if (__builtin_expect(near_any_odd<T>(vch), 0))
        odd = near_take_out(vrows, kVPitch, step, NV, [&](int i, int* e, int* col) {
          *e = (tid + i * NT) / CPR;
          *col = 8 * (tid % CPR);
        });
      if (odd) odd_flag = 1;
      __syncthreads();
#pragma unroll
      for (int x = 0; x < QB; ++x)
        see_bits[x] = (uint32_t)(near_bits(step, mask_words[tq[x]]) >> (16 * lg)) & 0xffffu;
      with_k(0);
      weigh(a.scale_log2, kLift, std::true_type{});
      with_v(0, std::true_type{});
    } while (near_next(&step, a.T));
    if (kLift != 1.f)
#pragma unroll
      for (int x = 0; x < QB; ++x)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) o[x][dt] *= 1.f / kLift;
  }

#pragma unroll
  for (int x = 0; x < QB; ++x) {
    const int row = row0 + 16 * x;
    if (row >= a.M) continue;
    if (a.direct) {
      const int h = a.div_t.div(row), t = row - h * a.T;
      T* out = static_cast<T*>(a.out) + (int64_t)b * a.o_sb + (int64_t)t * a.o_st + (int64_t)(hkv * g + h) * a.o_sh;
      const float l = lsum[x], inv = l == 0.f ? 0.f : 1.f / l;
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
      st_dev(a.part_m + base, m[x]);
      st_dev(a.part_l + base, lsum[x]);
    }
  }
  if (part.tail && __builtin_expect(odd_flag != 0, 0)) {
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    tree_add_odd<T, D, NT>(a, b, hkv, slot, mc * NW * 16 * QB, NW * 16 * QB);
  }
}

// How a call is cut: rows per workgroup (16: one wave), parts of the cache per
// sequence, and whether the 16-bit keys are parts of their own.
struct QuantPlan {
  int M, rows_wg, MC, S, P, apart;
  int one;  // the last workgroup of a KV head joins its parts (where there are counters)
  size_t rows, bytes;
};

// An estimate of a call's time in us, fitted to sweeps of both over calls of 1 to 512 rows
// per KV head, 2 to 60,000 keys and 2 to 64 heads (the host knows the capacity, not
// the rows): of 46 calls its choice is within a tenth of the best cut in 36, and 1.2 to
// 1.5 times it in 8, whose caches held less than a quarter of their room.  The sum of
// - the longest workgroup's blocks, a block's time by the rows (narrow: a wave's, every
//   fourth), 0.6 of it at D = 64, and longer where workgroups share a CU or take turns;
//   or, if longer, K and V at 5.2 TB/s, where 8 MB or a quarter of them are in flight,
//   and longer where the workgroups do not divide the CUs (of more than 30 MB);
// - the partial rows, written and read at 4 TB/s, and a round trip of the joining
//   kernel for every 16 (D = 128) or 32 parts; of one part, whose workgroup writes the
//   output, neither, but the new tokens' steps behind the blocks';
// - the kernels' fixed part.
struct QuantShape {
  int rows;
  double block_us, fixed_us, shared;  // shared: two workgroups on a CU, against one
  int per_cu;
};
constexpr QuantShape kQuantShapes[] = {
    {16, 1.6, 6.9, 1.2, 2}, {32, 2.1, 7.2, 1.0, 1}, {64, 1.25, 8.3, 1.45, 2}, {128, 1.45, 8.5, 1.7, 2}, {256, 2.1, 8.0, 1.0, 1}};

constexpr int64_t kOneJoin = 8192;  // elements

static double quant_cost(const QuantShape& w, double heads, double M, double D, double T, double blocks, int64_t S) {
  const double wgs = heads * std::ceil(M / w.rows) * S, wide = D / 128;
  const bool narrow = w.rows <= 32;
  const double per = std::ceil((blocks + narrow) / S), load = wgs / (256.0 * w.per_cu);
  double block = w.block_us * (wide < 1 ? 0.6 : 1);
  if (load > 1)
    block *= std::ceil(load) * w.shared;
  else if (w.per_cu == 2 && load > 0.5)
    block *= w.shared;
  const double steps = narrow ? std::ceil(per / kNarrowWaves) : per;
  const double flight = std::min(wgs, 256.0 * w.per_cu) * (narrow ? 65536 : 16384) * wide;
  const double bytes = heads * blocks * kQBlock * D * 2;
  double stream = bytes / 5.2e6 / std::min(1.0, flight / std::max(1.0, std::min(8e6, bytes / 4)));
  if (bytes > 3e7) stream *= 0.5 + 0.5 * std::ceil(wgs / 256) * 256 / wgs;
  const double join = S > 1    ? S * heads * M * D * 8 / 4e6 + 0.6 * std::ceil((S + 1) * wide / 16)
                      : narrow ? -2.5
                               : -3. + 2. * wide * (std::ceil(T / kQBlock) - 1);
  return std::max(steps * block, stream) + join + w.fixed_us;
}

static QuantPlan quant_plan(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t T, int64_t C) {
  QuantPlan p;
  p.M = (int)(Hq / Hkv * T);
  const int64_t heads = B * Hkv, blocks = C / kQBlock;
  const int64_t most = std::max<int64_t>(1, std::min<int64_t>(kTreeMaxSplits, blocks));
  double best = 0;
  p.S = 0;
  for (const QuantShape& w : kQuantShapes) {
    // No shape that the rows would leave half empty; waves of their own blocks for up to
    // 32 rows, workgroups that share them beyond.
    if ((w.rows > 16 && p.M <= w.rows / 2) || (w.rows <= 32 && p.M > w.rows)) continue;
    const int64_t chunks = heads * ((p.M + w.rows - 1) / w.rows);
    const int64_t tries[] = {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 48, kTreeMaxSplits, 256 / chunks, 512 / chunks};
    for (int64_t S : tries) {
      S = std::max<int64_t>(1, std::min(S, most));
      const double cost = quant_cost(w, (double)heads, p.M, (double)D, (double)T, (double)blocks, S);
      if (p.S == 0 || cost < best) {
        best = cost;
        p.S = (int)S;
        p.rows_wg = w.rows;
      }
    }
  }
  p.MC = (p.M + p.rows_wg - 1) / p.rows_wg;
  p.apart = p.S > 1 && (p.rows_wg == 64 || (p.rows_wg > 64 && heads * p.MC * p.S < 192));
  p.P = (int)(B * (p.S + p.apart));
  // (What one workgroup reads in a round trip.)
  p.one = p.rows_wg <= 32 && p.S > 1 && p.S <= 16 && p.S * p.M * D <= kOneJoin;
  p.rows = (size_t)Hkv * p.P * p.M;
  p.bytes = kSyncBytes + kTreeDealBytes + p.rows * sizeof(float) * (2 + (size_t)D) + 256;
  return p;
}
size_t quant_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t D, int64_t T, int64_t C) {
  return quant_plan(B, Hq, Hkv, D, T, C).bytes;
}

template <typename T, typename S, int D>
static hipError_t launch_quant_t(const QuantAttnArgs& a, int rows_wg, hipStream_t st) {
  // fp16 output asks for more than P rounded to bf16.
  constexpr bool kLo = std::is_same<T, _Float16>::value;
  const dim3 grid(a.Hkv * a.P * a.MC);
  if (rows_wg == 16)
    launch((quant_narrow_kernel<T, S, D, 1>), grid, dim3(64 * kNarrowWaves), 0, st, a);
  else if (rows_wg == 32)
    launch((quant_narrow_kernel<T, S, D, 2>), grid, dim3(64 * kNarrowWaves), 0, st, a);
  else if (rows_wg == 64)
    launch((quant_wide_kernel<T, S, D, 1, 4, true, false>), grid, dim3(256), 0, st, a);
  else if (rows_wg == 128)
    launch((quant_wide_kernel<T, S, D, 2, 4, kLo, false>), grid, dim3(256), 0, st, a);
  else
    launch((quant_wide_kernel<T, S, D, 2, 8, kLo, true>), grid, dim3(512), 0, st, a);
  if (!a.direct && !a.arrived)
    launch((tree_merge_kernel<T, D>), dim3((a.B * a.Hkv * a.M + 3) / 4), dim3(256), 0, st, static_cast<const TreeArgs&>(a));
  return hipGetLastError();
}

hipError_t launch_quant_attention(const dropkv_quant_attention_args& p, size_t* need, hipStream_t st) {
  const QuantPlan pl = quant_plan(p.B, p.Hq, p.Hkv, p.D, p.T, p.capacity);
  *need = pl.bytes;
  if (p.workspace_bytes < 0 || (size_t)p.workspace_bytes < pl.bytes) return hipSuccess;  // (the caller says so)
  QuantAttnArgs a{};
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
  a.kbuf = p.k;
  a.vbuf = p.v;
  a.ks = p.k_scale;
  a.vs = p.v_scale;
  a.ktail = p.k_tail;
  a.vtail = p.v_tail;
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
  a.tail_tiles = pl.apart ? 0 : pl.rows_wg <= 32 ? 2 : 3 + (a.T + kQBlock - 1) / kQBlock;
  a.ragged = p.n_sb != 0 && p.B > 1 && p.B <= kTreeRaggedB && pl.S > 1;
  a.direct = pl.S == 1 && !pl.apart;
  a.div_t = Div::of(a.T);
  a.scale_log2 = (float)p.scale * 1.4426950408889634f;
  char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(p.workspace) + 15) & ~(uintptr_t)15);
  if (pl.one) a.arrived = sync_counters(p.workspace, p.B * p.Hkv, &a.arrived_s);
  a.deal = reinterpret_cast<int*>(ws + kSyncBytes);
  a.part_m = reinterpret_cast<float*>(ws + kSyncBytes + kTreeDealBytes);
  a.part_l = a.part_m + pl.rows;
  a.part_o = a.part_m + ((2 * pl.rows + 3) & ~(size_t)3);
  a.out = p.out;
  a.o_sb = p.o_s[0];
  a.o_st = p.o_s[1];
  a.o_sh = p.o_s[2];
  return quant_types(p.dtype, p.store, p.D, [&](auto t, auto s, auto d) {
    return launch_quant_t<decltype(t), decltype(s), decltype(d)::value>(a, pl.rows_wg, st);
  });
}

}  // namespace dkv
