// Rows quantised as they are written to a cache in 8 bits, and read back (the
// layout: dkv_quant_dev.h).  The reference keeps its cache in the model's type
// and appends with torch.cat (dropkv_cache.py:609-620).
//
// Append: one workgroup per block of 64 rows of K or of V that the call touches,
// which takes rows before the first new one from the tail.  It holds the block in
// registers, finds the largest magnitude, and writes the block once: 2 bytes read
// and 1 written an element.  The first workgroup of a head also puts the rows of
// the last block that is not full into the tail, after it has read its own block's
// (both may be in the same half of the tail).  Bound by memory: 4 x 8 heads of 26214 rows
// of 128 (644 MB) take 115 us (5.6 TB/s), reading them back 122 (5.3).
//
// The quotient x top / a is rounded correctly in fp32 (one reciprocal a block, a
// product and a residual each element), and no other value than a tie between two
// steps rounds to that tie: x top has at most 18 significant bits and a 11, so a
// quotient that is not a tie is at least 2^-19 of itself away from one.  So q is
// that of exact arithmetic.
#include "dkv_internal.h"
#include "dkv_quant_dev.h"
#include "dkv_select_dev.h"
#include "dkv_tree_dev.h"

namespace dkv {

struct QuantStore {
  uint8_t* x8[2];   // K, V: [N, B, H, C / 64] blocks of 64 D bytes
  float* scale[2];  // [N, B, H, C / 64]
  void* tail[2];    // [N, B, H, 128, D]
};

struct QuantAppendArgs {
  QuantStore to;
  const void* src[2];  // [N, B, H, L, D], D contiguous
  int64_t s_n[2], s_b[2], s_h[2], s_l[2];
  const int* n_rows;
  int64_t n_sn, n_sb;
  const int* counts;  // [B]; null: L each
  const int* path;    // [B, L]; null: rows 0, 1, ..
  int B, H, L, C, slots;
};

// Eight elements as floats.
template <typename T>
__device__ __forceinline__ void floats8(typename Elem<T>::v8 x, float* f) {
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = static_cast<float>(x[e]);
}

template <typename T, typename S, int D>
__global__ void __launch_bounds__(256) quant_append_kernel(QuantAppendArgs a) {
  typedef typename Elem<T>::v8 v8;
  typedef uint16_t us2 __attribute__((ext_vector_type(2)));
  constexpr int UPR = D / 16, NU = kQBlock * UPR / 256;  // units of 16 elements: per row, per thread
  constexpr int kPitch = D / 4 + 1;                      // dwords per row in LDS
  __shared__ uint32_t most[4];
  __shared__ uint32_t bytes[kQBlock * kPitch];
  const int slot = blockIdx.x % a.slots, head2 = blockIdx.x / a.slots;
  const int v = head2 & 1, head = head2 >> 1;
  const int h = head % a.H, b = (head / a.H) % a.B, l = head / (a.H * a.B);
  const int n = a.n_rows[l * a.n_sn + b * a.n_sb];
  if (n < 0 || n >= a.C) return;
  const int want = a.counts ? min(max(a.counts[b], 0), a.L) : a.L;
  const int end = n + min(want, a.C - n);  // (rows past the capacity are not stored)
  const int j0 = n / kQBlock, j = j0 + slot, tid = threadIdx.x;
  const bool full = (j + 1) * kQBlock <= end;
  if (!full && slot != 0) return;
  const T* src = static_cast<const T*>(a.src[v]) + l * a.s_n[v] + b * a.s_b[v] + h * a.s_h[v];
  T* tail = static_cast<T*>(a.to.tail[v]) + (int64_t)head * kQTail * D;
  auto fresh = [&](int i) {  // the i-th new row
    const int p = a.path ? min(max(a.path[(int64_t)b * a.L + i], 0), a.L - 1) : i;
    return src + p * a.s_l[v];
  };

  if (full) {
    v8 x[2 * NU];
    us2 m2 = {0, 0};
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int u = tid + 256 * i, r = kQBlock * j + u / UPR, col = 16 * (u % UPR);
      const T* row = r < n ? tail + (r % kQTail) * D : fresh(r - n);
      x[2 * i] = tree_load8(row + col);
      x[2 * i + 1] = tree_load8(row + col + 8);
    }
#pragma unroll
    for (int i = 0; i < 2 * NU; ++i) {
      const u32x4 w = __builtin_bit_cast(u32x4, x[i]) & 0x7fff7fffu;
#pragma unroll
      for (int e = 0; e < 4; ++e) m2 = __builtin_elementwise_max(m2, __builtin_bit_cast(us2, (uint32_t)w[e]));
    }
    // (As whole numbers magnitudes keep their order, infinities and NaN above all.)
    const uint32_t wave_most = wave_reduce_max((uint32_t)max(m2[0], m2[1]));
    if ((tid & 63) == 0) most[tid >> 6] = wave_most;
    __syncthreads();
    const uint16_t bits = (uint16_t)max(max(most[0], most[1]), max(most[2], most[3]));
    const T at = __builtin_bit_cast(T, bits);
    const float top = kQTop<S>, big = static_cast<float>(at);
    // A block that holds a value that is not finite comes back as NaN; magnitudes
    // below 2^-100 (where 1 / a would leave fp32's range) as zeros.
    const bool odd = not_finite(at), none = odd || big < 0x1p-100f;
    const float scale = odd ? __builtin_nanf("") : none ? 0.f : big / top;
    // a and x by the same power of two, a in [2, 4).
    const float pow2 = __uint_as_float((255u - (__float_as_uint(none ? 1.f : big) >> 23)) << 23);
    const float den = none ? 2.f : big * pow2, inv = 1.f / den, mul = none ? 0.f : pow2 * top;
    uint32_t q[4 * NU];
#pragma unroll
    for (int i = 0; i < 2 * NU; ++i) {
      float f[8];
      floats8<T>(x[i], f);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float num = none ? 0.f : f[e] * mul, q0 = num * inv;
        f[e] = fmaf(fmaf(-q0, den, num), inv, q0);
      }
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const float* g = f + 4 * w;
        if (std::is_same<S, Int8>::value) {
          // (Rounded to a whole number in the low bits of a float of that size.)
          constexpr float kRound = 12582912.f;
          uint32_t c[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) c[e] = __float_as_uint(g[e] + kRound);
          const uint32_t lo = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400), hi = __builtin_amdgcn_perm(c[3], c[2], 0x04000c0c);
          q[2 * i + w] = lo | hi;
        } else {
          q[2 * i + w] = __builtin_amdgcn_cvt_pk_fp8_f32(g[2], g[3], __builtin_amdgcn_cvt_pk_fp8_f32(g[0], g[1], 0, false), true);
        }
      }
    }
    const int64_t block = (int64_t)head * (a.C / kQBlock) + j;
    uint8_t* out = a.to.x8[v] + block * (kQBlock * D);
    if (tid == 0) a.to.scale[v][block] = scale;
    if (v == 0) {
#pragma unroll
      for (int i = 0; i < NU; ++i)
        *reinterpret_cast<u32x4*>(out + 16 * (tid + 256 * i)) = u32x4{q[4 * i], q[4 * i + 1], q[4 * i + 2], q[4 * i + 3]};
    } else {
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int u = tid + 256 * i;
#pragma unroll
        for (int e = 0; e < 4; ++e) bytes[(u / UPR) * kPitch + 4 * (u % UPR) + e] = q[4 * i + e];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < NU; ++i) {
        const int t = tid + 256 * i, kg = t % 16, cg = t / 16;
        uint32_t r[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = bytes[(4 * kg + e) * kPitch + cg];
        transpose4(r);
#pragma unroll
        for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(out + (4 * cg + e) * kQBlock + 4 * kg) = r[e];
      }
    }
  }
  if (slot != 0) return;
  __syncthreads();  // (the tail's rows of the block have been read)
  const int first = max(n, end / kQBlock * kQBlock);
  constexpr int CPR = D / 8;
  for (int x = tid; x < (end - first) * CPR; x += 256) {
    const int r = first + x / CPR, col = 8 * (x % CPR);
    *reinterpret_cast<v8*>(tail + (r % kQTail) * D + col) = tree_load8(fresh(r - n) + col);
  }
}

struct QuantReadArgs {
  QuantStore from;
  void* out[2];  // [N, B, H, L, D] contiguous
  const int* n_rows;
  int64_t n_sn, n_sb;
  int B, H, L, C, row0, slots;
};

// One workgroup per block of K or of V: 1 byte read and 2 written an element.
// V's bytes are transposed in LDS.
template <typename T, typename S, int D>
__global__ void __launch_bounds__(256) quant_read_kernel(QuantReadArgs a) {
  typedef typename Elem<T>::v8 v8;
  constexpr int UPR = D / 16, NU = kQBlock * UPR / 256, kPitch = D / 4 + 1;
  __shared__ uint32_t bytes[kQBlock * kPitch];
  const int slot = blockIdx.x % a.slots, head2 = blockIdx.x / a.slots;
  const int v = head2 & 1, head = head2 >> 1, b = (head / a.H) % a.B, l = head / (a.H * a.B);
  const int n = min(max(a.n_rows[l * a.n_sn + b * a.n_sb], 0), a.C);
  const int j = a.row0 / kQBlock + slot, tid = threadIdx.x;
  const bool full = (j + 1) * kQBlock <= n;
  const int64_t block = (int64_t)head * (a.C / kQBlock) + j;
  const uint8_t* x8 = a.from.x8[v] + block * (kQBlock * D);
  const T* tail = static_cast<const T*>(a.from.tail[v]) + (int64_t)head * kQTail * D;
  T* out = static_cast<T*>(a.out[v]) + (int64_t)head * a.L * D;
  if (full && v) {
#pragma unroll
    for (int i = 0; i < NU; ++i) {
      const int t = tid + 256 * i, kg = t % 16, cg = t / 16;
      uint32_t r[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = *reinterpret_cast<const uint32_t*>(x8 + (4 * cg + e) * kQBlock + 4 * kg);
      transpose4(r);
#pragma unroll
      for (int e = 0; e < 4; ++e) bytes[(4 * kg + e) * kPitch + cg] = r[e];
    }
    __syncthreads();
  }
  const float scale = full ? a.from.scale[v][block] : 0.f;
#pragma unroll
  for (int i = 0; i < NU; ++i) {
    const int u = tid + 256 * i, r = kQBlock * j + u / UPR, col = 16 * (u % UPR);
    if (r < a.row0 || r >= a.row0 + a.L) continue;
    v8 y[2] = {};
    if (full) {
      uint32_t w[4];
      if (v) {
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = bytes[(u / UPR) * kPitch + 4 * (u % UPR) + e];
      } else {
        const u32x4 x = *reinterpret_cast<const u32x4*>(x8 + 16 * u);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = x[e];
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        float f[4];
        unpack_f32<S>(w[e], f);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[e / 2][4 * (e % 2) + k] = static_cast<T>(f[k] * scale);
      }
    } else if (r < n) {
      y[0] = *reinterpret_cast<const v8*>(tail + (r % kQTail) * D + col);
      y[1] = *reinterpret_cast<const v8*>(tail + (r % kQTail) * D + col + 8);
    }
    T* to = out + (int64_t)(r - a.row0) * D + col;
    *reinterpret_cast<v8*>(to) = y[0];
    *reinterpret_cast<v8*>(to + 8) = y[1];
  }
}

hipError_t launch_quant_append(const dropkv_quant_append_args& p, hipStream_t st) {
  QuantAppendArgs a{};
  a.to = QuantStore{{static_cast<uint8_t*>(p.k), static_cast<uint8_t*>(p.v)}, {p.k_scale, p.v_scale}, {p.k_tail, p.v_tail}};
  a.src[0] = p.k_new;
  a.src[1] = p.v_new;
  for (int v = 0; v < 2; ++v) {
    const int64_t* s = v ? p.vn_s : p.kn_s;
    a.s_n[v] = s[0];
    a.s_b[v] = s[1];
    a.s_h[v] = s[2];
    a.s_l[v] = s[3];
  }
  a.n_rows = p.n_rows;
  a.n_sn = p.n_s[0];
  a.n_sb = p.n_s[1];
  a.counts = p.counts;
  a.path = p.path;
  a.B = (int)p.B;
  a.H = (int)p.H;
  a.L = (int)p.L;
  a.C = (int)p.capacity;
  // (n % 64 rows of a block, then L: so many blocks can be filled up.)
  a.slots = (int)std::max<int64_t>(1, (kQBlock - 1 + p.L) / kQBlock);
  const dim3 grid((unsigned)(2 * p.N * p.B * p.H * a.slots));
  return quant_types(p.dtype, p.store, p.D, [&](auto t, auto s, auto d) {
    launch((quant_append_kernel<decltype(t), decltype(s), decltype(d)::value>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
  });
}

hipError_t launch_quant_read(const dropkv_quant_read_args& p, hipStream_t st) {
  QuantReadArgs a{};
  a.from = QuantStore{{static_cast<uint8_t*>(const_cast<void*>(p.k)), static_cast<uint8_t*>(const_cast<void*>(p.v))},
                      {const_cast<float*>(p.k_scale), const_cast<float*>(p.v_scale)},
                      {const_cast<void*>(p.k_tail), const_cast<void*>(p.v_tail)}};
  a.out[0] = p.k_out;
  a.out[1] = p.v_out;
  a.n_rows = p.n_rows;
  a.n_sn = p.n_s[0];
  a.n_sb = p.n_s[1];
  a.B = (int)p.B;
  a.H = (int)p.H;
  a.L = (int)p.L;
  a.C = (int)p.capacity;
  a.row0 = (int)p.row0;
  a.slots = (int)((p.row0 + p.L - 1) / kQBlock - p.row0 / kQBlock + 1);
  const dim3 grid((unsigned)(2 * p.N * p.B * p.H * a.slots));
  return quant_types(p.dtype, p.store, p.D, [&](auto t, auto s, auto d) {
    launch((quant_read_kernel<decltype(t), decltype(s), decltype(d)::value>), grid, dim3(256), 0, st, a);
    return hipGetLastError();
  });
}

}  // namespace dkv
