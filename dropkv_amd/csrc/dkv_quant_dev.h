// A cache in 8 bits: its layout and its values.
//
// Per (layer, batch, KV head) the rows lie in blocks of 64, and each block has one
// scale s for K and one for V: a stored q stands for s q, with
//   a = max |x| over the block,  s = a / top,  q = round(x top / a)
// to the nearest, ties to even; top is 127 for int8 and 448 for e4m3.  Only full
// blocks are stored so.  Rows of the last block, while it is not full, stay in 16
// bits, row r at r % 128 of the tail: every row is rounded once, whatever the
// lengths it was appended in, and a block that fills up leaves its 16-bit rows
// where they are until the block after next.
//
//   K  row-major [64][D]: a row's 16 bytes are a lane's share of the matrix operand
//      of two products
//   V  transposed [D][64] within the block: 16 bytes are 16 keys of one column, and
//      so too the operand of two products, with no transposing reads
#pragma once

#include "dkv_common.h"
#include "dkv_internal.h"

#include <type_traits>

namespace dkv {

constexpr int kQBlock = 64;
constexpr int kQTail = 2 * kQBlock;

struct Int8 {};
struct E4m3 {};
template <typename S>
constexpr float kQTop = std::is_same<S, Int8>::value ? 127.f : 448.f;

// Four stored values as the element type (exact: they have at most eight
// significant bits).
template <typename S, typename T>
struct Unpack;
template <typename T>
struct Pair {
  typedef T v2 __attribute__((ext_vector_type(2)));
};
template <>
struct Unpack<E4m3, __bf16> {
  static __device__ __forceinline__ u32x2 four(uint32_t w) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))};
  }
};
template <>
struct Unpack<E4m3, _Float16> {
  static __device__ __forceinline__ u32x2 four(uint32_t w) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, true))};
  }
};
template <typename T>
struct Unpack<Int8, T> {
  static __device__ __forceinline__ u32x2 four(uint32_t w) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = {(float)(int8_t)w, (float)(int8_t)(w >> 8)}, hi = {(float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24)};
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_convertvector(lo, typename Pair<T>::v2)),
                 __builtin_bit_cast(uint32_t, __builtin_convertvector(hi, typename Pair<T>::v2))};
  }
};
// The operand of one product: bytes 8 h .. 8 h + 7 of a lane's 16.
template <typename S, typename T>
__device__ __forceinline__ typename Elem<T>::v8 unpack8(u32x4 x, int h) {
  const u32x2 a = Unpack<S, T>::four(x[2 * h]), b = Unpack<S, T>::four(x[2 * h + 1]);
  return bitcast_u4<typename Elem<T>::v8>(u32x4{a[0], a[1], b[0], b[1]});
}

// The same as floats.
template <typename S>
__device__ __forceinline__ void unpack_f32(uint32_t w, float* f) {
  if (std::is_same<S, Int8>::value) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = (float)(int8_t)(w >> (8 * i));
  } else {
    f[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0);
    f[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1);
    f[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2);
    f[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3);
  }
}

// Four rows of four bytes to four columns, and back.
__device__ __forceinline__ void transpose4(uint32_t* r) {
  const uint32_t ab02 = __builtin_amdgcn_perm(r[1], r[0], 0x06020400), ab13 = __builtin_amdgcn_perm(r[1], r[0], 0x07030501);
  const uint32_t cd02 = __builtin_amdgcn_perm(r[3], r[2], 0x06020400), cd13 = __builtin_amdgcn_perm(r[3], r[2], 0x07030501);
  r[0] = __builtin_amdgcn_perm(cd02, ab02, 0x05040100);
  r[1] = __builtin_amdgcn_perm(cd13, ab13, 0x05040100);
  r[2] = __builtin_amdgcn_perm(cd02, ab02, 0x07060302);
  r[3] = __builtin_amdgcn_perm(cd13, ab13, 0x07060302);
}

// A call's kernel by its types: f(T, S, D).
template <typename T, typename F>
inline hipError_t quant_stores(int64_t store, int64_t D, F&& f) {
  constexpr std::integral_constant<int, 64> d64{};
  constexpr std::integral_constant<int, 128> d128{};
  if (store == kStoreInt8) return D == 64 ? f(T{}, Int8{}, d64) : f(T{}, Int8{}, d128);
  return D == 64 ? f(T{}, E4m3{}, d64) : f(T{}, E4m3{}, d128);
}
template <typename F>
inline hipError_t quant_types(int64_t dtype, int64_t store, int64_t D, F&& f) {
  return dtype == kDtypeBf16 ? quant_stores<__bf16>(store, D, f) : quant_stores<_Float16>(store, D, f);
}

}  // namespace dkv
