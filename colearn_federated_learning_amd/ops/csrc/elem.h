// Element access of the encoder-training kernels: fp32, bf16 and fp16 memory,
// fp32 registers.  Conversions to 16 bits are the hardware's, to nearest even,
// and keep NaN.
#pragma once

#include "common.h"

namespace colearn {

using f16 = _Float16;

template <typename T>
struct Bits16;
template <>
struct Bits16<bf16> {
  using hw = __bf16;
};
template <>
struct Bits16<f16> {
  using hw = _Float16;
};

DEV_INLINE float elem_load(const float* p) { return *p; }
DEV_INLINE float elem_load(const bf16* p) {
  return bits2f(*reinterpret_cast<const short*>(p));
}
DEV_INLINE float elem_load(const f16* p) { return static_cast<float>(*p); }
DEV_INLINE void elem_store(float* p, float x) { *p = x; }
DEV_INLINE void elem_store(bf16* p, float x) {
  *reinterpret_cast<__bf16*>(p) = static_cast<__bf16>(x);
}
DEV_INLINE void elem_store(f16* p, float x) { *p = static_cast<f16>(x); }

// four neighbours at once: 16 bytes of fp32, 8 of the others
DEV_INLINE void elem_load4(const float* p, float* x) {
  const float4 v = *reinterpret_cast<const float4*>(p);
  x[0] = v.x;
  x[1] = v.y;
  x[2] = v.z;
  x[3] = v.w;
}
template <typename T>
DEV_INLINE void elem_load4(const T* p, float* x) {
  typedef __attribute__((ext_vector_type(4))) typename Bits16<T>::hw V;
  const V v = *reinterpret_cast<const V*>(p);
#pragma unroll
  for (int j = 0; j < 4; ++j) x[j] = static_cast<float>(v[j]);
}
DEV_INLINE void elem_store4(float* p, const float* x) {
  *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
}
template <typename T>
DEV_INLINE void elem_store4(T* p, const float* x) {
  typedef __attribute__((ext_vector_type(4))) typename Bits16<T>::hw V;
  typedef __attribute__((ext_vector_type(4))) float F;
  const F f = {x[0], x[1], x[2], x[3]};
  *reinterpret_cast<V*>(p) = __builtin_convertvector(f, V);
}

// x rounded to T and back
DEV_INLINE float elem_round(float x, const float*) { return x; }
DEV_INLINE float elem_round(float x, const bf16*) {
  return static_cast<float>(static_cast<__bf16>(x));
}
DEV_INLINE float elem_round(float x, const f16*) {
  return static_cast<float>(static_cast<f16>(x));
}

// ---- wave reductions in registers -------------------------------------------
// Every lane gets the result; no LDS and no lane index arithmetic.  Exchanges
// within 16 lanes are DPP moves (xor 1, xor 2, mirrored halves, mirrored row:
// after each, the lanes that were joined agree), the last two swap rows.
template <int CTRL>
DEV_INLINE float dpp_move(float v) {
  return __int_as_float(
      __builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true));
}
DEV_INLINE float swap32(float v) {  // lane ^ 32
  const auto r = __builtin_amdgcn_permlane32_swap(
      __float_as_int(v), __float_as_int(v), false, false);
  return __int_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}
DEV_INLINE float lanes_sum(float v) {
  v += dpp_move<0xB1>(v);
  v += dpp_move<0x4E>(v);
  v += dpp_move<0x141>(v);
  v += dpp_move<0x140>(v);
  // a swap returns both sides: their sum is the same in either lane
  const auto a = __builtin_amdgcn_permlane16_swap(
      __float_as_int(v), __float_as_int(v), false, false);
  v = __int_as_float(a[0]) + __int_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(
      __float_as_int(v), __float_as_int(v), false, false);
  return __int_as_float(b[0]) + __int_as_float(b[1]);
}
DEV_INLINE float lanes_max(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  v = fmaxf(v, dpp_move<0x140>(v));
  const auto a = __builtin_amdgcn_permlane16_swap(
      __float_as_int(v), __float_as_int(v), false, false);
  v = fmaxf(__int_as_float(a[0]), __int_as_float(a[1]));
  const auto b = __builtin_amdgcn_permlane32_swap(
      __float_as_int(v), __float_as_int(v), false, false);
  return fmaxf(__int_as_float(b[0]), __int_as_float(b[1]));
}

}  // namespace colearn
