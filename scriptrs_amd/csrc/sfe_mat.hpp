// Matrix instructions, loads into LDS and the softmax's small parts, shared by the attention kernels
// (sfe_attn.hip, sfe_cache_attn.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sfe {

typedef __bf16 Bf;
typedef _Float16 Hf;
typedef float F2 __attribute__((ext_vector_type(2)));
typedef float F4 __attribute__((ext_vector_type(4)));
typedef float F16 __attribute__((ext_vector_type(16)));
typedef int I4 __attribute__((ext_vector_type(4)));
typedef short S4 __attribute__((ext_vector_type(4)));
typedef short S8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Mat;
template <>
struct Mat<Bf> {
  typedef Bf V8 __attribute__((ext_vector_type(8)));
  typedef Bf V2 __attribute__((ext_vector_type(2)));
  static __device__ F16 m32(V8 a, V8 b, F16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ F4 m16(V8 a, V8 b, F4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static constexpr uint32_t kExp = 0x7f807f80, kCarry = 0x00800080, kOne = 0x3f80;
  // the reference moves when a score passes it by kRise, to kBelow below the maximum
  static constexpr float kRise = 0.0f, kBelow = -8.0f;
};
template <>
struct Mat<Hf> {
  typedef Hf V8 __attribute__((ext_vector_type(8)));
  typedef Hf V2 __attribute__((ext_vector_type(2)));
  static __device__ F16 m32(V8 a, V8 b, F16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ F4 m16(V8 a, V8 b, F4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static constexpr uint32_t kExp = 0x7c007c00, kCarry = 0x04000400, kOne = 0x3c00;
  static constexpr float kRise = 15.0f, kBelow = 7.0f;
};

constexpr float kNever = -3e38f;  // reference exponent before the first visible key: below every score that counts
// Scores past this are scaled and rounded before the reference is taken off: the f32 reference of such
// a row is a rounded score itself, and exact products less it would be off by its rounding.
constexpr float kLarge = 1048576.0f;
constexpr uint32_t kOutside = 0x80000000u;  // an offset past every buffer's range
constexpr int kBufWord3 = 0x00020000;

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

// 16 bytes a lane from buffer offset `off` (a lane's own) into LDS at `lds` +
// 16 * lane.  Completion is waited for with vmcnt.
__device__ __forceinline__ void load_lds(I4 buf, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(buf)
               : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// s * c rounded, less m (never one fused operation).
__device__ __forceinline__ float scaled_less(float s, float c, float m) {
#pragma clang fp contract(off)
  const float x = s * c;
  return x - m;
}

// a - b, where a is a rounded product already (never one fused operation with it: the reference b of a row of large scores is
// such a product, and an exact one less it would be off by its rounding).
__device__ __forceinline__ float rounded_less(float a, float b) {
#pragma clang fp contract(off)
  return a - b;
}

// The larger (sum) of this lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_halves(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// Whether any of a V operand's 8 values is infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t nonfinite(typename Mat<T>::V8 v) {
  const I4 w = __builtin_bit_cast(I4, v);
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= ((uint32_t)w[i] & Mat<T>::kExp) + Mat<T>::kCarry;
  return bad & 0x80008000u;
}

// A V operand with infinite or NaN values, of keys that some queries see and
// others do not: *clean has zeros for them, *pos and *neg ones where a query that sees
// the key has to get +inf or -inf (both: NaN).
template <typename T>
__device__ __forceinline__ void split_nonfinite(S8 v, S8* clean, S8* pos, S8* neg) {
  constexpr uint32_t e = Mat<T>::kExp & 0xffff;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t x = (uint16_t)v[j];
    const bool bad = (x & e) == e, nan = bad && (x & 0x7fff) != e;
    (*clean)[j] = bad ? 0 : v[j];
    (*pos)[j] = bad && (nan || !(x & 0x8000)) ? Mat<T>::kOne : 0;
    (*neg)[j] = bad && (nan || (x & 0x8000)) ? Mat<T>::kOne : 0;
  }
}

}  // namespace sfe
