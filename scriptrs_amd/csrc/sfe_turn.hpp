// What the kernels that turn channel pairs share (sfe_rotary.hip, sfe_norm_rotary.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace sfe {

template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

// cos and sin of 2 pi t / 2^32.
__device__ __forceinline__ void turn_cos_sin(uint32_t t, float* c, float* s) {
  const uint32_t quadrant = (t + 0x20000000u) >> 30;  // nearest quarter turn
  const float x = (float)(int32_t)(t - (quadrant << 30)) * 1.46291807926715968e-9f;  // 2 pi / 2^32
  const float z = x * x;
  float sn = __builtin_fmaf(z, 2.75573192e-6f, -1.98412698e-4f);
  sn = __builtin_fmaf(z, sn, 8.33333333e-3f);
  sn = __builtin_fmaf(z, sn, -1.66666667e-1f);
  sn = __builtin_fmaf(z * x, sn, x);
  float cn = __builtin_fmaf(z, -2.75573192e-7f, 2.48015873e-5f);
  cn = __builtin_fmaf(z, cn, -1.38888889e-3f);
  cn = __builtin_fmaf(z, cn, 4.16666667e-2f);
  cn = __builtin_fmaf(z, cn, -0.5f);
  cn = __builtin_fmaf(z, cn, 1.0f);
  const float a = quadrant & 1 ? sn : cn, b = quadrant & 1 ? cn : sn;
  *c = (quadrant + 1) & 2 ? -a : a;
  *s = quadrant & 2 ? -b : b;
}

}  // namespace sfe
