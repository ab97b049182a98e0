// Norms before and after a block, fused with the block's gate and residual scale:
//   h = N_post(y) (or y);  h *= gate or sigmoid(gate);  x' = x + scale h;  z = N_pre(x')
// with N(v) = (v - mean) / sqrt(var + eps) w + b (layer) or
// v / sqrt(mean(v^2) + eps) w (rms) over a row's channels.
//
// A row stays in registers between its one read and its one write.  Statistics
// are f32, the variance from the deviations from the mean (a second pass over the
// registers); z is the norm of x' before x' is rounded to the stream's type.
// Bound by memory; a row is one wave's up to 2048 channels (no barrier), 4 up to
// 8192, 16 up to 16384.  52,640 rows of 1024 channels, f32 stream and bf16 block, both norms
// and a gate: 125 us, 5.2 TB/s; 126 rows in bf16: 4 us, most of it the launch.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sfe_internal.hpp"
#include "sfe_ops.hpp"

namespace sfe {
namespace {

template <typename T, int N>
struct alignas(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Vec {
  T v[N];
};

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// Sum over the row's WAVES waves, in one order for every thread.
template <int WAVES>
__device__ __forceinline__ float row_sum(float x, float* lds, int slot) {
  x = wave_sum(x);
  if constexpr (WAVES > 1) {
    float* p = lds + slot * WAVES;
    if ((threadIdx.x & 63) == 0) p[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0.0f;
#pragma unroll
    for (int i = 0; i < WAVES; ++i) x += p[i];
  }
  return x;
}

// A row's values in registers: NV vectors of N channels a lane, vector j of
// lane l at (j * lanes + l) * N.  Normalised in place; slot: row_sum slots used.
// LAYER: the kind may be a layer norm; the mean is then selected or zero
// (a branch over the three kinds came out of the compiler with the rms norm's
// values undefined).
template <bool LAYER, int WAVES, int N, int NV>
__device__ __forceinline__ void norm_row(float (&v)[NV][N], int kind, const float* w, const float* b, int width,
                                         float eps, int lane, float* lds, int slot) {
  constexpr int kLanes = 64 * WAVES;
  float mean = 0.0f;
  if constexpr (LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < N; ++i) s += v[j][i];
    mean = row_sum<WAVES>(s, lds, slot) / (float)width;
    mean = kind == kNormLayer ? mean : 0.0f;
  }
  float s = 0.0f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if ((j * kLanes + lane) * N < width)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float d = v[j][i] - mean;
        s = __builtin_fmaf(d, d, s);
      }
  const float r = 1.0f / sqrtf(row_sum<WAVES>(s, lds, slot + 1) / (float)width + eps);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * kLanes + lane) * N;
    if (c < width) {
      const Vec<float, N> wv = *reinterpret_cast<const Vec<float, N>*>(w + c);
      Vec<float, N> bv;
#pragma unroll
      for (int i = 0; i < N; ++i) bv.v[i] = 0.0f;
      if (b) bv = *reinterpret_cast<const Vec<float, N>*>(b + c);
#pragma unroll
      for (int i = 0; i < N; ++i) v[j][i] = __builtin_fmaf((v[j][i] - mean) * r, wv.v[i], bv.v[i]);
    }
  }
}

// XT: stream, YT: block output, gate and norm.  WAVES a row; one-wave rows go 4
// to a workgroup.  Channels past the width are zero in registers.
template <typename XT, typename YT, bool LAYER, int WAVES, int N, int NV>
__global__ __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) void sfe_residual_kernel(ResidualArgs a, int64_t row0) {
  constexpr int kLanes = 64 * WAVES;
  __shared__ float lds[4 * WAVES];
  const int64_t row = row0 + (WAVES == 1 ? (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6) : (int64_t)blockIdx.x);
  if (row >= a.rows) return;
  const int lane = WAVES == 1 ? (int)(threadIdx.x & 63) : (int)threadIdx.x;
  const XT* x = reinterpret_cast<const XT*>(a.x) + row * a.x_row;
  const YT* y = reinterpret_cast<const YT*>(a.y) + row * a.y_row;
  Vec<XT, N> xv[NV];
  Vec<YT, N> yv[NV], gv[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * kLanes + lane) * N;
    if (c < a.width) {
      xv[j] = *reinterpret_cast<const Vec<XT, N>*>(x + c);
      yv[j] = *reinterpret_cast<const Vec<YT, N>*>(y + c);
      if (a.gate) gv[j] = *reinterpret_cast<const Vec<YT, N>*>(reinterpret_cast<const YT*>(a.gate) + row * a.gate_row + c);
    }
  }
  float h[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const bool in = (j * kLanes + lane) * N < a.width;
#pragma unroll
    for (int i = 0; i < N; ++i) h[j][i] = in ? (float)yv[j].v[i] : 0.0f;
  }
  if (a.post != kNormNone) norm_row<LAYER, WAVES, N, NV>(h, a.post, a.post_w, a.post_b, a.width, a.eps, lane, lds, 0);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * kLanes + lane) * N;
    if (c < a.width) {
      if (a.gate)
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float g = (float)gv[j].v[i];
          h[j][i] *= a.sigmoid ? 1.0f / (1.0f + __expf(-g)) : g;
        }
      Vec<XT, N> xo;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        h[j][i] = __builtin_fmaf(a.scale, h[j][i], (float)xv[j].v[i]);
        xo.v[i] = (XT)h[j][i];
      }
      *reinterpret_cast<Vec<XT, N>*>(reinterpret_cast<XT*>(a.xo) + row * a.xo_row + c) = xo;
    }
  }
  if (a.pre == kNormNone) return;
  norm_row<LAYER, WAVES, N, NV>(h, a.pre, a.pre_w, a.pre_b, a.width, a.eps, lane, lds, 2);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = (j * kLanes + lane) * N;
    if (c < a.width) {
      Vec<YT, N> z;
#pragma unroll
      for (int i = 0; i < N; ++i) z.v[i] = (YT)h[j][i];
      *reinterpret_cast<Vec<YT, N>*>(reinterpret_cast<YT*>(a.z) + row * a.z_row + c) = z;
    }
  }
}

template <typename XT, typename YT, int WAVES, int N, int NV>
hipError_t run(const ResidualArgs& a, hipStream_t stream) {
  const int rows = WAVES == 1 ? 4 : 1;
  return for_launches((a.rows + rows - 1) / rows, rows * 64 * WAVES, [&](int64_t first, unsigned blocks) {
    if (a.post == kNormLayer || a.pre == kNormLayer)
      sfe_residual_kernel<XT, YT, true, WAVES, N, NV><<<dim3(blocks), dim3(rows * 64 * WAVES), 0, stream>>>(a, first * rows);
    else
      sfe_residual_kernel<XT, YT, false, WAVES, N, NV><<<dim3(blocks), dim3(rows * 64 * WAVES), 0, stream>>>(a, first * rows);
    return hipGetLastError();
  });
}

template <typename XT, typename YT>
hipError_t run_types(const ResidualArgs& a, hipStream_t stream) {
  bool vec = a.width % 8 == 0;
  auto ok = [&](const void* p, int64_t row, int size) {
    if (p) vec = vec && reinterpret_cast<uintptr_t>(p) % 16 == 0 && row * size % 16 == 0;
  };
  ok(a.x, a.x_row, sizeof(XT));
  ok(a.xo, a.xo_row, sizeof(XT));
  ok(a.y, a.y_row, sizeof(YT));
  ok(a.gate, a.gate_row, sizeof(YT));
  ok(a.z, a.z_row, sizeof(YT));
  for (const float* p : {a.post_w, a.post_b, a.pre_w, a.pre_b}) ok(p, 0, 4);
  if (vec) {
    if (a.width <= 512) return run<XT, YT, 1, 8, 1>(a, stream);
    if (a.width <= 1024) return run<XT, YT, 1, 8, 2>(a, stream);
    if (a.width <= 2048) return run<XT, YT, 1, 8, 4>(a, stream);
    if (a.width <= 8192) return run<XT, YT, 4, 8, 4>(a, stream);
    return run<XT, YT, 16, 8, 2>(a, stream);
  }
  if (a.width <= 512) return run<XT, YT, 1, 1, 8>(a, stream);
  if (a.width <= 2048) return run<XT, YT, 1, 1, 32>(a, stream);
  if (a.width <= 8192) return run<XT, YT, 4, 1, 32>(a, stream);
  return run<XT, YT, 16, 1, 16>(a, stream);
}

}  // namespace

hipError_t launch_residual(const ResidualArgs& a, int stream_type, int block_type, hipStream_t stream) {
  if (stream_type == kOpF32) {
    if (block_type == kOpF32) return run_types<float, float>(a, stream);
    if (block_type == kOpBf16) return run_types<float, __bf16>(a, stream);
    return run_types<float, _Float16>(a, stream);
  }
  if (stream_type == kOpBf16) return run_types<__bf16, __bf16>(a, stream);
  return run_types<_Float16, _Float16>(a, stream);
}

}  // namespace sfe
