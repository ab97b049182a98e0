// Rotary positions.
//
// A pair of channels (a, b) of a head turns by angle = position * f_p:
//   a' = m (a cos - b sin),  b' = m (b cos + a sin)
// (m: the magnitude of a table scaled for long contexts).  Pairs are (p, p +
// R/2) (half) or (2p, 2p + 1) (interleaved) of the first R channels; the others
// are copied.
//
// The angle of a far position has to be exact modulo a turn: f_p is held as a
// fraction of a turn in 64 bits and multiplied by the position modulo 2^64, so
// whole turns drop out and the top 32 bits are the turn's fraction, correct to
// 2^-32 at any 32-bit position (in f32, position * f_p would be off by 3e-3
// rad at 45,000).  Sine and cosine are their power series over an eighth of a
// turn to either side, in f32 (error below 1e-7).
//
// Bound by memory: each element is read and written once.  A thread takes 16
// bytes of each channel of a pair and walks a share of the row's heads with
// the same 4 or 8 sines and cosines.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sfe_internal.hpp"
#include "sfe_ops.hpp"

namespace sfe {
namespace {

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

constexpr int kRotaryThreads = 256;

// N: elements of a vector.  A unit is (row, slot, share of heads); slots
// 0..turning - 1 hold N pairs each (half: two vectors R/2 apart; interleaved:
// two consecutive vectors), the rest one vector of copied channels.
template <typename T, int N, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void sfe_rotary_kernel(RotaryArgs a, int64_t unit0, int64_t units,
                                                                    int slots, int shares) {
  const int64_t u = unit0 + (int64_t)blockIdx.x * kRotaryThreads + threadIdx.x;
  if (u >= units) return;
  const int slot = (int)(u % slots);
  const int64_t rest = u / slots;
  const int share = (int)(rest % shares);
  const int64_t row = rest / shares;
  const int turning = a.rotary / 2 / N;
  const bool turn = slot < turning;
  int d0, d1 = 0;
  if (turn) {
    d0 = INTERLEAVED ? 2 * N * slot : N * slot;
    d1 = INTERLEAVED ? d0 + N : d0 + a.rotary / 2;
  } else {
    d0 = a.rotary + N * (slot - turning);
  }
  float cs[N], sn[N];
  if (turn) {
    const uint64_t at = (uint64_t)(int64_t)a.positions[row];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      turn_cos_sin((uint32_t)((at * a.step[N * slot + i]) >> 32), &cs[i], &sn[i]);
      cs[i] *= a.magnitude;
      sn[i] *= a.inverse ? -a.magnitude : a.magnitude;
    }
  }
  const int heads = a.t[0].heads + a.t[1].heads;
  for (int h = share; h < heads; h += shares) {
    const bool second = h >= a.t[0].heads;
    const RotaryTensor& t = a.t[second];
    const int hh = second ? h - a.t[0].heads : h;
    const T* x = reinterpret_cast<const T*>(t.x) + row * t.x_row + hh * t.x_head;
    T* y = reinterpret_cast<T*>(t.y) + row * t.y_row + hh * t.y_head;
    typedef Vec<T, N> V;
    if (!turn) {
      if (x != y) *reinterpret_cast<V*>(y + d0) = *reinterpret_cast<const V*>(x + d0);
      continue;
    }
    const V p = *reinterpret_cast<const V*>(x + d0), q = *reinterpret_cast<const V*>(x + d1);
    V r, w;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (INTERLEAVED) {
        // values 2i and 2i + 1 of the two vectors
        const float e = (float)(2 * i < N ? p.v[(2 * i) % N] : q.v[(2 * i) % N]);
        const float f = (float)(2 * i < N ? p.v[(2 * i + 1) % N] : q.v[(2 * i + 1) % N]);
        const T ye = (T)__builtin_fmaf(e, cs[i], -f * sn[i]), yf = (T)__builtin_fmaf(f, cs[i], e * sn[i]);
        if (2 * i < N) {
          r.v[(2 * i) % N] = ye;
          r.v[(2 * i + 1) % N] = yf;
        } else {
          w.v[(2 * i) % N] = ye;
          w.v[(2 * i + 1) % N] = yf;
        }
      } else {
        const float e = (float)p.v[i], f = (float)q.v[i];
        r.v[i] = (T)__builtin_fmaf(e, cs[i], -f * sn[i]);
        w.v[i] = (T)__builtin_fmaf(f, cs[i], e * sn[i]);
      }
    }
    *reinterpret_cast<V*>(y + d0) = r;
    *reinterpret_cast<V*>(y + d1) = w;
  }
}

// The same a pair at a time, for tensors whose vectors are not aligned or whose
// R is no multiple of them.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(kRotaryThreads) void sfe_rotary_pairs_kernel(RotaryArgs a, int64_t unit0, int64_t units,
                                                                          int slots, int shares) {
  const int64_t u = unit0 + (int64_t)blockIdx.x * kRotaryThreads + threadIdx.x;
  if (u >= units) return;
  const int slot = (int)(u % slots);
  const int64_t rest = u / slots;
  const int share = (int)(rest % shares);
  const int64_t row = rest / shares;
  const int half = a.rotary / 2;
  const bool turn = slot < half;
  const int d0 = turn ? (INTERLEAVED ? 2 * slot : slot) : a.rotary + (slot - half);
  const int d1 = INTERLEAVED ? d0 + 1 : d0 + half;
  float c = 0.0f, s = 0.0f;
  if (turn) {
    turn_cos_sin((uint32_t)(((uint64_t)(int64_t)a.positions[row] * a.step[slot]) >> 32), &c, &s);
    c *= a.magnitude;
    s *= a.inverse ? -a.magnitude : a.magnitude;
  }
  const int heads = a.t[0].heads + a.t[1].heads;
  for (int h = share; h < heads; h += shares) {
    const bool second = h >= a.t[0].heads;
    const RotaryTensor& t = a.t[second];
    const int hh = second ? h - a.t[0].heads : h;
    const T* x = reinterpret_cast<const T*>(t.x) + row * t.x_row + hh * t.x_head;
    T* y = reinterpret_cast<T*>(t.y) + row * t.y_row + hh * t.y_head;
    if (!turn) {
      y[d0] = x[d0];
      continue;
    }
    const float e = (float)x[d0], f = (float)x[d1];
    y[d0] = (T)__builtin_fmaf(e, c, -f * s);
    y[d1] = (T)__builtin_fmaf(f, c, e * s);
  }
}

template <typename T, bool INTERLEAVED>
hipError_t run(const RotaryArgs& a, int cus, hipStream_t stream) {
  constexpr int N = 16 / (int)sizeof(T);
  bool vec = a.rotary % (2 * N) == 0 && a.dim % N == 0;
  for (const RotaryTensor& t : a.t)
    if (t.heads)
      vec = vec && (reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.y)) % 16 == 0 &&
            (t.x_row | t.x_head | t.y_row | t.y_head) % N == 0;
  const int step = vec ? N : 1;
  const int slots = a.rotary / 2 / step + (a.dim - a.rotary) / step;
  const int heads = a.t[0].heads + a.t[1].heads;
  // Heads of a row are shared out among threads until about 8 waves a CU are there.
  const int64_t want = (int64_t)cus * 8 * 64, have = a.rows * slots;
  const int shares = (int)(have >= want ? 1 : (heads < (want + have - 1) / have ? heads : (want + have - 1) / have));
  const int64_t units = have * shares;
  return for_launches((units + kRotaryThreads - 1) / kRotaryThreads, kRotaryThreads, [&](int64_t first, unsigned blocks) {
    const int64_t unit0 = first * kRotaryThreads;
    if (vec)
      sfe_rotary_kernel<T, N, INTERLEAVED><<<dim3(blocks), dim3(kRotaryThreads), 0, stream>>>(a, unit0, units, slots, shares);
    else
      sfe_rotary_pairs_kernel<T, INTERLEAVED><<<dim3(blocks), dim3(kRotaryThreads), 0, stream>>>(a, unit0, units, slots, shares);
    return hipGetLastError();
  });
}

template <typename T>
hipError_t run_layout(const RotaryArgs& a, bool interleaved, int cus, hipStream_t stream) {
  return interleaved ? run<T, true>(a, cus, stream) : run<T, false>(a, cus, stream);
}

}  // namespace

hipError_t launch_rotary(const RotaryArgs& a, int type, bool interleaved, int cus, hipStream_t stream) {
  if (type == kOpF32) return run_layout<float>(a, interleaved, cus, stream);
  if (type == kOpBf16) return run_layout<__bf16>(a, interleaved, cus, stream);
  return run_layout<_Float16>(a, interleaved, cus, stream);
}

}  // namespace sfe
