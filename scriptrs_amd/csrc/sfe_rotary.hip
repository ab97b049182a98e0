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
// 2^-31 at any 32-bit position: 2^-32 for the bits that are cut off and less than
// that for the step, which is off by half a unit and 2^-61 of it (in f32, position *
// f_p would be off by 3e-3 rad at 45,000).  Sine and cosine are their power series over an eighth of a
// turn to either side, in f32 (error below 1e-7).
//
// Bound by memory: each element is read and written once, and a row's sines and
// cosines are computed once for all of its heads.  52,640 rows of 2 x 8 heads of 128 in bf16:
// 89 us, 4.85 TB/s, the rate of a large copy; 64 rows of 20 heads: 3.6 us, most of it the launch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

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
constexpr int kRotaryTable = 4096;  // (cosine, sine) of a workgroup's rows and pairs

// A workgroup takes RB times `per` rows: their sines and cosines go into LDS, then
// a thread keeps its place in a row (head and channels) and turns it in RB rows,
// all RB loads issued before the first store (outputs may be the inputs, so the
// compiler cannot move loads past stores).  Places of a row, `places`: for each
// head turning units, then copied ones.  N > 1: a unit is 16 bytes of N channels:
// half, two vectors R/2 apart; interleaved, one vector of N / 2 pairs; 8 bytes where 16 do not divide
// the parts or are not aligned (52,640 rows of 2 x 8 heads of 80 in bf16, 40 turned in halves: 78 us, 198 by
// the pair; 80 turned, of 16 bytes, 54).  N = 1: a pair, or a copied channel (tensors whose
// vectors are not aligned).
template <typename T, int N, bool INTERLEAVED, int RB>
__global__ __launch_bounds__(kRotaryThreads) void sfe_rotary_kernel(RotaryArgs a, int64_t first, uint32_t places,
                                                                    uint32_t slots, uint32_t chunks, uint32_t per) {
  constexpr bool kOne = INTERLEAVED && N > 1;  // both channels of a pair in one vector
  constexpr int kPairs = kOne ? N / 2 : N;     // of a unit
  typedef Vec<T, N> V;
  __shared__ float2 table[kRotaryTable];
  const uint32_t group = blockIdx.x / chunks, chunk = blockIdx.x - group * chunks;
  const int64_t row0 = first + (int64_t)group * RB * per;
  const int pairs = a.rotary / 2, t = (int)threadIdx.x;
  const int rows = (int)(a.rows - row0 < (int64_t)(RB * per) ? a.rows - row0 : (int64_t)(RB * per));
  const float m = a.magnitude, ms = a.inverse ? -a.magnitude : a.magnitude;
  for (int e = t; e < rows * pairs; e += kRotaryThreads) {
    const int r = (int)((unsigned)e / (unsigned)pairs), p = e - r * pairs;
    float c, s;
    turn_cos_sin((uint32_t)(((uint64_t)(int64_t)a.positions[row0 + r] * a.step[p]) >> 32), &c, &s);
    table[e] = make_float2(m * c, ms * s);
  }
  __syncthreads();
  const uint32_t in = per > 1 ? (uint32_t)t / places : 0;  // row within a pass
  const uint32_t place = per > 1 ? (uint32_t)t - in * places : chunk * kRotaryThreads + (uint32_t)t;
  if (place >= places || in >= per) return;
  const int head = (int)(place / slots), slot = (int)(place - (uint32_t)head * slots);
  const int turning = pairs / kPairs;
  const bool turn = slot < turning;
  const int d0 = turn ? slot * (INTERLEAVED ? 2 * kPairs : kPairs) : a.rotary + N * (slot - turning);
  const int d1 = INTERLEAVED ? d0 + 1 : d0 + pairs;  // (not of one vector)
  const bool second = head >= a.t[0].heads;
  const RotaryTensor& tn = a.t[second];
  const int h = second ? head - a.t[0].heads : head;
  const T* x = reinterpret_cast<const T*>(tn.x) + (row0 + in) * tn.x_row + h * tn.x_head;
  T* y = reinterpret_cast<T*>(tn.y) + (row0 + in) * tn.y_row + h * tn.y_head;
  V p[RB], q[RB];
#pragma unroll
  for (int k = 0; k < RB; ++k)
    if ((int)(in + k * per) < rows) {
      p[k] = *reinterpret_cast<const V*>(x + k * (int64_t)per * tn.x_row + d0);
      if (!kOne && turn) q[k] = *reinterpret_cast<const V*>(x + k * (int64_t)per * tn.x_row + d1);
    }
#pragma unroll
  for (int k = 0; k < RB; ++k)
    if ((int)(in + k * per) < rows) {
      T* yk = y + k * (int64_t)per * tn.y_row;
      if (!turn) {
        *reinterpret_cast<V*>(yk + d0) = p[k];
        continue;
      }
      const float2* cs = table + (in + k * per) * pairs + slot * kPairs;
      V r, w;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float e = (float)(kOne ? p[k].v[(2 * i) % N] : p[k].v[i]), f = (float)(kOne ? p[k].v[(2 * i + 1) % N] : q[k].v[i]);
        const T ye = (T)__builtin_fmaf(e, cs[i].x, -f * cs[i].y), yf = (T)__builtin_fmaf(f, cs[i].x, e * cs[i].y);
        r.v[kOne ? (2 * i) % N : i] = ye;
        if (kOne) r.v[(2 * i + 1) % N] = yf;
        else w.v[i] = yf;
      }
      *reinterpret_cast<V*>(yk + d0) = r;
      if (!kOne) *reinterpret_cast<V*>(yk + d1) = w;
    }
}

template <typename T, int N, bool INTERLEAVED, int RB>
hipError_t run_rows(const RotaryArgs& a, uint32_t places, uint32_t slots, hipStream_t stream) {
  const uint32_t chunks = (places + kRotaryThreads - 1) / kRotaryThreads;
  const uint32_t per = chunks > 1 ? 1 : std::max(1u, std::min(kRotaryThreads / places, (uint32_t)(kRotaryTable / (RB * (a.rotary / 2)))));
  // (launches of at most 2^22 workgroups)
  const int64_t step = std::max<int64_t>(1, ((int64_t)1 << 22) / chunks) * RB * per;
  for (int64_t first = 0; first < a.rows; first += step) {
    const int64_t rows = std::min(step, a.rows - first);
    const unsigned blocks = (unsigned)((rows + RB * per - 1) / (RB * per) * chunks);
    sfe_rotary_kernel<T, N, INTERLEAVED, RB><<<dim3(blocks), dim3(kRotaryThreads), 0, stream>>>(a, first, places, slots, chunks, per);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int N, bool INTERLEAVED>
hipError_t run_units(const RotaryArgs& a, int cus, hipStream_t stream) {
  const int pairs = INTERLEAVED && N > 1 ? N / 2 : N;
  const uint32_t slots = (uint32_t)(a.rotary / 2 / pairs + (a.dim - a.rotary) / N);
  const uint32_t places = slots * (uint32_t)(a.t[0].heads + a.t[1].heads);
  // One row a thread while the machine is not full at 4 rows a thread.
  const bool many = a.rows * places >= (int64_t)cus * 8 * kRotaryThreads * 4;
  return many ? run_rows<T, N, INTERLEAVED, 4>(a, places, slots, stream) : run_rows<T, N, INTERLEAVED, 1>(a, places, slots, stream);
}

// Whether all vectors of N channels lie whole in a tensor's parts, aligned to their size.
template <typename T, int N, bool INTERLEAVED>
bool vectors(const RotaryArgs& a) {
  bool ok = a.rotary % (INTERLEAVED ? N : 2 * N) == 0 && a.dim % N == 0;
  for (const RotaryTensor& t : a.t)
    if (t.heads)
      ok = ok && (reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.y)) % (N * sizeof(T)) == 0 &&
           (t.x_row | t.x_head | t.y_row | t.y_head) % N == 0;
  return ok;
}

template <typename T, bool INTERLEAVED>
hipError_t run(const RotaryArgs& a, int cus, hipStream_t stream) {
  constexpr int N = 16 / (int)sizeof(T);
  if (vectors<T, N, INTERLEAVED>(a)) return run_units<T, N, INTERLEAVED>(a, cus, stream);
  if (vectors<T, N / 2, INTERLEAVED>(a)) return run_units<T, N / 2, INTERLEAVED>(a, cus, stream);
  return run_units<T, 1, INTERLEAVED>(a, cus, stream);
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
