// Norms of queries and keys for each head, and their rotary positions, in one pass.
//
// A head's channels x become y = N(x) w, with N(x) = x / sqrt(mean x^2 + eps) (rms) or
// (x - mean) / sqrt(var + eps) (layer), and pairs of the first R channels of y turn by the
// position's angle (sfe_rotary.hip has the formula and its exactness).  Statistics
// are f32, the variance from the deviations; the result is rounded once, where a norm and a rotary
// pass behind it would round twice.
//
// Bound by memory: each element is read and written once.  52,640 rows of 8 + 8 heads of 128 in bf16, 96 channels turned, layer
// norms: 431 MB in 106 us, 4.1 TB/s, where the turn alone (sfe_rotary.hip) runs at the copy's 4.9-5.1; vector instructions
// take 62% of the CUs' time.  Four rows a thread: 2 121, 8 117 us and more, 1 172 (what depends on the place is computed once, and
// there is enough in flight).  64 rows of 16 + 4 heads: 4.4 us, the launch and one trip.
//
// A head is a group of lanes, a power of two; a lane holds the channels that turn together (half: two vectors
// R / 2 apart, interleaved: one vector of whole pairs), so that sums are exchanges within the
// group and a turn is within a lane.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "sfe_decode.hpp"
#include "sfe_turn.hpp"

namespace sfe {
namespace {

constexpr int kThreads = 256;
constexpr int kTable = 4096;  // (cosine, sine) of a workgroup's rows and pairs at most

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// Sums of K values over groups of `lanes` lanes, a power of two; every lane has them, of the same order.
template <int K>
__device__ __forceinline__ void group_sums(float (&x)[K], int lanes) {
  if (lanes > 1)
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += dpp<0xb1>(x[k]);  // the other of 2
  if (lanes > 2)
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += dpp<0x4e>(x[k]);  // the other two of 4
  if (lanes > 4)
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += dpp<0x141>(x[k]);  // mirrored within 8
  if (lanes > 8)
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += dpp<0x140>(x[k]);  // mirrored within 16
  if (lanes > 16)
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += __shfl_xor(x[k], 16);
  if (lanes > 32)
#pragma unroll
    for (int k = 0; k < K; ++k) x[k] += __shfl_xor(x[k], 32);
}

// 1 / sqrt(x), to a step of f32 (x tiny: of 2^64 x).
__device__ __forceinline__ float over_root(float x) {
  const bool tiny = x < 0x1p-96f;
  return __builtin_amdgcn_rsqf(tiny ? x * 0x1p64f : x) * (tiny ? 0x1p32f : 1.0f);
}

// A workgroup takes K times `per` rows.  Places of a row: `lanes` for each of its heads, q's then k's; a thread
// keeps its place in K rows (so that what depends on the place is computed once), all K loads
// issued before the first store and before the rows' sines and cosines go into LDS.  Rows of more than 256 places
// go in `chunks` workgroups.  N: channels of a vector; a lane's unit is one or two vectors (two of those that do not
// turn as well), N = 1: one or two channels, U units a lane.
template <typename T, int N, bool INTERLEAVED, bool LAYER, int K, int U>
__global__ __launch_bounds__(kThreads) void sfe_norm_rotary_kernel(NormRotaryArgs a, int64_t first, int places, int lanes,
                                                                   int slots, int chunks, int per) {
  constexpr bool kOne = INTERLEAVED && N > 1;  // both channels of a pair in one vector
  constexpr int kPairs = kOne ? N / 2 : N;     // of a unit
  typedef Vec<T, N> V;
  extern __shared__ float2 table[];
  const int t = (int)threadIdx.x, pairs = a.rotary / 2;
  const uint32_t group = blockIdx.x / (uint32_t)chunks, chunk = blockIdx.x - group * (uint32_t)chunks;
  const int64_t row0 = first + (int64_t)group * K * per;
  const int rows = (int)(a.rows - row0 < K * per ? a.rows - row0 : K * per);
  const int in = per > 1 ? (int)((unsigned)t / (unsigned)places) : 0;  // row within a pass
  const int place = per > 1 ? t - in * places : (int)chunk * (int)blockDim.x + t;
  const bool mine = place < places && in < per;  // (all lanes of a head, or none)
  const int head = (int)((unsigned)place / (unsigned)lanes), lane = place - head * lanes;
  const bool second = head >= a.t[0].heads;
  const int of = second ? head - a.t[0].heads : head;
  const int64_t x_row = second ? a.t[1].x_row : a.t[0].x_row, y_row = second ? a.t[1].y_row : a.t[0].y_row;
  const T* x = reinterpret_cast<const T*>(second ? a.t[1].x : a.t[0].x) + (row0 + in) * x_row + of * (second ? a.t[1].x_head : a.t[0].x_head);
  T* y = reinterpret_cast<T*>(second ? a.t[1].y : a.t[0].y) + (row0 + in) * y_row + of * (second ? a.t[1].y_head : a.t[0].y_head);
  const float* weight = second ? a.weight[1] : a.weight[0];

  V p[K][U], q[K][U];
  float w0[U][N], w1[U][N];
  int d0[U], d1[U];
  bool turn[U], both[U];  // (both: the second vector is there too)
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int slot = lane + u * lanes, rest = slot - pairs / kPairs;
    turn[u] = rest < 0;
    d0[u] = turn[u] ? slot * (INTERLEAVED ? 2 * kPairs : kPairs) : a.rotary + (kOne ? N : 2 * N) * rest;
    d1[u] = turn[u] ? (INTERLEAVED ? d0[u] + 1 : d0[u] + pairs) : d0[u] + N;
    if (slot >= slots || !mine) d0[u] = -1;  // (no channels)
    both[u] = !kOne && d0[u] >= 0 && d1[u] < a.dim;
  }
  // what the table and the products need is asked for first, so that waiting for it is not waiting for the heads
  const int my_row = (int)((unsigned)t / (unsigned)pairs);
  const int32_t position = t < rows * pairs ? a.positions[row0 + my_row] : 0;
#pragma unroll
  for (int u = 0; u < U; ++u)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      w0[u][i] = weight && d0[u] >= 0 ? weight[d0[u] + i] : 1.0f;
      w1[u][i] = weight && both[u] ? weight[d1[u] + i] : 1.0f;
    }
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int u = 0; u < U; ++u) {
      p[k][u] = q[k][u] = V{};
      if (d0[u] >= 0 && in + k * per < rows) {
        p[k][u] = *reinterpret_cast<const V*>(x + k * (int64_t)per * x_row + d0[u]);
        if (!kOne && both[u]) q[k][u] = *reinterpret_cast<const V*>(x + k * (int64_t)per * x_row + d1[u]);
      }
    }
  // sines and cosines of the rows, while the heads are on their way
  auto turned = [&](int e, int r, int32_t at) {
    float c, s;
    turn_cos_sin((uint32_t)(((uint64_t)(int64_t)at * a.step[e - r * pairs]) >> 32), &c, &s);
    table[e] = make_float2(a.magnitude * c, a.magnitude * s);
  };
  if (t < rows * pairs) turned(t, my_row, position);
  for (int e = t + (int)blockDim.x; e < rows * pairs; e += (int)blockDim.x) {
    const int r = (int)((unsigned)e / (unsigned)pairs);
    turned(e, r, a.positions[row0 + r]);
  }
  // (the workgroup's LDS is waited for, and not its loads)
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  if (!mine) return;
  const float over = 1.0f / (float)a.dim;
  float e[K][U][N], f[K][U][N], sum[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sum[k] = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        e[k][u][i] = (float)p[k][u].v[i];
        f[k][u][i] = kOne ? 0.0f : (float)q[k][u].v[i];
        if (LAYER) sum[k] += kOne ? e[k][u][i] : e[k][u][i] + f[k][u][i];
      }
  }
  if (LAYER) {
    group_sums<K>(sum, lanes);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
      for (int u = 0; u < U; ++u) {  // (places that hold no channel stay zero)
        const float mean = sum[k] * over, me = d0[u] >= 0 ? mean : 0.0f, mf = both[u] ? mean : 0.0f;
#pragma unroll
        for (int i = 0; i < N; ++i) {
          e[k][u][i] -= me;
          if (!kOne) f[k][u][i] -= mf;
        }
      }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) {
    sum[k] = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        sum[k] = __builtin_fmaf(e[k][u][i], e[k][u][i], sum[k]);
        if (!kOne) sum[k] = __builtin_fmaf(f[k][u][i], f[k][u][i], sum[k]);
      }
  }
  group_sums<K>(sum, lanes);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (in + k * per >= rows) continue;
    const float inv = over_root(sum[k] * over + a.eps);
    T* yk = y + k * (int64_t)per * y_row;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (d0[u] < 0) continue;
      V r, s;
#pragma unroll
      for (int i = 0; i < N; ++i) e[k][u][i] *= inv * w0[u][i];
      if (!turn[u]) {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = (T)e[k][u][i], s.v[i] = (T)(f[k][u][i] * (inv * w1[u][i]));
        *reinterpret_cast<V*>(yk + d0[u]) = r;
        if (both[u]) *reinterpret_cast<V*>(yk + d1[u]) = s;
        continue;
      }
      const float2* cs = table + (in + k * per) * pairs + (lane + u * lanes) * kPairs;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float x0 = e[k][u][kOne ? (2 * i) % N : i];
        const float x1 = kOne ? e[k][u][(2 * i + 1) % N] : f[k][u][i] * (inv * w1[u][i]);
        const T y0 = (T)__builtin_fmaf(x0, cs[i].x, -x1 * cs[i].y), y1 = (T)__builtin_fmaf(x1, cs[i].x, x0 * cs[i].y);
        r.v[kOne ? (2 * i) % N : i] = y0;
        if (kOne) r.v[(2 * i + 1) % N] = y1;
        else s.v[i] = y1;
      }
      *reinterpret_cast<V*>(yk + d0[u]) = r;
      if (!kOne) *reinterpret_cast<V*>(yk + d1[u]) = s;
    }
  }
}

template <typename T, int N, bool INTERLEAVED, bool LAYER, int K, int U>
hipError_t run_rows(const NormRotaryArgs& a, int lanes, int slots, hipStream_t stream) {
  const int places = (a.t[0].heads + a.t[1].heads) * lanes, pairs = a.rotary / 2;
  const int chunks = (places + kThreads - 1) / kThreads;
  const int per = chunks > 1 ? 1 : std::max(1, std::min(kThreads / places, kTable / (K * pairs)));
  // whole waves, as few as hold the places (a head's lanes never cross a chunk: both are powers of two of a wave)
  const int threads = ((chunks > 1 ? (places + chunks - 1) / chunks : places * per) + 63) / 64 * 64;
  const size_t lds = (size_t)K * per * pairs * sizeof(float2);
  // (launches of at most 2^22 workgroups)
  const int64_t step = std::max<int64_t>(1, ((int64_t)1 << 22) / chunks) * K * per;
  for (int64_t first = 0; first < a.rows; first += step) {
    const int64_t rows = std::min(step, a.rows - first);
    const unsigned blocks = (unsigned)((rows + K * per - 1) / (K * per) * chunks);
    sfe_norm_rotary_kernel<T, N, INTERLEAVED, LAYER, K, U><<<dim3(blocks), dim3(threads), lds, stream>>>(a, first, places, lanes, slots, chunks, per);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <typename T, int N, bool INTERLEAVED, bool LAYER>
hipError_t run_units(const NormRotaryArgs& a, int slots, int cus, hipStream_t stream) {
  int lanes = 1;
  while (lanes < slots && lanes < 64) lanes *= 2;
  if constexpr (N == 1) {
    return run_rows<T, N, INTERLEAVED, LAYER, 1, kNormRotaryMaxDim / 64>(a, lanes, slots, stream);
  } else {
    // One row a thread while the machine is not full at 4.
    const int64_t places = a.rows * (a.t[0].heads + a.t[1].heads) * lanes;
    const bool many = places >= (int64_t)cus * 8 * kThreads * 4;
    return many ? run_rows<T, N, INTERLEAVED, LAYER, 4, 1>(a, lanes, slots, stream)
                : run_rows<T, N, INTERLEAVED, LAYER, 1, 1>(a, lanes, slots, stream);
  }
}

// Whether all vectors of N channels lie whole in a tensor's parts, aligned to their size.
template <typename T, int N, bool INTERLEAVED>
bool vectors(const NormRotaryArgs& a) {
  bool ok = a.rotary % (INTERLEAVED ? N : 2 * N) == 0 && a.dim % N == 0;
  for (const RotaryTensor& t : a.t)
    if (t.heads)
      ok = ok && (reinterpret_cast<uintptr_t>(t.x) | reinterpret_cast<uintptr_t>(t.y)) % (N * sizeof(T)) == 0 &&
           (t.x_row | t.x_head | t.y_row | t.y_head) % N == 0;
  return ok;
}

template <typename T, int N, bool INTERLEAVED>
int slots_of(const NormRotaryArgs& a) {
  const bool one = INTERLEAVED && N > 1;
  const int pairs = one ? N / 2 : N, copied = one ? N : 2 * N;
  return a.rotary / 2 / pairs + (a.dim - a.rotary + copied - 1) / copied;
}

template <typename T, bool INTERLEAVED, bool LAYER>
hipError_t run(const NormRotaryArgs& a, int cus, hipStream_t stream) {
  constexpr int N = 16 / (int)sizeof(T);
  if (vectors<T, N, INTERLEAVED>(a)) return run_units<T, N, INTERLEAVED, LAYER>(a, slots_of<T, N, INTERLEAVED>(a), cus, stream);
  const int slots = slots_of<T, N / 2, INTERLEAVED>(a);
  if (vectors<T, N / 2, INTERLEAVED>(a) && slots <= 64) return run_units<T, N / 2, INTERLEAVED, LAYER>(a, slots, cus, stream);
  return run_units<T, 1, INTERLEAVED, LAYER>(a, slots_of<T, 1, INTERLEAVED>(a), cus, stream);
}

template <typename T>
hipError_t run_kind(const NormRotaryArgs& a, bool interleaved, bool layer, int cus, hipStream_t stream) {
  if (interleaved) return layer ? run<T, true, true>(a, cus, stream) : run<T, true, false>(a, cus, stream);
  return layer ? run<T, false, true>(a, cus, stream) : run<T, false, false>(a, cus, stream);
}

}  // namespace

hipError_t launch_norm_rotary(const NormRotaryArgs& a, int type, bool interleaved, bool layer, int cus, hipStream_t stream) {
  if (type == kOpF32) return run_kind<float>(a, interleaved, layer, cus, stream);
  if (type == kOpBf16) return run_kind<__bf16>(a, interleaved, layer, cus, stream);
  return run_kind<_Float16>(a, interleaved, layer, cus, stream);
}

}  // namespace sfe
