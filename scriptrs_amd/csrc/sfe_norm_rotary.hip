// Norms of queries and keys for each head, and their rotary positions, in one pass.
//
// A head's channels x become y = N(x) w, with N(x) = x / sqrt(mean x^2 + eps) (rms) or
// (x - mean) / sqrt(var + eps) (layer), and pairs of the first R channels of y turn by the
// position's angle (sfe_rotary.hip has the formula and its exactness).  Statistics
// are f32, the variance from the deviations; the result is rounded once, where a norm and a rotary
// pass behind it would round twice.
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
constexpr int kTable = 4096;  // (cosine, sine) of a workgroup's rows and pairs

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}

// Sum over groups of `lanes` lanes, a power of two; every lane has it, of the same order.
__device__ __forceinline__ float group_sum(float x, int lanes) {
  if (lanes > 1) x += dpp<0xb1>(x);   // the other of 2
  if (lanes > 2) x += dpp<0x4e>(x);   // the other two of 4
  if (lanes > 4) x += dpp<0x141>(x);  // mirrored within 8
  if (lanes > 8) x += dpp<0x140>(x);  // mirrored within 16
  if (lanes > 16) x += __shfl_xor(x, 16);
  if (lanes > 32) x += __shfl_xor(x, 32);
  return x;
}

// A workgroup takes `heads` consecutive heads of the rows' q and k heads, laid end to end, K a
// lane group.  N: channels of a vector; N = 1: a unit is a pair or a channel that does not turn, U of them a lane.
template <typename T, int N, bool INTERLEAVED, bool LAYER, int K, int U>
__global__ __launch_bounds__(kThreads) void sfe_norm_rotary_kernel(NormRotaryArgs a, int64_t first, int heads, int lanes,
                                                                   int slots) {
  constexpr bool kOne = INTERLEAVED && N > 1;  // both channels of a pair in one vector
  constexpr int kPairs = kOne ? N / 2 : N;     // of a unit
  typedef Vec<T, N> V;
  __shared__ float2 table[kTable];
  __shared__ float weights[2][kNormRotaryMaxDim];
  const int t = (int)threadIdx.x, pairs = a.rotary / 2, in_row = a.t[0].heads + a.t[1].heads;
  const int groups = kThreads / lanes, group = t / lanes, lane = t - group * lanes;
  // (workgroups count heads, rows of them: 64 bits)
  const int64_t head0 = first + (int64_t)blockIdx.x * heads, row0 = head0 / in_row;
  const int skip = (int)(head0 - row0 * in_row);
  const int64_t left = a.rows * in_row - head0;
  const int mine = left < heads ? (int)left : heads;

  V p[K][U], q[K][U];
  bool second[K];
  T* y[K];
  int local[K];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int h = group + k * groups;
    local[k] = -1;
    if (h >= mine) continue;
    const int r = (int)((unsigned)(skip + h) / (unsigned)in_row), head = skip + h - r * in_row;
    local[k] = r;
    second[k] = head >= a.t[0].heads;
    const RotaryTensor& tn = a.t[second[k]];
    const int of = second[k] ? head - a.t[0].heads : head;
    const T* x = reinterpret_cast<const T*>(tn.x) + (row0 + r) * tn.x_row + of * tn.x_head;
    y[k] = reinterpret_cast<T*>(tn.y) + (row0 + r) * tn.y_row + of * tn.y_head;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = lane + u * lanes;
      const bool turn = slot < pairs / kPairs;
      const int d0 = turn ? slot * (INTERLEAVED ? 2 * kPairs : kPairs) : a.rotary + N * (slot - pairs / kPairs);
      const int d1 = INTERLEAVED ? d0 + 1 : d0 + pairs;
      p[k][u] = q[k][u] = V{};
      if (slot < slots) {
        p[k][u] = *reinterpret_cast<const V*>(x + d0);
        if (!kOne && turn) q[k][u] = *reinterpret_cast<const V*>(x + d1);
      }
    }
  }
  // sines and cosines of the rows, and the weights, while the heads are on their way
  const int rows = (int)((unsigned)(skip + mine - 1) / (unsigned)in_row) + 1;
  for (int e = t; e < rows * pairs; e += kThreads) {
    const int r = (int)((unsigned)e / (unsigned)pairs), i = e - r * pairs;
    float c, s;
    turn_cos_sin((uint32_t)(((uint64_t)(int64_t)a.positions[row0 + r] * a.step[i]) >> 32), &c, &s);
    table[e] = make_float2(a.magnitude * c, a.magnitude * s);
  }
  for (int e = t; e < a.dim; e += kThreads) {
    weights[0][e] = a.weight[0] ? a.weight[0][e] : 1.0f;
    weights[1][e] = a.weight[1] ? a.weight[1][e] : 1.0f;
  }
  __syncthreads();
  const float over = 1.0f / (float)a.dim;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    // (a group's lanes agree; those of a wave may not, and sums take all that are there)
    float e[U][N], f[U][N], sum = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        e[u][i] = local[k] < 0 ? 0.0f : (float)p[k][u].v[i];
        f[u][i] = local[k] < 0 || kOne ? 0.0f : (float)q[k][u].v[i];
        sum += e[u][i] + f[u][i];
      }
    const float mean = LAYER ? group_sum(sum, lanes) * over : 0.0f;
    float square = 0.0f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = lane + u * lanes;
      const bool in = slot < slots, turn = slot < pairs / kPairs;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        if (LAYER) {  // (places that hold no channel stay zero)
          e[u][i] = in ? e[u][i] - mean : 0.0f;
          f[u][i] = in && turn && !kOne ? f[u][i] - mean : 0.0f;
        }
        square = __builtin_fmaf(e[u][i], e[u][i], square);
        if (!kOne) square = __builtin_fmaf(f[u][i], f[u][i], square);
      }
    }
    const float inv = 1.0f / sqrtf(group_sum(square, lanes) * over + a.eps);
    if (local[k] < 0) continue;
    const float* w = weights[second[k]];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int slot = lane + u * lanes;
      if (slot >= slots) continue;
      const bool turn = slot < pairs / kPairs;
      const int d0 = turn ? slot * (INTERLEAVED ? 2 * kPairs : kPairs) : a.rotary + N * (slot - pairs / kPairs);
      const int d1 = INTERLEAVED ? d0 + 1 : d0 + pairs;
      V r, s;
#pragma unroll
      for (int i = 0; i < N; ++i) e[u][i] *= inv * w[d0 + i];
      if (!turn) {
#pragma unroll
        for (int i = 0; i < N; ++i) r.v[i] = (T)e[u][i];
        *reinterpret_cast<V*>(y[k] + d0) = r;
        continue;
      }
      const float2* cs = table + local[k] * pairs + slot * kPairs;
#pragma unroll
      for (int i = 0; i < kPairs; ++i) {
        const float x0 = e[u][kOne ? (2 * i) % N : i];
        const float x1 = kOne ? e[u][(2 * i + 1) % N] : f[u][i] * (inv * w[d1 + i]);
        const T y0 = (T)__builtin_fmaf(x0, cs[i].x, -x1 * cs[i].y), y1 = (T)__builtin_fmaf(x1, cs[i].x, x0 * cs[i].y);
        r.v[kOne ? (2 * i) % N : i] = y0;
        if (kOne) r.v[(2 * i + 1) % N] = y1;
        else s.v[i] = y1;
      }
      *reinterpret_cast<V*>(y[k] + d0) = r;
      if (!kOne) *reinterpret_cast<V*>(y[k] + d1) = s;
    }
  }
}

template <typename T, int N, bool INTERLEAVED, bool LAYER, int K, int U>
hipError_t run_heads(const NormRotaryArgs& a, int lanes, int slots, hipStream_t stream) {
  const int in_row = a.t[0].heads + a.t[1].heads, pairs = a.rotary / 2;
  // as many heads as the lane groups take at K each, of rows that the table has room for
  const int heads = (int)std::min<int64_t>(K * (kThreads / lanes), ((int64_t)(kTable / pairs) - 1) * in_row);
  const int64_t total = a.rows * in_row, step = (int64_t)heads << 22;  // (launches of at most 2^22 workgroups)
  for (int64_t first = 0; first < total; first += step) {
    const int64_t n = std::min(step, total - first);
    sfe_norm_rotary_kernel<T, N, INTERLEAVED, LAYER, K, U><<<dim3((unsigned)((n + heads - 1) / heads)), dim3(kThreads), 0, stream>>>(
        a, first, heads, lanes, slots);
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
    return run_heads<T, N, INTERLEAVED, LAYER, 1, kNormRotaryMaxDim / 64>(a, lanes, slots, stream);
  } else {
    // One head a lane group while the machine is not full at 4.
    const int64_t heads = a.rows * (a.t[0].heads + a.t[1].heads);
    const bool many = heads * lanes >= (int64_t)cus * 8 * kThreads * 4;
    return many ? run_heads<T, N, INTERLEAVED, LAYER, 4, 1>(a, lanes, slots, stream)
                : run_heads<T, N, INTERLEAVED, LAYER, 1, 1>(a, lanes, slots, stream);
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
  const int pairs = INTERLEAVED && N > 1 ? N / 2 : N;
  return a.rotary / 2 / pairs + (a.dim - a.rotary) / N;
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
