// Steering of logits before a choice: penalties for tokens said before, a bias, and a grammar's masks.
//
// With c the times that token t stands in its row's history:
//   z = logit; c > 0: z = z / repetition (z > 0) or z * repetition, then z -= presence + frequency c;
//   z += bias[t]; a token that the row's mask lacks: z = -inf.
// In f32, rounded once.
//
// Bound by memory and, with histories, by the vector instructions of their penalties (82% of the CUs' time): 512 rows of 128,000 in
// bf16 with histories of up to 1,500, biases and a grammar, 266 MB in 60 us (4.4 TB/s), 183 before all
// loads were in flight together; 64 rows in f16 with histories of up to 8,192 13 us, the history's scan by each span the rest.
//
// One pass over the logits: a workgroup takes a span of one row's tokens, has all of its
// logits in flight, counts the history's tokens of its span in LDS meanwhile (whole numbers:
// their order does not matter), and writes.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sfe_decode.hpp"
#include "sfe_internal.hpp"
#include "sfe_turn.hpp"

namespace sfe {
namespace {

constexpr int kThreads = 256;

// Waits for the workgroup's LDS accesses, not for its loads.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// N: elements of a vector (16 bytes, or one); V: vectors of a thread.  Vectors begin at multiples of 16 bytes:
// the first of a row may begin up to N - 1 elements before it.
// H: bytes of a count, 0 without a history.
template <typename T, int N, int V, int H, bool BIAS, bool MASK>
__global__ __launch_bounds__(kThreads) void sfe_logits_kernel(LogitsArgs a, int64_t first_row, uint32_t first_span, uint32_t spans) {
  typedef Vec<T, N> Vector;
  constexpr int kSpan = kThreads * N * V;
  __shared__ __align__(16) uint32_t counts[H ? kSpan * H / 4 : 4];
  const uint32_t block = first_span + blockIdx.x, of_first = block / spans;
  const int64_t r = first_row + of_first;
  const int t = (int)threadIdx.x;
  const T* in = reinterpret_cast<const T*>(a.in) + r * a.in_row;
  T* out = reinterpret_cast<T*>(a.out) + r * a.out_row;
  const int before = N > 1 ? (int)((uintptr_t)in / sizeof(T) % N) : 0;
  const LogitsSpan span = logits_span((int)(block - of_first * spans), kSpan, before, a.vocab);
  const int span0 = span.first;

  // ---- all loads, those of the history first
  int n = 0;
  float rep = 1.0f, over = 1.0f, presence = 0.0f, frequency = 0.0f;
  const int32_t* said = a.history + (H ? r * a.history_row : 0);
  constexpr int kAhead = 4;  // tokens of a thread in flight
  int32_t token[kAhead];
  auto tokens = [&](int e) {
#pragma unroll
    for (int i = 0; i < kAhead; ++i) token[i] = e + i * kThreads < a.history_most ? said[e + i * kThreads] : -1;
  };
  if (H) {
    tokens(t);
    n = a.lengths ? min(a.lengths[r], a.history_most) : a.history_most;
    rep = a.repetitions ? a.repetitions[r] : a.repetition;
    presence = a.presences ? a.presences[r] : a.presence;
    frequency = a.frequencies ? a.frequencies[r] : a.frequency;
  }
  Vector x[V];
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int at = span0 + (v * kThreads + t) * N;
    if (N > 1 && at >= 0 && at + N <= a.vocab) {
      x[v] = *reinterpret_cast<const Vector*>(in + at);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[v].v[i] = at + i >= 0 && at + i < a.vocab ? in[at + i] : (T)0.0f;
    }
  }
  const uint32_t* words = nullptr;
  if (MASK) {
    const int64_t state = a.states ? a.states[r] : r;
    if (state >= 0 && state < a.n_allowed) words = a.allowed + state * a.allowed_row;
  }
  float bias[V][BIAS ? N : 1];
  uint32_t low_word[V], high_word[V];  // of the mask: that of a vector's first token and the next
  if (BIAS) {
    const float* from = a.bias + r * a.bias_row;
    const bool whole = N > 1 && ((uintptr_t)from / 4 - before) % 4 == 0;  // vectors of 16 bytes
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = span0 + (v * kThreads + t) * N;
      if (whole && at >= 0 && at + N <= a.vocab) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          const float4 b = *reinterpret_cast<const float4*>(from + at + i);
          bias[v][i % N] = b.x, bias[v][(i + 1) % N] = b.y, bias[v][(i + 2) % N] = b.z, bias[v][(i + 3) % N] = b.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) bias[v][i] = at + i >= 0 && at + i < a.vocab ? from[at + i] : 0.0f;
      }
    }
  }
  if (MASK)
#pragma unroll
    for (int v = 0; v < V; ++v) {
      const int at = span0 + (v * kThreads + t) * N;
      const int w = at >> 5;
      low_word[v] = high_word[v] = ~0u;
      if (words && at < a.vocab) {
        low_word[v] = w >= 0 ? words[w] : 0;
        if (before && 32 * (w + 1) < a.vocab) high_word[v] = words[w + 1];  // (else a vector's bits are in one)
      }
    }
  // ---- the history's tokens of the span, counted in LDS
  if (H) {
    for (int e = 4 * t; e < kSpan * H / 4; e += 4 * kThreads) *reinterpret_cast<uint4*>(counts + e) = make_uint4(0, 0, 0, 0);
    over = 1.0f / rep;
    lds_barrier();
    for (int e = t; e < n;) {
      int32_t now[kAhead];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) now[i] = e + i * kThreads < n ? token[i] : -1;
      e += kAhead * kThreads;
      tokens(e);
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        if (!span.has(now[i])) continue;
        const int at = span.place(now[i]);
        if (H == 2) atomicAdd(counts + at / 2, at & 1 ? 0x10000u : 1u);
        else atomicAdd(counts + at, 1u);
      }
    }
    lds_barrier();
  }
#pragma unroll
  for (int v = 0; v < V; ++v) {
    const int place = (v * kThreads + t) * N, at = span0 + place;
    if (at >= a.vocab || at + N <= 0) continue;
    float z[N];
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = (float)x[v].v[i];
    if (H) {
      constexpr int kWords = N * H < 4 ? 1 : N * H / 4;
      uint32_t c[kWords], any = 0;
#pragma unroll
      for (int i = 0; i < kWords; ++i) c[i] = counts[place * H / 4 + i], any |= c[i];
      if (N == 1 && H == 2) any = c[0] = place & 1 ? c[0] >> 16 : c[0] & 0xffffu;
      if (any) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const uint32_t count = H == 2 ? (i % 2 ? c[i / 2] >> 16 : c[i / 2] & 0xffffu) : c[i];
          float y;
          if constexpr (sizeof(T) == 2) {
            // (off by 1.5 steps of f32 before the one rounding to 16 bits)
            y = z[i] * (z[i] > 0.0f ? over : rep);
          } else {
            // the quotient by its reciprocal, corrected by the remainder; where that is past the largest number,
            // by a division (the quotient may be it yet, and an infinity has no remainder)
            y = z[i] * over;
            if (__builtin_isfinite(y)) y = __builtin_fmaf(__builtin_fmaf(-y, rep, z[i]), over, y);
            else y = z[i] / rep;
            y = z[i] > 0.0f ? y : z[i] * rep;
          }
          y -= presence + frequency * (float)count;
          z[i] = count ? y : z[i];
        }
      }
    }
    Vector y;
    const uint32_t bits = MASK ? __builtin_amdgcn_alignbit(high_word[v], low_word[v], at & 31) : 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if (BIAS) z[i] += bias[v][i];
      if (MASK) {  // (as whole numbers: two operations)
        const uint32_t m = (uint32_t)((int32_t)(bits << (31 - i)) >> 31);
        z[i] = __uint_as_float((__float_as_uint(z[i]) & m) | (0xff800000u & ~m));
      }
      y.v[i] = (T)z[i];
    }
    if (N > 1 && at >= 0 && at + N <= a.vocab) {
      *reinterpret_cast<Vector*>(out + at) = y;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at + i >= 0 && at + i < a.vocab) out[at + i] = y.v[i];
    }
  }
}

template <typename T, int N, int V, int H, bool BIAS, bool MASK>
hipError_t run(const LogitsArgs& a, hipStream_t stream) {
  constexpr int kSpan = kThreads * N * V;
  const int spans = logits_spans(a.vocab, N, kSpan);
  return for_launches((int64_t)a.rows * spans, kThreads, [&](int64_t first, unsigned blocks) {
    sfe_logits_kernel<T, N, V, H, BIAS, MASK><<<dim3(blocks), dim3(kThreads), 0, stream>>>(a, first / spans, (uint32_t)(first % spans), (uint32_t)spans);
    return hipGetLastError();
  });
}

template <typename T, int N, int V, int H>
hipError_t run_what(const LogitsArgs& a, hipStream_t stream) {
  if (a.bias) return a.allowed ? run<T, N, V, H, true, true>(a, stream) : run<T, N, V, H, true, false>(a, stream);
  return a.allowed ? run<T, N, V, H, false, true>(a, stream) : run<T, N, V, H, false, false>(a, stream);
}

template <typename T, int N, int V>
hipError_t run_history(const LogitsArgs& a, hipStream_t stream) {
  if (!a.history) return run_what<T, N, V, 0>(a, stream);
  // counts of 16 bits where they hold a whole history
  return a.history_most < 65536 ? run_what<T, N, V, 2>(a, stream) : run_what<T, N, V, 4>(a, stream);
}

template <typename T>
hipError_t run_type(const LogitsArgs& a, hipStream_t stream) {
  constexpr int N = 16 / (int)sizeof(T);
  // vectors where a row's input and output lie alike
  const bool alike = (uintptr_t)a.in % 16 == (uintptr_t)a.out % 16 && (a.in_row - a.out_row) % N == 0;
  // Spans of 4,096 tokens, 8,192 where a long history is read by every one of them and no biases take
  // registers.  512 rows of 128,000 in bf16 with histories of up to 1,500: 4,096 58 us with a grammar, 62 with biases too; 8,192
  // 59 and 69; 2,048 62 and 71.  64 rows with histories of up to 8,192: 14.0 and 12.7.
  constexpr int V = 4096 / (kThreads * N);
  if (!alike) return run_history<T, 1, 4>(a, stream);
  if (a.history && a.history_most > 4096 && !a.bias) return run_history<T, N, 2 * V>(a, stream);
  return run_history<T, N, V>(a, stream);
}

}  // namespace

hipError_t launch_logits(const LogitsArgs& a, int type, hipStream_t stream) {
  if (type == kOpF32) return run_type<float>(a, stream);
  if (type == kOpBf16) return run_type<__bf16>(a, stream);
  return run_type<_Float16>(a, stream);
}

}  // namespace sfe
