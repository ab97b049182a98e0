// A step of beam search.
//
// total(w, t) = score_w + (logit_wt - log sum_t exp(logit_wt)); a finished beam
// has the one candidate (score_w, end token).  A stream's next beams are the best
// of its beams * vocabulary candidates, ties to the lowest (beam, token); totals of
// -inf or NaN are no candidates, and places without one hold score -inf, token
// -1 and their own beam as parent.
//
// Two launches.  Within a row, candidates order as its logits do, so the first reads
// each logit once, and a workgroup leaves its chunk's maximum, sum of exponentials and
// `beams` best logits; the second has beams * chunks * beams candidates a
// stream.  Bound by memory (the logits) where the vocabulary is large, by latency
// where it is small.  Sums are f32 and every order of addition is fixed.
#include <hip/hip_runtime.h>

#include <cstdint>

#include "sfe_internal.hpp"
#include "sfe_ops.hpp"

namespace sfe {
namespace {

typedef unsigned U4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kEach = 32;                  // logits of a thread
constexpr int kChunk = kThreads * kEach;   // logits of a workgroup
constexpr int kList = 256;                 // candidates held at once

// Scratch: [row][chunk] of (maximum, sum), then of beams (logit, token).
struct Part {
  float top, sum;
};
struct Cand {
  float x;
  int32_t t;
};

__device__ __forceinline__ bool before(float x, int64_t i, float y, int64_t j) { return x > y || (x == y && i < j); }

__device__ __forceinline__ float wave_max(float x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d));
  return x;
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

// The best (value, index) over the workgroup, every thread getting it.
__device__ __forceinline__ void block_best(float* x, int64_t* i, float* lx, int64_t* li) {
#pragma unroll
  for (int d = 32; d > 0; d >>= 1) {
    const float y = __shfl_xor(*x, d);
    const int64_t j = __shfl_xor(*i, d);
    if (before(y, j, *x, *i)) {
      *x = y;
      *i = j;
    }
  }
  __syncthreads();
  if ((threadIdx.x & 63) == 0) {
    lx[threadIdx.x >> 6] = *x;
    li[threadIdx.x >> 6] = *i;
  }
  __syncthreads();
  for (int w = 0; w < kWaves; ++w)
    if (before(lx[w], li[w], *x, *i)) {
      *x = lx[w];
      *i = li[w];
    }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void sfe_beam_rows_kernel(BeamArgs a, int chunks) {
  constexpr int N = 16 / (int)sizeof(T), NV = kEach / N;
  struct alignas(16) V {
    T v[N];
  };
  __shared__ float lx[kWaves];
  __shared__ int64_t li[kWaves];
  __shared__ int count;
  __shared__ float cx[kList];
  __shared__ int ct[kList];
  const int row = (int)(blockIdx.x / (unsigned)chunks), chunk = (int)(blockIdx.x % (unsigned)chunks);
  const int t = (int)threadIdx.x;
  Part* part = reinterpret_cast<Part*>(a.scratch);
  Cand* cand = reinterpret_cast<Cand*>(part + (int64_t)a.streams * a.beams * chunks);
  const int64_t at = (int64_t)row * chunks + chunk;
  if (a.finished && a.finished[row]) return;  // (its logits are not looked at)
  const T* p = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.row;
  // vectors on 16-byte boundaries: the row starts `lead` elements into its first
  const int lead = (int)(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
  float x[kEach];
  const int first = chunk * kChunk - lead;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = first + (j * kThreads + t) * N;
    if (e >= 0 && e + N <= a.vocab) {
      const V v = *reinterpret_cast<const V*>(p + e);
#pragma unroll
      for (int i = 0; i < N; ++i) x[j * N + i] = (float)v.v[i];
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) x[j * N + i] = e + i >= 0 && e + i < a.vocab ? (float)p[e + i] : -INFINITY;
    }
  }
  auto token = [&](int k) { return first + (k / N * kThreads + t) * N + k % N; };
  float tm = -INFINITY;  // (fmaxf passes NaN over)
#pragma unroll
  for (int k = 0; k < kEach; ++k) tm = fmaxf(tm, x[k]);
  // A lower bound of the chunk's beams-th best logit: the beams-th largest of a
  // wave's thread maxima, the best wave's.
  float wm = tm, bound = -INFINITY, top = 0.0f;
  for (int r = 0; r < a.beams; ++r) {
    bound = wave_max(wm);
    if (r == 0) top = bound;
    const uint64_t same = __ballot(wm == bound);
    if ((t & 63) == __builtin_ctzll(same ? same : 1)) wm = -INFINITY;
  }
  if ((t & 63) == 0) {
    lx[t >> 6] = top;
    cx[t >> 6] = bound;
  }
  if (t == 0) count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    top = fmaxf(top, lx[w]);
    bound = fmaxf(bound, cx[w]);
  }
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < kEach; ++k) sum += top == -INFINITY ? 0.0f : __expf(x[k] - top);
  sum = wave_sum(sum);
  __syncthreads();
  if ((t & 63) == 0) lx[t >> 6] = sum;
  // the candidates: every logit at or above the bound
#pragma unroll
  for (int k = 0; k < kEach; ++k)
    if (x[k] >= bound && x[k] > -INFINITY) {
      const int c = atomicAdd(&count, 1);
      if (c < kList) {
        cx[c] = x[k];
        ct[c] = token(k);
      }
    }
  __syncthreads();
  const int n = count;
  if (t == 0) {
    float s = 0.0f;
    for (int w = 0; w < kWaves; ++w) s += lx[w];
    part[at] = Part{top, s};
  }
  Cand* out = cand + at * a.beams;
  if (n <= kList) {
    // ranks: the list's order does not matter
    if (t < n) {
      int rank = 0;
      for (int c = 0; c < n; ++c) rank += before(cx[c], ct[c], cx[t], ct[t]);
      if (rank < a.beams) out[rank] = Cand{cx[t], ct[t]};
    }
    for (int c = n + t; c < a.beams; c += kThreads) out[c] = Cand{-INFINITY, -1};
    return;
  }
  // many equal logits: the best after the last one taken, beams times
  float lastx = INFINITY;
  int64_t lasti = -1;
  for (int r = 0; r < a.beams; ++r) {
    float bx = -INFINITY;
    int64_t bi = INT64_MAX;
#pragma unroll
    for (int k = 0; k < kEach; ++k)
      if (before(lastx, lasti, x[k], token(k)) && before(x[k], token(k), bx, bi)) {
        bx = x[k];
        bi = token(k);
      }
    block_best(&bx, &bi, lx, li);
    if (t == 0) out[r] = bi == INT64_MAX ? Cand{-INFINITY, -1} : Cand{bx, (int32_t)bi};
    lastx = bx;
    lasti = bi;
  }
}

__global__ __launch_bounds__(kThreads) void sfe_beam_streams_kernel(BeamArgs a, int chunks) {
  __shared__ float lx[kWaves];
  __shared__ int64_t li[kWaves];
  __shared__ float logz[kMaxBeams];
  const int b = (int)blockIdx.x, t = (int)threadIdx.x, W = a.beams;
  const Part* part = reinterpret_cast<const Part*>(a.scratch) + (int64_t)b * W * chunks;
  const Cand* cand = reinterpret_cast<const Cand*>(reinterpret_cast<const Part*>(a.scratch) +
                                                   (int64_t)a.streams * W * chunks) + (int64_t)b * W * chunks * W;
  for (int w = t >> 6; w < W; w += kWaves) {
    if (a.finished && a.finished[(int64_t)b * W + w]) continue;
    float top = -INFINITY, sum = 0.0f;
    for (int c = t & 63; c < chunks; c += 64) top = fmaxf(top, part[w * chunks + c].top);
    top = wave_max(top);
    for (int c = t & 63; c < chunks; c += 64) {
      const Part p = part[w * chunks + c];
      if (p.top > -INFINITY) sum += p.sum * __expf(p.top - top);
    }
    sum = wave_sum(sum);
    if ((t & 63) == 0) logz[w] = top + logf(sum);
  }
  __syncthreads();
  const int n = W * chunks * W;
  auto total = [&](int e, int64_t* index) -> float {
    const int w = e / (chunks * W);
    const float score = a.scores[(int64_t)b * W + w];
    if (a.finished && a.finished[(int64_t)b * W + w]) {
      *index = (int64_t)w * a.vocab + a.end;
      return e == w * chunks * W ? score : -INFINITY;
    }
    const Cand c = cand[e];
    *index = (int64_t)w * a.vocab + c.t;
    return score + (c.x - logz[w]);
  };
  float lastx = INFINITY;
  int64_t lasti = -1;
  for (int r = 0; r < W; ++r) {
    float bx = -INFINITY;
    int64_t bi = INT64_MAX;
    for (int e = t; e < n; e += kThreads) {
      int64_t i;
      const float x = total(e, &i);
      if (x > -INFINITY && before(lastx, lasti, x, i) && before(x, i, bx, bi)) {
        bx = x;
        bi = i;
      }
    }
    block_best(&bx, &bi, lx, li);
    if (t == 0) {
      const bool found = bi != INT64_MAX;
      const int parent = found ? (int)(bi / a.vocab) : r, token = found ? (int)(bi % a.vocab) : -1;
      const int64_t o = (int64_t)b * W + r;
      a.out_scores[o] = found ? bx : -INFINITY;
      a.parents[o] = parent;
      a.tokens[o] = token;
      if (a.out_finished)
        a.out_finished[o] = (a.finished && a.finished[(int64_t)b * W + parent]) || token == a.end;
    }
    lastx = bx;
    lasti = bi;
  }
}

// ---- states ------------------------------------------------------------------------------

// A thread moves one column (sizeof(V) bytes) of all of a stream's beams: every
// beam is read before any is written, so a state may be reordered in place.
template <typename V, int BEAMS>
__global__ __launch_bounds__(kThreads) void sfe_beam_reorder_kernel(ReorderArgs a, int64_t unit0) {
  int64_t u = unit0 + (int64_t)blockIdx.x * kThreads + threadIdx.x;
  int k = 0;
  int64_t cols = 0;
  for (; k < a.n; ++k) {
    cols = a.s[k].inner / (int64_t)sizeof(V);
    const int64_t units = a.s[k].outer * a.streams * cols;
    if (u < units) break;
    u -= units;
  }
  if (k == a.n) return;
  const BeamState& s = a.s[k];
  const int64_t col = u % cols, os = u / cols;
  const int stream = (int)(os % a.streams);
  const int64_t base = os * a.beams * s.inner + col * (int64_t)sizeof(V);
  V v[BEAMS];
#pragma unroll
  for (int w = 0; w < BEAMS; ++w)
    if (w < a.beams) {
      int p = a.parents[(int64_t)stream * a.beams + w];
      if (p < 0 || p >= a.beams) p = w;  // (no such beam: stays)
      v[w] = *reinterpret_cast<const V*>(s.in + base + p * s.inner);
    }
#pragma unroll
  for (int w = 0; w < BEAMS; ++w)
    if (w < a.beams) *reinterpret_cast<V*>(s.out + base + w * s.inner) = v[w];
}

template <typename V, int BEAMS>
hipError_t reorder(const ReorderArgs& a, hipStream_t stream) {
  int64_t units = 0;
  for (int k = 0; k < a.n; ++k) units += a.s[k].outer * a.streams * (a.s[k].inner / (int64_t)sizeof(V));
  return for_launches((units + kThreads - 1) / kThreads, kThreads, [&](int64_t first, unsigned blocks) {
    sfe_beam_reorder_kernel<V, BEAMS><<<dim3(blocks), dim3(kThreads), 0, stream>>>(a, first * kThreads);
    return hipGetLastError();
  });
}
template <typename V>
hipError_t reorder_beams(const ReorderArgs& a, hipStream_t stream) {
  if (a.beams <= 4) return reorder<V, 4>(a, stream);
  if (a.beams <= 8) return reorder<V, 8>(a, stream);
  return reorder<V, 32>(a, stream);
}

int chunks_of(int vocab) { return (vocab + 15 + kChunk - 1) / kChunk; }  // (+ a row's lead)

}  // namespace

size_t beam_scratch_bytes(int streams, int beams, int vocab) {
  const int64_t parts = (int64_t)streams * beams * chunks_of(vocab);
  return (size_t)(parts * (int64_t)sizeof(Part) + parts * beams * (int64_t)sizeof(Cand));
}

hipError_t launch_beam_select(const BeamArgs& a, int type, hipStream_t stream) {
  const int chunks = chunks_of(a.vocab);
  const dim3 grid((unsigned)((int64_t)a.streams * a.beams * chunks));
  if (type == kOpF32)
    sfe_beam_rows_kernel<float><<<grid, dim3(kThreads), 0, stream>>>(a, chunks);
  else if (type == kOpBf16)
    sfe_beam_rows_kernel<__bf16><<<grid, dim3(kThreads), 0, stream>>>(a, chunks);
  else
    sfe_beam_rows_kernel<_Float16><<<grid, dim3(kThreads), 0, stream>>>(a, chunks);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  sfe_beam_streams_kernel<<<dim3((unsigned)a.streams), dim3(kThreads), 0, stream>>>(a, chunks);
  return hipGetLastError();
}

hipError_t launch_beam_reorder(const ReorderArgs& a, hipStream_t stream) {
  uintptr_t bits = 0;
  for (int k = 0; k < a.n; ++k)
    bits |= reinterpret_cast<uintptr_t>(a.s[k].in) | reinterpret_cast<uintptr_t>(a.s[k].out) | (uintptr_t)a.s[k].inner;
  if (bits % 16 == 0) return reorder_beams<U4>(a, stream);
  if (bits % 4 == 0) return reorder_beams<uint32_t>(a, stream);
  return reorder_beams<uint8_t>(a, stream);
}

}  // namespace sfe
