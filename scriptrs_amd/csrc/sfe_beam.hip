// A step of beam search.
//
// total(w, t) = score_w + (logit_wt - log sum_t exp(logit_wt)); a finished beam
// has the one candidate (score_w, end token).  A stream's next beams are the best
// of its beams * vocabulary candidates, ties to the lowest (beam, token); totals of
// -inf or NaN are no candidates, and places without one hold score -inf, token
// -1 and their own beam as parent.
//
// Within a row, candidates order as its logits do.  Small vocabularies: one launch, a
// workgroup per stream and a wave per row, the row in registers.  Others: two; the
// first reads each logit once, a workgroup leaving its span's maximum, sum of
// exponentials and `beams` best logits, and the second chooses among beams * spans *
// beams candidates a stream.  Bound by memory (the logits) where the vocabulary is
// large, by latency where it is small.  Sums are f32 and every order of addition is
// fixed.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "sfe_ops.hpp"

namespace sfe {
namespace {

typedef unsigned U4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kEach = 32;                // logits of a thread and step
constexpr int kStep = kThreads * kEach;  // logits of a workgroup and step
constexpr int kSmall = 64 * kEach;       // logits of a wave
constexpr int kList = 512;               // candidates held at once
constexpr float kLog2e = 1.44269504f;

// Scratch: [row][span] of (maximum, sum), then of beams (logit, token).
struct Part {
  float top, sum;
};
struct Cand {
  float x;
  int32_t t;
};

__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(x), CTRL, 0xf, 0xf, true));
}
// Maximum (sum) over a wave's 64 lanes, in every lane: within rows of 16 by
// rotations, then across the rows.
__device__ __forceinline__ float across_rows_max(float x) {
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(q[0]), __uint_as_float(q[1]));
}
__device__ __forceinline__ float wave_max(float x) {
  x = fmaxf(x, dpp<0x128>(x));  // row_ror:8, 4, 2, 1
  x = fmaxf(x, dpp<0x124>(x));
  x = fmaxf(x, dpp<0x122>(x));
  x = fmaxf(x, dpp<0x121>(x));
  return across_rows_max(x);
}
__device__ __forceinline__ float wave_sum(float x) {
  x += dpp<0x128>(x);
  x += dpp<0x124>(x);
  x += dpp<0x122>(x);
  x += dpp<0x121>(x);
  const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = __uint_as_float(p[0]) + __uint_as_float(p[1]);
  const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(q[0]) + __uint_as_float(q[1]);
}
// The n-th largest of a wave's values (-inf where fewer are above that).
__device__ __forceinline__ float wave_nth(float x, int n) {
  float top = -INFINITY;
  const int lane = (int)(threadIdx.x & 63);
  for (int r = 0; r < n; ++r) {
    top = wave_max(x);
    if (top == -INFINITY) break;
    const uint64_t same = __ballot(x == top);
    if (lane == __builtin_ctzll(same)) x = -INFINITY;
  }
  return top;
}

// The best `n` candidates (value, index) that a workgroup has seen, in LDS, best
// first.  A candidate is entered if it is not below `bound`, which is never above the
// n-th best: after the first values few are.
struct Best {
  float bound;
  int count, kept, cur;
  float wx[16];
  int wi[16];
  float cx[kList], kx[2][kMaxBeams];
  int ci[kList], ki[2][kMaxBeams];
};

__device__ __forceinline__ void best_clear(Best& b) {
  if (threadIdx.x == 0) {
    b.bound = -INFINITY;
    b.count = b.kept = b.cur = 0;
  }
  __syncthreads();
}

// Enters a thread's values x[0..E) of indexes index(k); top: their maximum.  Called by
// the whole workgroup; first: a first bound is taken from the thread maxima.
template <int E, class F>
__device__ __forceinline__ void best_add(Best& b, int n, const float (&x)[E], float top, bool first, F&& index) {
  const int t = (int)threadIdx.x, waves = (int)blockDim.x / 64;
  if (first) {
    const float w = wave_nth(top, n);
    if ((t & 63) == 0) b.wx[t >> 6] = w;
    __syncthreads();
    float m = b.bound;
    for (int i = 0; i < waves; ++i) m = fmaxf(m, b.wx[i]);
    __syncthreads();
    if (t == 0) b.bound = m;
    __syncthreads();
  }
  const float bound = b.bound;
  if (top >= bound && top > -INFINITY) {
#pragma unroll
    for (int k = 0; k < E; ++k)
      if (x[k] >= bound && x[k] > -INFINITY) {
        const int c = atomicAdd(&b.count, 1);
        if (c < kList) {
          b.cx[c] = x[k];
          b.ci[c] = index(k);
        }
      }
  }
  __syncthreads();
  const int add = b.count, have = b.kept, cur = b.cur;
  __syncthreads();
  if (add == 0) return;
  const float* ox = b.kx[cur];
  const int* oi = b.ki[cur];
  float* nx = b.kx[cur ^ 1];
  int* ni = b.ki[cur ^ 1];
  int found = 0;
  if (add <= kList) {
    // by rank: the list's order does not matter
    for (int c = t; c < add + have; c += (int)blockDim.x) {
      const float y = c < add ? b.cx[c] : ox[c - add];
      const int i = c < add ? b.ci[c] : oi[c - add];
      int rank = 0;
      for (int d = 0; d < add; ++d) rank += before(b.cx[d], b.ci[d], y, i);
      for (int d = 0; d < have; ++d) rank += before(ox[d], oi[d], y, i);
      if (rank < n) {
        nx[rank] = y;
        ni[rank] = i;
      }
    }
    found = min(n, add + have);
  } else {
    // many equal values: the best after the last one taken, n times
    float lastx = INFINITY;
    int lasti = -1;
    for (; found < n; ++found) {
      float y = -INFINITY;
      int i = INT32_MAX;
      if (t < have && before(lastx, lasti, ox[t], oi[t])) {
        y = ox[t];
        i = oi[t];
      }
#pragma unroll
      for (int k = 0; k < E; ++k) {
        const int j = index(k);
        if (x[k] > -INFINITY && before(lastx, lasti, x[k], j) && before(x[k], j, y, i)) {
          y = x[k];
          i = j;
        }
      }
      const float wy = wave_max(y);
      int wi = y == wy ? i : INT32_MAX;
#pragma unroll
      for (int d = 32; d > 0; d >>= 1) wi = min(wi, __shfl_xor(wi, d));
      if ((t & 63) == 0) {
        b.wx[t >> 6] = wy;
        b.wi[t >> 6] = wi;
      }
      __syncthreads();
      lastx = b.wx[0];
      lasti = b.wi[0];
      for (int w = 1; w < waves; ++w)
        if (before(b.wx[w], b.wi[w], lastx, lasti)) {
          lastx = b.wx[w];
          lasti = b.wi[w];
        }
      __syncthreads();
      if (lasti == INT32_MAX) break;
      if (t == 0) {
        nx[found] = lastx;
        ni[found] = lasti;
      }
    }
  }
  __syncthreads();
  if (t == 0) {
    b.count = 0;
    b.kept = found;
    b.cur = cur ^ 1;
    if (found == n) b.bound = fmaxf(b.bound, nx[n - 1]);
  }
  __syncthreads();
}

// 16 bytes at an element's own alignment: which thread adds which logit does not
// depend on where a row starts (a vocabulary of odd size puts rows on every alignment).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Vec {
  T v[16 / sizeof(T)];
};

// Vector j of thread t: the elements first + (j * THREADS + t) * N.. of a row, -inf past
// its end.
template <typename T, int NV, int THREADS>
__device__ __forceinline__ void load_row(const T* p, int first, int t, int vocab, Vec<T> (&v)[NV]) {
  constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = first + (j * THREADS + t) * N;
    if (e + N <= vocab) {
      v[j] = *reinterpret_cast<const Vec<T>*>(p + e);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[j].v[i] = e + i < vocab ? p[e + i] : (T)-INFINITY;
    }
  }
}

// Sum of exponentials of x relative to m (0 where all is -inf; NaN stays).
template <int E>
__device__ __forceinline__ float exp_sum(const float (&x)[E], float m) {
  const float c = m == -INFINITY ? 0.0f : m;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < E; ++k) s[k % 4] += __builtin_amdgcn_exp2f((x[k] - c) * kLog2e);
  return (s[0] + s[1]) + (s[2] + s[3]);
}
template <int E>
__device__ __forceinline__ float max_of(const float (&x)[E]) {
  float m = x[0];  // (fmaxf passes NaN over)
#pragma unroll
  for (int k = 1; k < E; ++k) m = fmaxf(m, x[k]);
  return m;
}

__device__ __forceinline__ void write_beams(const BeamArgs& a, const Best& b, int stream) {
  const int r = (int)threadIdx.x;
  if (r >= a.beams) return;
  const bool found = r < b.kept;
  const int i = b.ki[b.cur][r];
  const int parent = found ? i / a.vocab : r, token = found ? i - parent * a.vocab : -1;
  const int64_t o = (int64_t)stream * a.beams + r;
  a.out_scores[o] = found ? b.kx[b.cur][r] : -INFINITY;
  a.parents[o] = parent;
  a.tokens[o] = token;
  if (a.out_finished)
    a.out_finished[o] = (a.finished && a.finished[(int64_t)stream * a.beams + parent]) || (found && token == a.end);
}

// ---- small vocabularies -----------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(1024) void sfe_beam_small_kernel(BeamArgs a) {
  constexpr int N = 16 / (int)sizeof(T), NV = kEach / N;
  __shared__ Best best;
  const int stream = (int)blockIdx.x, lane = (int)(threadIdx.x & 63), waves = (int)blockDim.x / 64;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  best_clear(best);
  for (int w0 = 0; w0 < a.beams; w0 += waves) {
    const int w = w0 + wave;
    float x[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) x[k] = -INFINITY;
    bool over = false;
    if (w < a.beams) {
      const int64_t row = (int64_t)stream * a.beams + w;
      over = a.finished && a.finished[row];
      const float score = a.scores[row];
      if (over) {
        if (lane == 0) x[0] = score;
      } else {
        const T* p = reinterpret_cast<const T*>(a.logits) + row * a.row;
        Vec<T> v[NV];
        load_row<T, NV, 64>(p, 0, lane, a.vocab, v);
#pragma unroll
        for (int k = 0; k < kEach; ++k) x[k] = (float)v[k / N].v[k % N];
        const float m = wave_max(max_of(x));
        const float logz = m + logf(wave_sum(exp_sum(x, m)));
#pragma unroll
        for (int k = 0; k < kEach; ++k) x[k] = score + (x[k] - logz);
      }
    }
    best_add(best, a.beams, x, max_of(x), w0 == 0, [&](int k) {
      return w * a.vocab + (over ? a.end : (k / N * 64 + lane) * N + k % N);
    });
  }
  write_beams(a, best, stream);
}

// ---- others: spans of rows, then streams -----------------------------------------------------

// One workgroup: the steps of a span, the next step's loads in flight while one is
// worked on.  Each thread keeps the sum of exponentials relative to its own running
// maximum.
template <typename T>
__global__ __launch_bounds__(kThreads) void sfe_beam_rows_kernel(BeamArgs a, int spans) {
  constexpr int N = 16 / (int)sizeof(T), NV = kEach / N;
  __shared__ Best best;
  const int row = (int)(blockIdx.x / (unsigned)spans), span = (int)(blockIdx.x % (unsigned)spans);
  const int t = (int)threadIdx.x;
  Part* part = reinterpret_cast<Part*>(a.scratch);
  Cand* cand = reinterpret_cast<Cand*>(part + (int64_t)a.streams * a.beams * spans);
  const int64_t at = (int64_t)row * spans + span;
  if (a.finished && a.finished[row]) return;  // (its logits are not looked at)
  const T* p = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.row;
  const int steps = (a.vocab + kStep - 1) / kStep;
  const int step0 = (int)((int64_t)steps * span / spans), step1 = (int)((int64_t)steps * (span + 1) / spans);
  best_clear(best);
  float tm = -INFINITY, sum = 0.0f;
  Vec<T> next[NV];
  if (step0 < step1) load_row<T, NV, kThreads>(p, step0 * kStep, t, a.vocab, next);
  for (int step = step0; step < step1; ++step) {
    float x[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) x[k] = (float)next[k / N].v[k % N];
    if (step + 1 < step1) load_row<T, NV, kThreads>(p, (step + 1) * kStep, t, a.vocab, next);
    const float sm = max_of(x), m = fmaxf(tm, sm);
    sum = sum * (tm == m ? 1.0f : __builtin_amdgcn_exp2f((tm - m) * kLog2e)) + exp_sum(x, m);
    tm = m;
    best_add(best, a.beams, x, sm, step == step0,
             [&](int k) { return step * kStep + (k / N * kThreads + t) * N + k % N; });
  }
  const float wm = wave_max(tm);
  const float ws = wave_sum(sum * (tm == wm ? 1.0f : __builtin_amdgcn_exp2f((tm - wm) * kLog2e)));
  __shared__ Part waves[kWaves];
  if ((t & 63) == 0) waves[t >> 6] = Part{wm, ws};
  __syncthreads();
  if (t == 0) {
    Part r{-INFINITY, 0.0f};
    for (int w = 0; w < kWaves; ++w) r.top = fmaxf(r.top, waves[w].top);
    for (int w = 0; w < kWaves; ++w)
      r.sum += waves[w].sum * (waves[w].top == r.top ? 1.0f : __builtin_amdgcn_exp2f((waves[w].top - r.top) * kLog2e));
    part[at] = r;
  }
  if (t < a.beams)
    cand[at * a.beams + t] = t < best.kept ? Cand{best.kx[best.cur][t], best.ki[best.cur][t]} : Cand{-INFINITY, -1};
}

__global__ __launch_bounds__(kThreads) void sfe_beam_streams_kernel(BeamArgs a, int spans) {
  __shared__ Best best;
  __shared__ float logz[kMaxBeams];
  const int b = (int)blockIdx.x, t = (int)threadIdx.x, W = a.beams;
  const Part* part = reinterpret_cast<const Part*>(a.scratch) + (int64_t)b * W * spans;
  const Cand* cand = reinterpret_cast<const Cand*>(reinterpret_cast<const Part*>(a.scratch) +
                                                   (int64_t)a.streams * W * spans) + (int64_t)b * W * spans * W;
  const float* scores = a.scores + (int64_t)b * W;
  const uint8_t* finished = a.finished ? a.finished + (int64_t)b * W : nullptr;
  for (int w = t >> 6; w < W; w += kWaves) {
    if (finished && finished[w]) continue;
    float top = -INFINITY, sum = 0.0f;
    for (int c = t & 63; c < spans; c += 64) top = fmaxf(top, part[w * spans + c].top);
    top = wave_max(top);
    for (int c = t & 63; c < spans; c += 64) {
      const Part p = part[w * spans + c];
      sum += p.sum * (p.top == top ? 1.0f : __builtin_amdgcn_exp2f((p.top - top) * kLog2e));
    }
    sum = wave_sum(sum);
    if ((t & 63) == 0) logz[w] = top + logf(sum);
  }
  best_clear(best);
  const int each = spans * W;  // candidates of a row
  for (int e0 = 0; e0 < W * each; e0 += kThreads) {
    const int e = e0 + t;
    float x[1] = {-INFINITY};
    int i = 0;
    if (e < W * each) {
      const int w = e / each;
      if (finished && finished[w]) {
        if (e == w * each) x[0] = scores[w];
        i = w * a.vocab + a.end;
      } else {
        const Cand c = cand[e];
        i = w * a.vocab + c.t;
        if (c.t >= 0) x[0] = scores[w] + (c.x - logz[w]);
      }
    }
    best_add(best, W, x, x[0], e0 == 0, [&](int) { return i; });
  }
  write_beams(a, best, b);
}

// ---- states ------------------------------------------------------------------------------

// A thread moves one column (sizeof(V) bytes) of all of a stream's beams: every
// beam is read before any is written, so a state may be reordered in place.  A
// workgroup's columns are of one state, outer index and stream, so the parents are
// scalars.  first[k]: workgroups of the states before k.
struct ReorderGrid {
  uint32_t first[kReorderStates + 1];
  uint32_t blocks[kReorderStates];   // workgroups of a stream
  uint32_t stream0[kReorderStates];  // stream of the first
};

template <typename V, int BEAMS>
__global__ __launch_bounds__(kThreads) void sfe_beam_reorder_kernel(ReorderArgs a, ReorderGrid g) {
  int k = 0;
  while (blockIdx.x >= g.first[k + 1]) ++k;
  const uint32_t b = blockIdx.x - g.first[k];
  const uint32_t os = b / g.blocks[k], stream = (g.stream0[k] + os) % (uint32_t)a.streams;
  const BeamState& s = a.s[k];
  const int64_t col = ((int64_t)(b - os * g.blocks[k]) * kThreads + threadIdx.x) * (int64_t)sizeof(V);
  if (col >= s.inner) return;
  const int32_t* parents = a.parents + (int64_t)stream * a.beams;
  const char* in = s.in + (int64_t)os * a.beams * s.inner + col;
  char* out = s.out + (int64_t)os * a.beams * s.inner + col;
  V v[BEAMS];
#pragma unroll
  for (int w = 0; w < BEAMS; ++w)
    if (w < a.beams) {
      int p = parents[w];
      if (p < 0 || p >= a.beams) p = w;  // (no such beam: stays)
      v[w] = *reinterpret_cast<const V*>(in + p * s.inner);
    }
#pragma unroll
  for (int w = 0; w < BEAMS; ++w)
    if (w < a.beams) *reinterpret_cast<V*>(out + w * s.inner) = v[w];
}

// The states of `all` in as few launches as hold them, each of at most 2^23
// workgroups.
template <typename V, int BEAMS>
hipError_t reorder(const ReorderArgs& all, hipStream_t stream) {
  constexpr int64_t kMost = (int64_t)1 << 23;
  ReorderArgs a = all;
  ReorderGrid g{};
  a.n = 0;
  auto go = [&]() -> hipError_t {
    if (a.n == 0) return hipSuccess;
    sfe_beam_reorder_kernel<V, BEAMS><<<dim3(g.first[a.n]), dim3(kThreads), 0, stream>>>(a, g);
    a.n = 0;
    return hipGetLastError();
  };
  for (int k = 0; k < all.n; ++k) {
    const BeamState& s = all.s[k];
    const int64_t blocks = (s.inner / (int64_t)sizeof(V) + kThreads - 1) / kThreads;  // (at most kMost: 2^31 bytes)
    const int64_t groups = s.outer * all.streams;
    for (int64_t o = 0; o < groups;) {
      if (a.n == kReorderStates || (a.n && g.first[a.n] + blocks > kMost)) {
        const hipError_t e = go();
        if (e != hipSuccess) return e;
      }
      const int64_t n = std::min(groups - o, (kMost - g.first[a.n]) / blocks);
      const int64_t skip = o * all.beams * s.inner;
      a.s[a.n] = BeamState{s.in + skip, s.out + skip, s.outer, s.inner};
      g.blocks[a.n] = (uint32_t)blocks;
      g.stream0[a.n] = (uint32_t)(o % all.streams);
      g.first[a.n + 1] = g.first[a.n] + (uint32_t)(blocks * n);
      ++a.n;
      o += n;
    }
  }
  return go();
}
template <typename V>
hipError_t reorder_beams(const ReorderArgs& a, hipStream_t stream) {
  if (a.beams <= 4) return reorder<V, 4>(a, stream);
  if (a.beams <= 8) return reorder<V, 8>(a, stream);
  return reorder<V, 32>(a, stream);
}

// Spans of a row: enough workgroups for 4 a CU (a span is at least one step).
int spans_of(int rows, int vocab, int cus) {
  const int64_t steps = (vocab + kStep - 1) / kStep;
  return (int)std::max<int64_t>(1, std::min<int64_t>(steps, ((int64_t)4 * cus + rows - 1) / rows));
}
bool small(int vocab) { return vocab <= kSmall; }

template <typename T>
hipError_t select(const BeamArgs& a, int cus, hipStream_t stream) {
  if (small(a.vocab)) {
    sfe_beam_small_kernel<T><<<dim3((unsigned)a.streams), dim3(64 * std::min(a.beams, 16)), 0, stream>>>(a);
    return hipGetLastError();
  }
  const int rows = a.streams * a.beams, spans = spans_of(rows, a.vocab, cus);
  sfe_beam_rows_kernel<T><<<dim3((unsigned)rows * (unsigned)spans), dim3(kThreads), 0, stream>>>(a, spans);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  sfe_beam_streams_kernel<<<dim3((unsigned)a.streams), dim3(kThreads), 0, stream>>>(a, spans);
  return hipGetLastError();
}

}  // namespace

size_t beam_scratch_bytes(int streams, int beams, int vocab, int cus) {
  if (small(vocab)) return 0;
  const int64_t parts = (int64_t)streams * beams * spans_of(streams * beams, vocab, cus);
  return (size_t)(parts * (int64_t)sizeof(Part) + parts * beams * (int64_t)sizeof(Cand));
}

hipError_t launch_beam_select(const BeamArgs& a, int type, int cus, hipStream_t stream) {
  if (type == kOpF32) return select<float>(a, cus, stream);
  if (type == kOpBf16) return select<__bf16>(a, cus, stream);
  return select<_Float16>(a, cus, stream);
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
