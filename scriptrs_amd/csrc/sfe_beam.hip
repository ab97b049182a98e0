// A step of beam search.
//
// total(w, t) = score_w + ((logit_wt - m_w) - log sum_t exp(logit_wt - m_w)), m_w the row's
// maximum: the sum and its logarithm do not see where a row lies, so that neither do its totals
// (formed as logit - (m + log sum), rows at 10^6 were off by 0.02 against each other, and a row wholly at
// the lowest f32 had none).  A finished beam has the one candidate (score_w, end token).  A stream's next beams are the best
// of its beams * vocabulary candidates, ties to the lowest (beam, token); totals of
// -inf or NaN are no candidates, and places without one hold score -inf, token
// -1 and their own beam as parent.
//
// Within a row, candidates order as its logits do, but that unequal logits may have totals that round to
// the same f32: the row's cut to `beams` is then by the logits, which say more.  Small vocabularies: one launch, a
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
typedef float F4 __attribute__((ext_vector_type(4)));
typedef int I4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kEach = 32;                // logits of a thread and step
constexpr int kStep = kThreads * kEach;  // logits of a workgroup and step
constexpr int kSmall = 64 * kEach;       // logits of a wave
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
// The n-th largest of a wave's values (-inf where fewer are above that); *qth the q-th, q <= n.
__device__ __forceinline__ float wave_nth(float x, int n, int q, float* qth) {
  float top = -INFINITY;
  const int lane = (int)(threadIdx.x & 63);
  *qth = -INFINITY;
  for (int r = 0; r < n; ++r) {
    top = wave_max(x);
    if (top == -INFINITY) break;
    if (r == q - 1) *qth = top;
    const uint64_t same = __ballot(x == top);
    if (lane == __builtin_ctzll(same)) x = -INFINITY;
  }
  return top;
}

// The best candidates (value, index) that a wave has seen: up to 64 in its part of
// LDS, in no order.  A candidate is entered if it comes before (bx, bi), which is
// never before the n-th best of all that the wave has seen; when the list is full it is cut to
// its n best, and the n-th of them is the new bound.  So ties, however many, cost
// cuts and lose nothing, and no wave waits for another.
constexpr int kListed = 64, kSlack = 4;
struct alignas(16) Lists {
  float x[16][kListed];
  int i[16][kListed];
  int n[16];
};
struct Best {
  float bx;
  int bi, n;  // n: entries (the same in every lane)
};

__device__ __forceinline__ Best best_none() { return Best{-INFINITY, INT32_MAX, 0}; }

__device__ __forceinline__ void lds_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

__device__ __forceinline__ void best_cut(Best& b, int keep, float* lx, int* li) {
  const int lane = (int)(threadIdx.x & 63);
  lds_done();
  float x = -INFINITY;
  int i = INT32_MAX;
  if (lane < b.n) {
    x = lx[lane];
    i = li[lane];
  }
  int rank = 0;
  for (int d = 0; d < b.n; ++d) {
    const float y = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), d));
    rank += before(y, __builtin_amdgcn_readlane(i, d), x, i);
  }
  if (lane < b.n && rank < keep) {
    lx[rank] = x;
    li[rank] = i;
  }
  lds_done();
  if (b.n >= keep) {
    b.n = keep;
    const float x = lx[keep - 1];
    const int i = li[keep - 1];
    if (before(x, i, b.bx, b.bi)) {  // (not where the other waves' values already say more)
      b.bx = x;
      b.bi = i;
    }
  }
}

// Enters the lanes' values v of indexes i that come before the bound.
__device__ __forceinline__ void best_enter(Best& b, int keep, float* lx, int* li, float v, int i) {
  bool c = v > -INFINITY && before(v, i, b.bx, b.bi);
  for (uint64_t mask = __ballot(c); mask; mask = __ballot(c)) {
    const int room = kListed - b.n;
    const int place = (int)__builtin_amdgcn_mbcnt_hi((uint32_t)(mask >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)mask, 0));
    if (c && place < room) {
      lx[b.n + place] = v;
      li[b.n + place] = i;
    }
    c = c && place >= room;
    b.n += min(__builtin_popcountll(mask), room);
    if (b.n == kListed) {
      best_cut(b, keep, lx, li);
      c = c && before(v, i, b.bx, b.bi);
    }
  }
}

// Maxima of a lane's values in groups of kGroup.
constexpr int kGroup = 8;
template <int E>
__device__ __forceinline__ float max_of(const float (&x)[E], float (&groups)[E / kGroup]) {
#pragma unroll
  for (int g = 0; g < E / kGroup; ++g) {
    groups[g] = x[g * kGroup];  // (fmaxf passes NaN over)
#pragma unroll
    for (int k = 1; k < kGroup; ++k) groups[g] = fmaxf(groups[g], x[g * kGroup + k]);
  }
  float m = groups[0];
#pragma unroll
  for (int g = 1; g < E / kGroup; ++g) m = fmaxf(m, groups[g]);
  return m;
}

// What the waves of a workgroup tell each other in passing: each one's share-th best value so
// far, waves * share >= keep, so that keep values are not below the least of them.  Written and
// read without a barrier: an older value is a lower bound.
struct Told {
  F4* all;  // of kWaves waves, -inf before the first; null: nobody tells
  int share;
};
__device__ __forceinline__ void tell(const Told& told, float mine) {
  if ((threadIdx.x & 63) == 0) reinterpret_cast<float*>(told.all)[threadIdx.x >> 6] = mine;
}
__device__ __forceinline__ void learn(const Told& told, Best& b) {
  asm volatile("" ::: "memory");  // (read again each time)
  const F4 v = *told.all;
  const float least = fminf(fminf(v[0], v[1]), fminf(v[2], v[3]));
  if (least > b.bx) {
    b.bx = least;
    b.bi = INT32_MAX;  // (values equal to it are entered)
  }
}

// Enters a lane's values x[0..E) of indexes index(k); top and groups: their maxima.  Only groups in
// which some lane reaches the bound are looked at value by value, each lane's values that may
// come in one a turn (a copy of the code for each of the E values would not fit the
// instruction cache).
template <int E, class F>
__device__ __forceinline__ void best_add(Best& b, int keep, float* lx, int* li, const float (&x)[E], float top,
                                         const float (&groups)[E / kGroup], F&& index, const Told& told = {nullptr, 1}) {
  if (told.all) learn(told, b);
  if (b.n == 0) {  // a first bound: the keep-th largest of the lanes' maxima
    float mine;
    const float first = wave_nth(top, keep, told.share, &mine);
    if (first > b.bx) b.bx = first;  // (b.bi stays: values equal to it are entered)
    if (told.all) tell(told, mine);
  }
  if (__ballot(top >= b.bx) == 0) return;
#pragma unroll
  for (int g = 0; g < E / kGroup; ++g) {
    if (__ballot(groups[g] >= b.bx) == 0) continue;
    uint32_t may = 0;
#pragma unroll
    for (int k = 0; k < kGroup; ++k) may |= x[g * kGroup + k] >= b.bx ? 1u << k : 0u;
    while (__ballot(may != 0)) {
      const int k = may ? __builtin_ctz(may) : 0;
      float v = x[g * kGroup];
#pragma unroll
      for (int j = 1; j < kGroup; ++j) v = k == j ? x[g * kGroup + j] : v;
      best_enter(b, keep, lx, li, may ? v : -INFINITY, index(g * kGroup + k));
      may &= may - 1;
    }
  }
  // (a bound that stays behind costs more than cutting the list: 512 rows of 128,000, 8 beams, 39.4 us
  // with a cut at every entry, 37.8 at 4 and at 8 past the beams, 43.9 when full, all of them before the maximum
  // was taken off each logit)
  if (b.n >= keep + kSlack) {
    best_cut(b, keep, lx, li);
    if (told.all) tell(told, lx[told.share - 1]);
  }
}

// The workgroup's best of its waves' lists: entry `rank` of the result is given to
// give(rank, value, index); returns how many there are (at most keep).  Barriers on
// both sides of the lists.
template <class F>
__device__ __forceinline__ int best_join(Best& b, Lists& l, int keep, F&& give) {
  const int waves = (int)blockDim.x / 64, w = (int)(threadIdx.x >> 6), e = (int)(threadIdx.x & 63);
  if (b.n > keep) best_cut(b, keep, l.x[w], l.i[w]);
  if (e >= b.n) {  // (comes before nothing)
    l.x[w][e] = -INFINITY;
    l.i[w][e] = INT32_MAX;
  }
  if (e == 0) l.n[w] = b.n;
  __syncthreads();
  int total = 0;
  for (int v = 0; v < waves; ++v) total += l.n[v];
  // a thread takes entry t % 64 of wave t / 64
  if (e < b.n) {
    const float x = l.x[w][e];
    const int i = l.i[w][e];
    int rank = 0;
    for (int v = 0; v < waves; ++v)
      for (int d = 0; d < keep; d += 4) {
        const F4 y = *reinterpret_cast<const F4*>(&l.x[v][d]);
        const I4 j = *reinterpret_cast<const I4*>(&l.i[v][d]);
#pragma unroll
        for (int c = 0; c < 4; ++c) rank += before(y[c], j[c], x, i);
      }
    if (rank < keep) give(rank, x, i);
  }
  return min(keep, total);
}

// 16 bytes of a row, read at an element's own alignment: which thread adds which logit
// does not depend on where a row starts (a vocabulary of odd size puts rows on every
// alignment).
struct __attribute__((packed, aligned(2))) Raw {
  U4 v;
};
template <typename T>
struct Bits;
template <>
struct Bits<float> {
  static __device__ float at(const U4& v, int i) { return __uint_as_float(v[i]); }
};
template <>
struct Bits<__bf16> {
  static __device__ float at(const U4& v, int i) {
    return __uint_as_float(i % 2 ? v[i / 2] & 0xffff0000u : v[i / 2] << 16);
  }
};
template <>
struct Bits<_Float16> {
  static __device__ float at(const U4& v, int i) {
    return (float)__builtin_bit_cast(_Float16, (unsigned short)(v[i / 2] >> (i % 2 * 16)));
  }
};

// Vector j of thread t of a row holds the elements from first + (j * THREADS + t) * N on;
// one that would pass the row's end is moved back to end with it, and its elements that
// belong to the vector before do not count.  (Rows shorter than a vector are read by the
// element.)
template <int N, int THREADS>
__device__ __forceinline__ int vector_at(int first, int j, int t) { return first + (j * THREADS + t) * N; }
template <int N>
__device__ __forceinline__ int moved_back(int e, int vocab) { return vocab >= N ? min(e, vocab - N) : e; }

template <typename T, int NV, int THREADS>
__device__ __forceinline__ void load_row(const T* p, int first, int t, int vocab, U4 (&v)[NV]) {
  constexpr int N = 16 / (int)sizeof(T);
  if (vocab >= N) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
      v[j] = reinterpret_cast<const Raw*>(p + moved_back<N>(vector_at<N, THREADS>(first, j, t), vocab))->v;
    return;
  }
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = vector_at<N, THREADS>(first, j, t);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4) {
        v[j][i] = e + i < vocab ? __float_as_uint((float)p[e + i]) : 0;
      } else {
        const unsigned short* h = reinterpret_cast<const unsigned short*>(p);
        const unsigned lo = e + 2 * i < vocab ? h[e + 2 * i] : 0, hi = e + 2 * i + 1 < vocab ? h[e + 2 * i + 1] : 0;
        v[j][i] = lo | hi << 16;
      }
    }
  }
}
// The vectors as floats, -inf where they do not count.
template <typename T, int NV, int THREADS>
__device__ __forceinline__ void row_values(const U4 (&v)[NV], int first, int t, int vocab, float (&x)[NV * 16 / sizeof(T)]) {
  constexpr int N = 16 / (int)sizeof(T);
#pragma unroll
  for (int k = 0; k < NV * N; ++k) x[k] = Bits<T>::at(v[k / N], k % N);
  if (first + NV * THREADS * N <= vocab) return;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int e = vector_at<N, THREADS>(first, j, t), at = moved_back<N>(e, vocab);
#pragma unroll
    for (int i = 0; i < N; ++i) x[j * N + i] = at + i >= e && at + i < vocab ? x[j * N + i] : -INFINITY;
  }
}
// The token of value k.
template <typename T, int THREADS>
__device__ __forceinline__ int token_of(int k, int first, int t, int vocab) {
  constexpr int N = 16 / (int)sizeof(T);
  return moved_back<N>(vector_at<N, THREADS>(first, k / N, t), vocab) + k % N;
}

// Sum of exponentials of x - m (0 where all is -inf; NaN stays).
template <int E>
__device__ __forceinline__ float exp_sum(const float (&x)[E], float m) {
  const float r = m == -INFINITY ? 0.0f : m;
  float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int k = 0; k < E; ++k) s[k % 4] += __builtin_amdgcn_exp2f((x[k] - r) * kLog2e);
  return (s[0] + s[1]) + (s[2] + s[3]);
}
__device__ __forceinline__ void write_beam(const BeamArgs& a, int stream, int r, bool found, float x, int i) {
  const int parent = found ? i / a.vocab : r, token = found ? i - parent * a.vocab : -1;
  const int64_t o = (int64_t)stream * a.beams + r;
  a.out_scores[o] = x;
  a.parents[o] = parent;
  a.tokens[o] = token;
  if (a.out_finished)
    a.out_finished[o] = (a.finished && a.finished[(int64_t)stream * a.beams + parent]) || (found && token == a.end);
}
__device__ __forceinline__ void write_beams(const BeamArgs& a, int stream, Best& b, Lists& l) {
  const int found = best_join(b, l, a.beams, [&](int r, float x, int i) { write_beam(a, stream, r, true, x, i); });
  const int t = (int)threadIdx.x;
  if (t >= found && t < a.beams) write_beam(a, stream, t, false, -INFINITY, 0);
}

// ---- small vocabularies -----------------------------------------------------------------

// E: logits of a lane.  16 streams of 4 beams over 1,025 tokens in f32: 7.6 us, bound by latency (a
// row's loads, its sum, the choice, the join).
template <typename T, int E>
__global__ __launch_bounds__(1024) void sfe_beam_small_kernel(BeamArgs a) {
  constexpr int NV = E * (int)sizeof(T) / 16;
  __shared__ Lists lists;
  const int stream = (int)blockIdx.x, lane = (int)(threadIdx.x & 63), waves = (int)blockDim.x / 64;
  const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
  Best best = best_none();
  for (int w = wave; w < a.beams; w += waves) {
    const int64_t row = (int64_t)stream * a.beams + w;
    const float score = a.scores[row];
    if (a.finished && a.finished[row]) {
      best_enter(best, a.beams, lists.x[wave], lists.i[wave], lane == 0 ? score : -INFINITY, w * a.vocab + a.end);
      continue;
    }
    U4 v[NV];
    load_row<T, NV, 64>(reinterpret_cast<const T*>(a.logits) + row * a.row, 0, lane, a.vocab, v);
    float x[E], groups[E / kGroup];
    row_values<T, NV, 64>(v, 0, lane, a.vocab, x);
    const float m = wave_max(max_of(x, groups));
    const float log_sum = logf(wave_sum(exp_sum(x, m)));
#pragma unroll
    for (int k = 0; k < E; ++k) x[k] = score + ((x[k] - m) - log_sum);
    const float top = max_of(x, groups);
    best_add(best, a.beams, lists.x[wave], lists.i[wave], x, top, groups,
             [&](int k) { return w * a.vocab + token_of<T, 64>(k, 0, lane, a.vocab); });
  }
  write_beams(a, stream, best, lists);
}

// ---- others: spans of rows, then streams -----------------------------------------------------

// One workgroup: the steps of a span, the next step's loads in flight while one is
// worked on.  512 rows of 128,000 in bf16, 8 beams: 40 us, of which the pass over the logits
// alone takes 25 (5.2 TB/s), the best 8 of the first step and of the waves 4 each, and the maximum taken off
// each logit 2.  Each thread keeps the sum of exponentials relative to its own running maximum.  (4 workgroups a CU: with 3, which 155 registers allow, 1,024 of them
// went in two turns, 90 us against 55.)
template <typename T>
__global__ __launch_bounds__(kThreads, 4) void sfe_beam_rows_kernel(BeamArgs a, int spans) {
  constexpr int N = 16 / (int)sizeof(T), NV = kEach / N;
  __shared__ Lists lists;
  __shared__ Part parts[kWaves];
  __shared__ F4 known;
  const int row = (int)(blockIdx.x / (unsigned)spans), span = (int)(blockIdx.x % (unsigned)spans);
  const int t = (int)threadIdx.x, wave = __builtin_amdgcn_readfirstlane(t >> 6);
  Part* part = reinterpret_cast<Part*>(a.scratch);
  Cand* cand = reinterpret_cast<Cand*>(part + (int64_t)a.streams * a.beams * spans);
  const int64_t at = (int64_t)row * spans + span;
  if (a.finished && a.finished[row]) return;  // (its logits are not looked at)
  const T* p = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.row;
  const int steps = (a.vocab + kStep - 1) / kStep;
  const int step0 = (int)((int64_t)steps * span / spans), step1 = (int)((int64_t)steps * (span + 1) / spans);
  static_assert(kWaves == 4, "Told");
  if (t < kWaves) reinterpret_cast<float*>(&known)[t] = -INFINITY;
  __syncthreads();
  const Told told{&known, (a.beams + kWaves - 1) / kWaves};
  Best best = best_none();
  float tm = -INFINITY, sum = 0.0f;
  U4 next[NV];
  if (step0 < step1) load_row<T, NV, kThreads>(p, step0 * kStep, t, a.vocab, next);
  for (int step = step0; step < step1; ++step) {
    float x[kEach], groups[kEach / kGroup];
    row_values<T, NV, kThreads>(next, step * kStep, t, a.vocab, x);
    if (step + 1 < step1) load_row<T, NV, kThreads>(p, (step + 1) * kStep, t, a.vocab, next);
    const float sm = max_of(x, groups), m = fmaxf(tm, sm);
    sum = sum * (tm == m ? 1.0f : __builtin_amdgcn_exp2f((tm - m) * kLog2e)) + exp_sum(x, m);
    tm = m;
    best_add(best, a.beams, lists.x[wave], lists.i[wave], x, sm, groups,
             [&](int k) { return token_of<T, kThreads>(k, step * kStep, t, a.vocab); }, told);
  }
  const float wm = wave_max(tm);
  const float ws = wave_sum(sum * (tm == wm ? 1.0f : __builtin_amdgcn_exp2f((tm - wm) * kLog2e)));
  if ((t & 63) == 0) parts[wave] = Part{wm, ws};
  const int found = best_join(best, lists, a.beams, [&](int r, float x, int i) { cand[at * a.beams + r] = Cand{x, i}; });
  if (t >= found && t < a.beams) cand[at * a.beams + t] = Cand{-INFINITY, -1};
  if (t == 0) {
    Part r{-INFINITY, 0.0f};
    for (int w = 0; w < kWaves; ++w) r.top = fmaxf(r.top, parts[w].top);
    for (int w = 0; w < kWaves; ++w)
      r.sum += parts[w].sum * (parts[w].top == r.top ? 1.0f : __builtin_amdgcn_exp2f((parts[w].top - r.top) * kLog2e));
    part[at] = r;
  }
}

// A workgroup per stream, over the candidates its rows' spans left: 9 us for 64 streams of 8 beams, bound by
// latency (one row's sums, one round of candidates, the join).
__global__ __launch_bounds__(kThreads) void sfe_beam_streams_kernel(BeamArgs a, int spans) {
  __shared__ Lists lists;
  __shared__ float tops[kMaxBeams], log_sums[kMaxBeams];
  const int b = (int)blockIdx.x, t = (int)threadIdx.x, W = a.beams;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const Part* part = reinterpret_cast<const Part*>(a.scratch) + (int64_t)b * W * spans;
  const Cand* cand = reinterpret_cast<const Cand*>(reinterpret_cast<const Part*>(a.scratch) +
                                                   (int64_t)a.streams * W * spans) + (int64_t)b * W * spans * W;
  const float* scores = a.scores + (int64_t)b * W;
  const uint8_t* finished = a.finished ? a.finished + (int64_t)b * W : nullptr;
  for (int w = wave; w < W; w += kWaves) {
    if (finished && finished[w]) continue;
    float top = -INFINITY, sum = 0.0f;
    for (int c = t & 63; c < spans; c += 64) top = fmaxf(top, part[w * spans + c].top);
    top = wave_max(top);
    for (int c = t & 63; c < spans; c += 64) {
      const Part p = part[w * spans + c];
      sum += p.sum * (p.top == top ? 1.0f : __builtin_amdgcn_exp2f((p.top - top) * kLog2e));
    }
    sum = wave_sum(sum);
    if ((t & 63) == 0) {
      tops[w] = top;
      log_sums[w] = logf(sum);
    }
  }
  __syncthreads();
  Best best = best_none();
  const int each = spans * W;  // candidates of a row
  for (int e0 = 64 * wave; e0 < W * each; e0 += kThreads) {
    const int e = e0 + (t & 63);
    float x = -INFINITY;
    int i = 0;
    if (e < W * each) {
      const int w = e / each;
      if (finished && finished[w]) {
        if (e == w * each) x = scores[w];
        i = w * a.vocab + a.end;
      } else {
        const Cand c = cand[e];
        i = w * a.vocab + c.t;
        if (c.t >= 0) x = scores[w] + ((c.x - tops[w]) - log_sums[w]);
      }
    }
    best_enter(best, W, lists.x[wave], lists.i[wave], x, i);
  }
  write_beams(a, b, best, lists);
}

// ---- states ------------------------------------------------------------------------------

// A thread moves one column (sizeof(V) bytes) of all of a stream's beams: every
// beam is read before any is written, so a state may be reordered in place.  A
// workgroup's columns are of one state, outer index and stream, so the parents are
// scalars.  Bound by memory: 50 MB read and 50 written in 17 us, 5.9 TB/s (all loads at once without a
// branch; 27 us with one for each beam).  first[k]: workgroups of the states before k.
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
  for (int w = 0; w < BEAMS; ++w) {
    const int u = min(w, a.beams - 1);  // (past the last: read again, not written)
    int p = parents[u];
    if (p < 0 || p >= a.beams) p = u;  // (no such beam: stays)
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
    const dim3 grid((unsigned)a.streams), block(64 * std::min(a.beams, 16));
    if (a.vocab <= 64 * 16)
      sfe_beam_small_kernel<T, 16><<<grid, block, 0, stream>>>(a);
    else if (a.vocab <= 64 * 24)
      sfe_beam_small_kernel<T, 24><<<grid, block, 0, stream>>>(a);
    else
      sfe_beam_small_kernel<T, kEach><<<grid, block, 0, stream>>>(a);
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
