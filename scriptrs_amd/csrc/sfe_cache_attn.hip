// Attention of a sequence's new tokens, drafted as a tree or following each other, over its paged cache.
//
// For new token i of n of a sequence of L tokens, head h reading kv head h / group:
// o_i = sum_j softmax_j(scale q_i . k_j) v_j over the context (j < L - n) and the new tokens that i sees:
// those of its tree's bits, or without a tree itself and those before.  One pass over the keys with a running
// reference exponent and sum in f32, as in sfe_attn.hip: a step's maximum m' replaces m only when it is kRise above it, and
// o and l are then multiplied by 2^(m - m').
//
// Rows of a unit (a kv head and up to 128 of a sequence's token x head of the group) are the columns of both matrix products,
// so that a group's heads share the reads of their kv head: S^T = K Q^T leaves a lane with one query's scores of the 8
// keys that O^T = V^T P^T takes from it, once V's rows are paired by key in registers.  The order of channels in a product
// is free, so lanes read whole chunks of K and of V.
//
// Codes of 8 bits are of the queries' type in the first product and f16 in the second, both of which hold them exactly: a
// key's scale multiplies its scores, a value's scale its weight, in f32.  Weights times value scales are kept relative to a power of
// two, since f16 lacks their range: it goes down with the weights and up with the largest product seen, so that a token's
// scale counts only as far as its weight does.  They are rounded once to 11 bits, or where the queries are f16 (and outputs have 11
// bits too) to 22, as two numbers; to multiples of 2^-28 of a row's largest where that is more.  16-bit caches multiply in their
// own type, weights rounded once to it.
//
// A step is 32 keys.  Pages are looked up a step ahead; rows go from memory into LDS directly, and what lies past a
// sequence's end or in no page is read as zeros by the buffer's range, so that nothing is read outside a record.  Up to 32 rows
// a workgroup's four waves take steps of their own, through rings of two stages of their own, without a barrier in the
// loop; of 64 and 128 rows two and four waves read the same steps from a ring of three, with one barrier a step (codes are then
// converted once for 32 rows a wave; 64 rows a wave took 180 us where this takes 84, since its accumulators left the
// registers that the products write).
//
// What bounds it: one token a sequence, memory and the trip of a unit (256 x 126-1,500 tokens, 16/4 heads of 128 in e4m3:
// 152 MB in 40 us, 3.8 TB/s; 2 x 5 tokens over 45,000, 8 heads of 64 in f16: 184 MB in 35 us, 5.2 TB/s, and 5 of the
// join); trees, vector instructions beside the matrix cores (32 x 16 over 700-8,192, 32/8 heads of 128 in int8: 204 MB in 76
// us and 9 of the join; 63% of the CUs' time issues vector instructions, 15% of it products).  A step of 32 keys and 32 rows takes
// about 450 of them: conversions of both operands' codes (by both waves of a pair, the same), two products a weight for its
// scale, exponentials and maxima.  Runs of hundreds of tokens are bound by the same: 380-670 TFLOP/s where long products reach 1,352.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "sfe_cache.hpp"
#include "sfe_internal.hpp"
#include "sfe_mat.hpp"

namespace sfe {
namespace {

constexpr int kWaves = kCacheAttnWaves, kStep = kCacheAttnStep;

__device__ __forceinline__ void load_lds_word(I4 buf, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(buf) : "memory");
}
__device__ __forceinline__ I4 buffer(uint64_t at, int bytes) {
  I4 r;
  r.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)at);
  r.y = __builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu));
  r.z = __builtin_amdgcn_readfirstlane(bytes);
  r.w = kBufWord3;
  return r;
}
// Waits for the workgroup's LDS accesses, not for its loads.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }
template <typename V>
__device__ __forceinline__ V lds_read(uint32_t at) {
  return *(const __attribute__((address_space(3))) V*)(uintptr_t)at;
}

// Rows of a step in LDS: DP channels of E bytes, 16-byte chunks permuted by the row (as far as a row has them).
template <int DP, int E>
struct Ring {
  static constexpr int kPitch = DP * E, kChunks = kPitch / 16;
  static constexpr int kHalf = 16 * kPitch;                      // 16 rows of K, or of V
  static constexpr int kScales = 4 * kHalf;                      // then 256 bytes of scales for each half
  static constexpr int kBytes = kScales + (E == 1 ? 512 : 0);    // a step: K, V, scales
  static constexpr int kLoads = 2 * (2 * (kHalf / 1024) + (E == 1 ? 1 : 0));  // of a step
  static __device__ int swizzle(int row) { return kChunks == 16 ? row & 15 : (kChunks == 8 ? row & 7 : (row >> 1) & 3); }
};

typedef uint32_t U2 __attribute__((ext_vector_type(2)));
typedef uint32_t U4 __attribute__((ext_vector_type(4)));

// Two e4m3 codes as 16-bit values.
template <typename T, int WORD>
__device__ __forceinline__ uint32_t pair_of(uint32_t x) {
  if constexpr (std::is_same<T, Bf>::value)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, WORD != 0));
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.0f, WORD != 0));
}
// Two int8 codes as 16-bit values.
template <typename T>
__device__ __forceinline__ uint32_t whole_pair(int8_t x, int8_t y) {
  const float a = (float)x, b = (float)y;
  if constexpr (std::is_same<T, Bf>::value)  // (8 bits: the lower half of the f32 is zero)
    return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302);
  else
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// Codes 2 WORD and 2 WORD + 1 of four int8 codes in f16: with 128 more they are the low bits of 1024, of which 1152 are taken
// off.  (1152 times the queries' sum taken off the product instead is an operation a pair less, and 4% of an output where
// queries of 1,000 meet keys of one channel.)
template <int WORD>
__device__ __forceinline__ uint32_t offset_pair(uint32_t x) {
  typedef Mat<Hf>::V2 V2;
  const V2 more = __builtin_bit_cast(V2, __builtin_amdgcn_perm(0x64646464u, x ^ 0x80808080u, WORD ? 0x04030402 : 0x04010400));
  return __builtin_bit_cast(uint32_t, more - V2{(Hf)1152.0f, (Hf)1152.0f});
}

// The type that the second product is in: f16 for codes, whose weights then keep 11 bits also where the queries are bf16.
template <typename T, int TYPE>
using Product = typename std::conditional<Kept<TYPE>::kSize == 1, Hf, T>::type;

// Operands of 16 keys' rows for all k steps of the first product: 32 channels each.
template <typename T, int TYPE, int DP>
__device__ __forceinline__ void keys_of(uint32_t (&addr)[4], uint32_t at, typename Mat<T>::V8 (&k)[DP / 32]) {
  typedef typename Mat<T>::V8 V8;
  if constexpr (Kept<TYPE>::kSize == 2) {
#pragma unroll
    for (int t = 0; t < DP / 32; ++t) k[t] = __builtin_bit_cast(V8, lds_read<U4>(addr[t] + at));
  } else {
#pragma unroll
    for (int t = 0; t < DP / 64; ++t) {
      const U4 x = lds_read<U4>(addr[t] + at);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        U4 y;
        if constexpr (TYPE == kCacheInt8) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const uint32_t w = x[2 * h + i];
            if constexpr (std::is_same<T, Bf>::value) {
              y[2 * i] = whole_pair<T>((int8_t)w, (int8_t)(w >> 8));
              y[2 * i + 1] = whole_pair<T>((int8_t)(w >> 16), (int8_t)(w >> 24));
            } else {
              y[2 * i] = offset_pair<0>(w);
              y[2 * i + 1] = offset_pair<1>(w);
            }
          }
        } else {
          y.x = pair_of<T, 0>(x[2 * h]);
          y.y = pair_of<T, 1>(x[2 * h]);
          y.z = pair_of<T, 0>(x[2 * h + 1]);
          y.w = pair_of<T, 1>(x[2 * h + 1]);
        }
        k[2 * t + h] = __builtin_bit_cast(V8, y);
      }
    }
  }
}

// Operands of the second product: values of the lane's 8 keys (16 u + 4 quarter + i) in each of its channels.
template <typename T, int TYPE, int DP>
__device__ __forceinline__ void values_of(uint32_t (&addr)[4], uint32_t at, typename Mat<T>::V8 (&v)[DP / 16]) {
  typedef typename Mat<T>::V8 V8;
  constexpr int C = DP / 16;  // a lane's channels
  constexpr int E = Kept<TYPE>::kSize, kPitch = DP * E;
  constexpr int W = C * E / 4;  // words of a row's channels
  uint32_t raw[8][W];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const uint32_t from = addr[e % 4] + at + (e / 4) * 16 * kPitch;
    if constexpr (W == 4) {
      const U4 x = lds_read<U4>(from);
      raw[e][0] = x.x, raw[e][1] = x.y, raw[e][2] = x.z, raw[e][3] = x.w;
    } else if constexpr (W == 2) {
      const U2 x = lds_read<U2>(from);
      raw[e][0] = x.x, raw[e][1] = x.y;
    } else {
      raw[e][0] = lds_read<uint32_t>(from);
    }
  }
  U4 y[C];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (TYPE == kCacheInt8) {
#pragma unroll
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          y[4 * w + i][e] = whole_pair<T>((int8_t)(raw[2 * e][w] >> 8 * i), (int8_t)(raw[2 * e + 1][w] >> 8 * i));
      }
    } else {
      uint32_t a[C / 2], b[C / 2];  // channels by twos of either row
#pragma unroll
      for (int w = 0; w < W; ++w) {
        if constexpr (E == 2) {
          a[w] = raw[2 * e][w], b[w] = raw[2 * e + 1][w];
        } else {
          a[2 * w] = pair_of<T, 0>(raw[2 * e][w]), a[2 * w + 1] = pair_of<T, 1>(raw[2 * e][w]);
          b[2 * w] = pair_of<T, 0>(raw[2 * e + 1][w]), b[2 * w + 1] = pair_of<T, 1>(raw[2 * e + 1][w]);
        }
      }
#pragma unroll
      for (int c = 0; c < C; ++c) y[c][e] = __builtin_amdgcn_perm(b[c / 2], a[c / 2], c % 2 ? 0x07060302 : 0x05040100);
    }
  }
#pragma unroll
  for (int c = 0; c < C; ++c) v[c] = __builtin_bit_cast(V8, y[c]);
}

// The lane's operand without its values that are not finite.
template <typename T>
__device__ __forceinline__ typename Mat<T>::V8 finite_part(typename Mat<T>::V8 v) {
  U4 w = __builtin_bit_cast(U4, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t bad = ((w[i] & Mat<T>::kExp) + Mat<T>::kCarry) & 0x80008000u;
    w[i] &= ~((bad >> 15) * 0xffffu);
  }
  return __builtin_bit_cast(typename Mat<T>::V8, w);
}

// Values of a row in LDS that are not finite, of the C channels that it has at `at`: bits of those that are +infinity or NaN,
// and of those that are -infinity or NaN.
template <int TYPE, int C>
__device__ __forceinline__ void not_finite_bits(uint32_t at, uint32_t* up, uint32_t* down) {
  *up = *down = 0;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    if constexpr (TYPE == kCacheE4m3) {
      const uint32_t x = lds_read<uint8_t>(at + i);
      if ((x & 0x7f) == 0x7f) *up |= 1u << i, *down |= 1u << i;
    } else {
      constexpr uint32_t e = TYPE == kCacheBf16 ? 0x7f80 : 0x7c00;
      const uint32_t x = lds_read<uint16_t>(at + 2 * i);
      const bool bad = (x & e) == e, nan = bad && (x & 0x7fff) != e;
      if (nan || (bad && !(x & 0x8000))) *up |= 1u << i;
      if (nan || (bad && (x & 0x8000))) *down |= 1u << i;
    }
  }
}

// The lowest n of 32 bits.
__device__ __forceinline__ uint32_t low_bits(int n) { return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1); }

// The least unit of weights times value scales (a weight of 2^-8 times the least scale has it).
constexpr float kLeastUnit = 0x1p-120f;
// 1 over a power of two.
__device__ __forceinline__ float over_power(float x) { return __uint_as_float(0x7f000000u - __float_as_uint(x)); }
// The power of two from x on, within 2^-126 and 2^126.  A result is kept divided by that of its sum of weights, so that it is no
// larger than the values that it is a mean of.
__device__ __forceinline__ float power_from(float x) {
  return __uint_as_float(min(max((__float_as_uint(x) + 0x7fffffu) & 0x7f800000u, 0x00800000u), 0x7e800000u));
}
// Results of the same row, each with its reference exponent and sum of weights, as one.
template <int N>
struct Joined {
  float weight[N];  // of each: 0 of one that saw nothing
  float m = kNever, sum = 0.0f;
  __device__ __forceinline__ Joined(const float2 (&x)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) m = fmaxf(m, x[i].x);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float f = x[i].x == kNever && x[i].y == 0.0f ? 0.0f : exp2_fast(x[i].x - m);
      sum += x[i].y * f;
      weight[i] = f * power_from(x[i].y);
    }
    const float over = over_power(power_from(sum));
#pragma unroll
    for (int i = 0; i < N; ++i) weight[i] *= over;
  }
  // What makes the sum of weighted results the row's (zero of a row that sees nothing).
  __device__ __forceinline__ float last() const {
    return sum > 0.0f || sum != sum ? 1.0f / (sum * over_power(power_from(sum))) : 0.0f;
  }
};

// What an item needs of its sequence's keys: those before `end`, in rounds.
struct Span {
  int context;  // tokens before the new ones (negative: the first new tokens are none)
  int end, rounds;
};
// round: keys of one.
__device__ __forceinline__ Span span_of(const CacheAttnArgs& a, const CacheTile& t, int round) {
  Span s;
  const int length = a.c.lengths[t.seq];
  s.context = (length > 0 ? length : 0) - t.n;
  int end = s.context + t.n;
  if (!a.tree) end = s.context + (t.at + t.count - 1) / a.group + 1;
  const int cap = a.c.table_pages << a.c.shift;
  end = end < cap ? end : cap;
  s.end = end < 0 ? 0 : end;
  s.rounds = s.end > 0 ? (s.end - 1) / round + 1 : 1;
  return s;
}

template <int CTRL, int MASK>
__device__ __forceinline__ int dpp_add(int x) {
  return x + __builtin_amdgcn_update_dpp(0, x, CTRL, MASK, 0xf, false);
}
// Inclusive sums over a wave's lanes.
__device__ __forceinline__ int wave_scan(int x) {
  x = dpp_add<0x111, 0xf>(x);  // from the lane 1, 2, 4 and 8 before, within 16
  x = dpp_add<0x112, 0xf>(x);
  x = dpp_add<0x114, 0xf>(x);
  x = dpp_add<0x118, 0xf>(x);
  x = dpp_add<0x142, 0xa>(x);  // the row before's last lane, then that of the first two
  x = dpp_add<0x143, 0xc>(x);
  return x;
}

// Where the workgroup's share of all rounds begins: the item that holds round `at` and the rounds before that
// item.  Units are (item, kv head), the heads of an item side by side.
struct Start {
  int total;           // rounds of all units
  int item, before;    // rounds of the units before the item
};
__device__ __forceinline__ Start start_of(const CacheAttnArgs& a, int w, int* lds, int* share, int round) {
  const int t = (int)threadIdx.x, per = (a.c.n_tiles + 64 * kWaves - 1) / (64 * kWaves);
  int mine = 0;
  for (int i = t * per; i < min((t + 1) * per, a.c.n_tiles); ++i) mine += span_of(a, a.c.tiles[i], round).rounds;
  int sum = wave_scan(mine);
  if ((t & 63) == 63) lds[t >> 6] = sum;
  __syncthreads();
  int total = 0;
#pragma unroll
  for (int v = 0; v < kWaves; ++v) {
    if (v < (t >> 6)) sum += lds[v];
    total += lds[v];
  }
  Start s;
  s.total = total * a.c.kv_heads;
  *share = (int)(((int64_t)s.total + gridDim.x - 1) / gridDim.x);
  const int64_t at = (int64_t)w * *share;
  int before = sum - mine;
  if (at >= (int64_t)before * a.c.kv_heads && at < (int64_t)sum * a.c.kv_heads) {
    int i = t * per;
    for (;; ++i) {
      const int r = span_of(a, a.c.tiles[i], round).rounds;
      if (at < (int64_t)(before + r) * a.c.kv_heads) break;
      before += r;
    }
    lds[kWaves] = i;
    lds[kWaves + 1] = before * a.c.kv_heads;
  }
  __syncthreads();
  s.item = __builtin_amdgcn_readfirstlane(lds[kWaves]);
  s.before = __builtin_amdgcn_readfirstlane(lds[kWaves + 1]);
  return s;
}

// T: the queries' type; NR: tiles of 16 packed rows of a wave.  SHARE waves read the same steps, each for rows of its own,
// from a ring of three stages that they fill together, with one barrier a step; the others take other steps.
// WHOLE: a workgroup takes one unit, all of its rounds; otherwise an equal share of all rounds, of
// which the first and last units may be cut: their parts go to a slot each and are joined by a second launch.
// The first loads of a share's next unit are in flight while the waves add their results of one up.
template <typename T, int TYPE, int DP, int NR, int SHARE, bool WHOLE>
__global__ __launch_bounds__(64 * kWaves, Kept<TYPE>::kSize == 2 && DP == 128 ? 1 : 2) void sfe_cache_attn_kernel(CacheAttnArgs a, int64_t first) {
  typedef Ring<DP, Kept<TYPE>::kSize> R;
  typedef Product<T, TYPE> W;
  typedef Mat<W> M;
  typedef typename M::V8 V8;
  typedef typename M::V2 V2;
  typedef typename Mat<T>::V2 O2;
  constexpr bool kCoded = Kept<TYPE>::kSize == 1;
  constexpr bool kFar = kCoded && std::is_same<T, Bf>::value;     // products of queries and codes may pass f32 where scores do not
  constexpr bool kSplit = kCoded && std::is_same<T, Hf>::value;  // a weight is two 16-bit numbers
  constexpr bool kNotFinite = TYPE != kCacheInt8;  // the cache's type has infinities or NaN
  // Weights of codes are at most 1, and fit f16 by a unit of their own.  Those over bf16 are at most 2^-16, so that a wave's sums over
  // its keys do not pass the largest value where their mean does not (2^16 keys of 3e38).
  constexpr float kRise = kCoded ? 0.0f : (TYPE == kCacheBf16 ? -16.0f : M::kRise);
  constexpr float kBelow = kCoded ? -8.0f : (TYPE == kCacheBf16 ? -24.0f : M::kBelow);
  constexpr int E = Kept<TYPE>::kSize, C = DP / 16;
  constexpr int kRowF = DP + 4;  // floats of a result's row in LDS (4 of padding)
  constexpr int kGroups = kWaves / SHARE, kRound = kGroups * kStep;  // waves by steps; keys of a round
  constexpr int kStages = SHARE > 1 ? 3 : 2, kStage = kGroups * R::kBytes;
  // the waves' results go behind the first stage
  constexpr int kResults = 4 * (kWaves * 16 * kRowF + 2 * kWaves * 16), kRest = (kStages - 1) * kStage;
  __shared__ __align__(1024) char lds[kStage + (kRest > kResults ? kRest : kResults)];
  __shared__ int lds_start[kWaves + 2];
  const CacheArgs& c = a.c;
  const int t = (int)threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), quarter = lane >> 4;
  const int group = wave / SHARE, member = wave % SHARE;
  const uint32_t base = lds_address(lds) + group * R::kBytes;

  // ---- addresses that stay
  uint32_t k_addr[4], v_addr[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    k_addr[i] = base + (lane & 15) * R::kPitch + 16 * (((4 * i + quarter) % R::kChunks) ^ R::swizzle(lane & 15));
    const int row = 4 * quarter + i, byte = C * E * (lane & 15);
    v_addr[i] = base + 2 * R::kHalf + row * R::kPitch + 16 * ((byte / 16) ^ R::swizzle(row)) + byte % 16;
  }
  // a lane's chunk of 32 rows in each load, its place in the record's rows or none
  constexpr int kRowLoads = R::kHalf / 1024;
  uint32_t from[2 * kRowLoads];
#pragma unroll
  for (int i = 0; i < 2 * kRowLoads; ++i) {
    const int row = (i * 64 + lane) / R::kChunks, chunk = ((i * 64 + lane) % R::kChunks) ^ R::swizzle(row & 15);
    from[i] = 16 * chunk < c.dim * E ? (uint32_t)(row * c.dim * E + 16 * chunk) : kOutside;
  }
  const int page_mask = (1 << c.shift) - 1;
  const uint32_t part = (uint32_t)(c.dim * E) << c.shift;  // bytes of a record's K, and V

  // ---- the workgroup's share
  int at = 0, stop = 1;  // rounds (WHOLE: one unit)
  int before = 0, share = 0, w = 0;
  // a unit, and the rounds of it that are the workgroup's
  struct Unit {
    int64_t first;
    int seq, n, at, count, total;
    int item, kvh, rounds, end, context, r0, r1;
  } u;
  auto unit_of = [&](int item, int kvh) {  // (but its rounds)
    typedef const __attribute__((address_space(4))) CacheTile* Tiles;
    const Tiles p = (Tiles)(uintptr_t)c.tiles + __builtin_amdgcn_readfirstlane(item);
    CacheTile tile;
    tile.first = p->first, tile.seq = p->seq, tile.n = p->n, tile.at = p->at, tile.count = p->count;
    const Span s = span_of(a, tile, kRound);
    Unit x;
    x.first = tile.first, x.seq = tile.seq, x.n = tile.n, x.at = tile.at, x.count = tile.count, x.total = tile.n * a.group;
    x.item = item, x.kvh = kvh;
    x.rounds = __builtin_amdgcn_readfirstlane(s.rounds), x.end = __builtin_amdgcn_readfirstlane(s.end);
    x.context = __builtin_amdgcn_readfirstlane(s.context);
    x.r0 = 0, x.r1 = x.rounds;
    return x;
  };
  if (WHOLE) {
    const int64_t unit = first + blockIdx.x;
    const int item = (int)(unit / c.kv_heads);
    u = unit_of(item, (int)(unit - (int64_t)item * c.kv_heads));
  } else {
    // consecutive workgroups go to the 8 XCDs in turn: each has a contiguous part of the shares
    w = (int)(blockIdx.x % 8) * (int)(gridDim.x / 8) + (int)(blockIdx.x / 8);
    const Start s = start_of(a, w, lds_start, &share, kRound);
    if ((int64_t)w * share >= s.total) return;
    at = w * share;
    stop = at + share < s.total ? at + share : s.total;
    before = s.before;
    u = unit_of(s.item, 0);
    u.kvh = (int)((unsigned)(at - before) / (unsigned)u.rounds);
    u.r0 = at - before - u.kvh * u.rounds;
    u.r1 = u.rounds - u.r0 < stop - at ? u.rounds : u.r0 + (stop - at);
  }

  // the pages of a step's halves (-1: none)
  auto look_up = [&](const Unit& x, int r, int (&page)[2]) {
    typedef const __attribute__((address_space(4))) int32_t* Pages;
    const Pages pages = (Pages)(uintptr_t)c.table + (int64_t)x.seq * c.table_row;
    const int key = __builtin_amdgcn_readfirstlane((r * kGroups + group) * kStep);
    page[0] = page[1] = -1;
    if (r < x.r1 && key < x.end) page[0] = pages[key >> c.shift];
    if (c.shift == 4 && r < x.r1 && key + 16 < x.end) page[1] = pages[(key + 16) >> c.shift];
  };
  // loads of 16 or 32 rows of a page that begin with token `key`, n of which there are, into a stage's half h and on
  auto load_rows = [&](const Unit& x, int key, int n, int page, int stage, int h, auto halves_) {
    constexpr int kHalves = decltype(halves_)::value;
    const uint64_t record = (uint64_t)(uintptr_t)c.data + (uint64_t)((int64_t)page * c.kv_heads + x.kvh) * (uint64_t)c.record;
    const int slot = key & page_mask, bytes = n * c.dim * E;
    const I4 kb = buffer(record + (uint32_t)(slot * c.dim * E), bytes);
    const I4 vb = buffer(record + part + (uint32_t)(slot * c.dim * E), bytes);
    const uint32_t to = __builtin_amdgcn_readfirstlane(base + stage * kStage + h * R::kHalf);
    // (of waves that share a step: two take a half of K and of V each, four half a half)
#pragma unroll
    for (int i = 0; i < kHalves * kRowLoads; ++i)
      if (SHARE == 1 || (SHARE == 2 ? member == 0 : member == (h * kRowLoads + i) / kRowLoads)) load_lds(kb, from[i], to + i * 1024);
#pragma unroll
    for (int i = 0; i < kHalves * kRowLoads; ++i)
      if (SHARE == 1 || (SHARE == 2 ? member == 1 : member == 2 + (h * kRowLoads + i) / kRowLoads))
        load_lds(vb, from[i], to + 2 * R::kHalf + i * 1024);
    if (kCoded) {
      // 16 scales of K, 16 of V, and the same of the second half
      const I4 sb = buffer(record + 2 * part + 4 * slot, n ? 4 * (page_mask + 1) + 4 * n : 0);
#pragma unroll
      for (int i = 0; i < kHalves; ++i) {
        if (SHARE > 1 && member != h + i) continue;
        const int l = (lane & 15) + 16 * i;
        const uint32_t off = lane < 32 && l < n ? (uint32_t)(4 * l + (lane < 16 ? 0 : 4 * (page_mask + 1))) : kOutside;
        load_lds_word(sb, off, __builtin_amdgcn_readfirstlane(base + stage * kStage + R::kScales + (h + i) * 256));
      }
    }
  };
  // a step's loads; returns the keys of either half that there are
  auto load_step = [&](const Unit& x, int r, int stage, const int (&page)[2]) {
    const int key = __builtin_amdgcn_readfirstlane((r * kGroups + group) * kStep);
    if (c.shift > 4) {
      const bool ok = page[0] >= 0 && page[0] < c.pages;
      const int left = x.end - key, n = ok ? (left < 32 ? left : 32) : 0;
      load_rows(x, key, n, ok ? page[0] : 0, stage, 0, std::integral_constant<int, 2>());
      return n <= 16 ? n : 16 | (n - 16) << 8;
    }
    int there = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const bool ok = page[h] >= 0 && page[h] < c.pages;
      const int left = x.end - key - 16 * h, n = ok ? (left < 16 ? left : 16) : 0;
      load_rows(x, key + 16 * h, n, ok ? page[h] : 0, stage, h, std::integral_constant<int, 1>());
      there |= n << (8 * h);
    }
    return there;
  };
  S8 q[NR][DP / 32];
  uint64_t bits[NR];
  int me[NR];  // the row's own place
  auto load_queries = [&](const Unit& x) {
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      const int row = x.at + 16 * (NR * member + n) + (lane & 15), rc = row < x.total ? row : x.total - 1;
      const int token = (int)((unsigned)rc / (unsigned)a.group), head = x.kvh * a.group + rc - token * a.group;
      const char* p = a.q.data + (x.first + token) * a.q.row + head * a.q.head;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) {
        const int channel = E == 2 ? 32 * i + 8 * quarter : 64 * (i / 2) + 16 * quarter + 8 * (i % 2);
        S8 v = {0, 0, 0, 0, 0, 0, 0, 0};
        if (channel < c.dim) v = *reinterpret_cast<const S8*>(p + 2 * channel);
        q[n][i] = v;
      }
      me[n] = x.context + token;
      bits[n] = a.tree ? a.tree[x.first + token] : 0;
    }
  };
  int page[2], page_next[2], there, there_next = 0, there_after = 0;
  look_up(u, u.r0, page);
  look_up(u, u.r0 + 1, page_next);
  there = load_step(u, u.r0, 0, page);
  load_queries(u);

  for (;;) {
    const int context = u.context, r0 = u.r0, r1 = u.r1;
    // the queries and the first step, waited for here: a wait for the queries within the loop would be one for its loads into LDS
#pragma unroll
    for (int n = 0; n < NR; ++n) {
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) asm volatile("" : "+v"(q[n][i]));
      if (u.n < 64) bits[n] &= (1ull << u.n) - 1;
      asm volatile("" : "+v"(bits[n]));
    }
    if (r0 + 1 < r1) {
      there_next = load_step(u, r0 + 1, 1, page_next);
      look_up(u, r0 + 2, page);
    }
    // rows of queries past 2^73 are taken down to it; the power of two is their scores' unit
    float unit[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      unit[n] = 1.0f;
      if constexpr (kFar) {
        uint32_t top = 0;  // (exponents of two queries at a time, those of infinities and NaN left out)
#pragma unroll
        for (int i = 0; i < DP / 32; ++i) {
          const U4 w = __builtin_bit_cast(U4, q[n][i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint32_t lo = w[j] & 0x7f80u, hi = (w[j] >> 16) & 0x7f80u;
            top = max(top, max(lo == 0x7f80u ? 0u : lo, hi == 0x7f80u ? 0u : hi));
          }
        }
        if (__any(top > 200u << 7)) {
          top = max(top, (uint32_t)__shfl_xor((int)top, 16));
          top = max(top, (uint32_t)__shfl_xor((int)top, 32));
          const int down = max((int)(top >> 7) - 200, 0);
          unit[n] = __uint_as_float((uint32_t)(127 + down) << 23);
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) {
            U4 w = __builtin_bit_cast(U4, q[n][i]);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const F2 y = {__builtin_amdgcn_ldexpf(__uint_as_float(w[j] << 16), -down),
                            __builtin_amdgcn_ldexpf(__uint_as_float(w[j] & 0xffff0000u), -down)};
              w[j] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, Mat<Bf>::V2));
            }
            q[n][i] = __builtin_bit_cast(S8, w);
          }
        }
      }
    }

    F4 o[NR][C];
    float m[NR], l[NR], unit_w[NR];  // unit_w: what weights times value scales are kept in (a power of two)
    uint32_t ups[NR], downs[NR];  // results that get +infinity and -infinity in the end, bits C j + i of o[i][j]
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      ups[n] = downs[n] = 0;
      m[n] = kNever, l[n] = 0.0f, unit_w[n] = kLeastUnit;
#pragma unroll
      for (int i = 0; i < C; ++i) o[n][i] = F4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    uint32_t in = 0;  // the step's stage
    for (int r = r0; r < r1; ++r) {
      // the step's loads of this wave, but not those of the next
      constexpr int kMine = 4 * kRowLoads / SHARE;
      if (r + 1 >= r1)
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      else if (SHARE == 1)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(R::kLoads) : "memory");
      else if (kCoded && member < 2)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kMine + 1) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(kMine) : "memory");
      if (SHARE > 1) {
        // everyone's loads of the step are there, and nobody reads the one before, whose stage takes the step after the next
        lds_barrier();
        if (r + 2 < r1) {
          there_after = load_step(u, r + 2, in == 0 ? 2 : (in == kStage ? 0 : 1), page);
          look_up(u, r + 3, page);
        }
      }
      const int key = (r * kGroups + group) * kStep, now = there;
      // ---- scores
      F4 s[NR][2], ks[2], vs[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        typename Mat<T>::V8 k[DP / 32];
        keys_of<T, TYPE, DP>(k_addr, in + u * R::kHalf, k);
        if (kCoded) {
          ks[u] = lds_read<F4>(base + in + R::kScales + u * 256 + 16 * quarter) * a.scale_log2;
          vs[u] = lds_read<F4>(base + in + R::kScales + u * 256 + 64 + 16 * quarter);
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          s[n][u] = F4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < DP / 32; ++i) s[n][u] = Mat<T>::m16(k[i], __builtin_bit_cast(typename Mat<T>::V8, q[n][i]), s[n][u]);
        }
      }
      V8 v[C];
      values_of<W, TYPE, DP>(v_addr, in, v);
      float top_value = 0.0f;  // (of the lane's keys)
      if (kCoded)
        top_value = fmaxf(fmaxf(fmaxf(vs[0][0], vs[0][1]), fmaxf(vs[0][2], vs[0][3])),
                          fmaxf(fmaxf(vs[1][0], vs[1][1]), fmaxf(vs[1][2], vs[1][3])));
      // keys that some rows do not see
      const bool uneven = key + kStep > context || now != 0x1010;
      uint32_t see[NR];
#pragma unroll
      for (int n = 0; n < NR; ++n) see[n] = ~0u;
      if (uneven) {
        const uint32_t there_bits = low_bits(now & 0xff) | low_bits(now >> 8) << 16;
#pragma unroll
        for (int n = 0; n < NR; ++n) {
          see[n] = low_bits(a.tree ? context - key : me[n] + 1 - key);
          if (a.tree) {
            const int d = context - key;
            if (d >= 0) see[n] |= d < 32 ? (uint32_t)(bits[n] << d) : 0;
            else see[n] |= d > -64 ? (uint32_t)(bits[n] >> -d) : 0;
          }
          see[n] &= there_bits;
          if (me[n] < 0) see[n] = 0;
        }
        if constexpr (kNotFinite) {
          // values that are not finite are kept from the rows that do not see them as 0 * inf: they are taken out, and
          // remembered for the rows that do
          uint32_t bad = 0;
#pragma unroll
          for (int i = 0; i < C; ++i) {
            U4 x = __builtin_bit_cast(U4, v[i]);
            asm volatile("" : "+v"(x));  // (or it would be looked at in every step)
            bad |= nonfinite<W>(__builtin_bit_cast(V8, x));
          }
          if (__any(bad != 0)) {
#pragma unroll 1
            for (int row = 0; row < kStep; ++row) {
              uint32_t up = 0, down = 0;
#pragma unroll 1
              for (int j = 0; j < 4; ++j) {
                const int byte = C * E * (4 * quarter + j);
                uint32_t u, d;
                not_finite_bits<TYPE, C>(base + in + 2 * R::kHalf + row * R::kPitch + 16 * ((byte / 16) ^ R::swizzle(row & 15)) + byte % 16, &u, &d);
                up |= u << (C * j), down |= d << (C * j);
              }
#pragma unroll
              for (int n = 0; n < NR; ++n) {
                const uint32_t mine = 0u - (see[n] >> row & 1);
                ups[n] |= up & mine, downs[n] |= down & mine;
              }
            }
#pragma unroll
            for (int i = 0; i < C; ++i) v[i] = finite_part<W>(v[i]);
          }
        }
#pragma unroll
        for (int n = 0; n < NR; ++n) see[n] >>= 4 * quarter;  // the lane's keys are 16 u + 4 quarter + i
      }
#pragma unroll
      for (int n = 0; n < NR; ++n) {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) s[n][u][i] *= kCoded ? ks[u][i] : a.scale_log2;
        if (uneven)
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[n][u][i] = (see[n] >> (16 * u + i)) & 1 ? s[n][u][i] : -INFINITY;
        float top = s[n][0][0];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int i = 0; i < 4; ++i) top = fmaxf(top, s[n][u][i]);
        if (kFar) top *= unit[n];
        if (__any(top > m[n] + kRise)) {
          top = max_halves(fmaxf(top, __shfl_xor(top, 16)));
          // (whole numbers where weights have a unit: it goes down by powers of two)
          const float nm = fmaxf(m[n], kCoded ? ceilf(top) - kBelow : top - kBelow);
          float f = exp2_fast(m[n] - nm);
          m[n] = nm;
          l[n] *= f;
          if (kCoded) {
            const float down = unit_w[n] * f;
            unit_w[n] = fmaxf(down, kLeastUnit);
            f = down * over_power(unit_w[n]);  // (1 but at the least unit)
          }
          if (!kCoded || __any(f != 1.0f))
#pragma unroll
            for (int i = 0; i < C; ++i) o[n][i] *= f;
        }
        float x[8];  // (the unit is a power of two: nothing is lost in the product)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = s[n][e / 4][e % 4];
          x[e] = exp2_fast(kFar ? __builtin_fmaf(y, unit[n], -m[n]) : rounded_less(y, m[n]));
        }
        l[n] += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        if (kCoded) {
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= vs[e / 4][e % 4];
          // weights are at most 1: up to this scale none times it passes 2^15 units
          if (__any(top_value > unit_w[n] * 0x1p15f)) {
            float most = 0.0f;  // (of seen keys: the others' weights are zero, or not numbers times a scale that is not finite)
#pragma unroll
            for (int e = 0; e < 8; ++e) most = fmaxf(most, x[e]);
            most = max_halves(fmaxf(most, __shfl_xor(most, 16)));
            if (__any(most > unit_w[n] * 0x1p7f)) {
              // the largest becomes 2^4 to 2^5 units, so that ordinary scales do not come here again
              const float to = most > unit_w[n] * 0x1p7f ? __uint_as_float((min(__float_as_uint(most) >> 23, 250u) - 4) << 23) : unit_w[n];
              const float f = unit_w[n] * over_power(to);
              unit_w[n] = to;
#pragma unroll
              for (int i = 0; i < C; ++i) o[n][i] *= f;
            }
          }
          const float relative = over_power(unit_w[n]);
#pragma unroll
          for (int e = 0; e < 8; ++e) x[e] *= relative;
          if (uneven)  // (0 times a scale that is not finite)
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (see[n] >> (16 * (e / 4) + e % 4)) & 1 ? x[e] : 0.0f;
        }
        V8 p, rest;
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          const F2 y = {x[e], x[e + 1]};
          const V2 z = __builtin_convertvector(y, V2);
          p[e] = z.x, p[e + 1] = z.y;
          if (kSplit) {
            const F2 d = {x[e] - (float)z.x, x[e + 1] - (float)z.y};
            const V2 f = __builtin_convertvector(d, V2);
            rest[e] = f.x, rest[e + 1] = f.y;
          }
        }
#pragma unroll
        for (int i = 0; i < C; ++i) o[n][i] = M::m16(v[i], p, o[n][i]);
        if (kSplit)
#pragma unroll
          for (int i = 0; i < C; ++i) o[n][i] = M::m16(v[i], rest, o[n][i]);
      }
      there = there_next;
      if (SHARE > 1) {
        there_next = there_after;
        in = in == 2 * kStage ? 0 : in + kStage;
      } else {
        // the buffer just read takes the step after the next
        if (r + 2 < r1) {
          asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
          there_next = load_step(u, r + 2, in ? 1 : 0, page);
          look_up(u, r + 3, page);
        }
        in ^= kStage;
      }
    }
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      l[n] += __shfl_xor(l[n], 16);
      l[n] = sum_halves(l[n]);
      const float over = over_power(power_from(l[n]));
#pragma unroll
      for (int i = 0; i < C; ++i) {
        o[n][i] *= over;
        if (kCoded) o[n][i] *= unit_w[n];
      }
    }
    if constexpr (kNotFinite)
#pragma unroll
      for (int n = 0; n < NR; ++n)
        if (__any((ups[n] | downs[n]) != 0))
#pragma unroll
          for (int i = 0; i < C; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              if (ups[n] >> (C * j + i) & 1) o[n][i][j] += INFINITY;
              if (downs[n] >> (C * j + i) & 1) o[n][i][j] -= INFINITY;
            }
    // ---- the next unit's first loads
    const Unit done = u;
    at += r1 - r0;
    const bool more = !WHOLE && at < stop;
    if (more) {
      if (SHARE > 1) lds_barrier();  // (a member may still read the first stage)
      if (done.kvh == c.kv_heads - 1) {
        before += done.rounds * c.kv_heads;
        u = unit_of(done.item + 1, 0);
      } else {
        u.kvh = done.kvh + 1;
      }
      u.r0 = 0;
      u.r1 = u.rounds < stop - at ? u.rounds : stop - at;
      look_up(u, 0, page);
      look_up(u, 1, page_next);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      there = load_step(u, 0, 0, page);
      load_queries(u);
    }
    // ---- the waves' results, added up through LDS, a tile of 16 rows at a time
    const bool cut = !WHOLE && (r0 > 0 || r1 < done.rounds);
    const int slot = 2 * w + (r1 < done.rounds);
    float* ow = reinterpret_cast<float*>(lds + kStage);                 // [wave][16][kRowF]
    float2* ml = reinterpret_cast<float2*>(ow + kWaves * 16 * kRowF);   // [wave][16]
#pragma unroll
    for (int n = 0; n < NR; ++n) {
      if (16 * n >= done.count) break;
      lds_barrier();
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < C; i += 4)
          *reinterpret_cast<F4*>(ow + (wave * 16 + (lane & 15)) * kRowF + C * (4 * quarter + j) + i) =
              F4{o[n][i][j], o[n][i + 1][j], o[n][i + 2][j], o[n][i + 3][j]};
      if (quarter == 0) ml[wave * 16 + lane] = make_float2(m[n], l[n]);
      lds_barrier();
      for (int e = t; e < SHARE * 16 * (DP / 4); e += 64 * kWaves) {
        const int of = e / (16 * (DP / 4)), row16 = e / (DP / 4) % 16, d = 4 * (e % (DP / 4));  // (of: the member)
        const int row = 16 * (NR * of + n) + row16;
        if (row >= done.count || d >= c.dim) continue;
        float2 each[kGroups];
#pragma unroll
        for (int v = 0; v < kGroups; ++v) each[v] = ml[(v * SHARE + of) * 16 + row16];
        const Joined<kGroups> joined(each);
        F4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int v = 0; v < kGroups; ++v)
          acc += *reinterpret_cast<const F4*>(ow + ((v * SHARE + of) * 16 + row16) * kRowF + d) * joined.weight[v];
        const int rr = done.at + row;
        if (cut) {
          const int64_t place = (int64_t)slot * (16 * NR * SHARE) + row;
          *reinterpret_cast<F4*>(a.part_o + place * DP + d) = acc;
          if (d == 0) a.part_ml[place] = make_float2(joined.m, joined.sum);
        } else {
          const float inv = joined.last();
          const int token = (int)((unsigned)rr / (unsigned)a.group);
          char* p = const_cast<char*>(a.o.data) + (done.first + token) * a.o.row + (int64_t)(done.kvh * a.group + rr - token * a.group) * a.o.head;
          const F2 x = {acc.x * inv, acc.y * inv}, y = {acc.z * inv, acc.w * inv};
          const O2 f = __builtin_convertvector(x, O2), g = __builtin_convertvector(y, O2);
          *reinterpret_cast<uint2*>(p + 2 * d) = make_uint2(__builtin_bit_cast(uint32_t, f), __builtin_bit_cast(uint32_t, g));
        }
      }
    }
    if (WHOLE) return;
    if (t == 0 && r0 == 0) {
      // what the join needs: the workgroup of the unit's first part, and how many parts
      const int last = (at - (r1 - r0) + done.rounds - 1) / share;
      a.units[(int64_t)done.item * c.kv_heads + done.kvh] = make_int2(w, cut ? last - w + 1 : 0);
    }
    if (!more) return;
    lds_barrier();  // (the second stage is the loads' again)
  }
}

// Parts of units that were cut, added up: a workgroup takes 4 rows of a unit, each of its teams every
// kTeams-th part with a reference exponent of its own.
template <typename T, int DP, int THREADS>
__global__ __launch_bounds__(THREADS) void sfe_cache_attn_join_kernel(CacheAttnArgs a, int64_t first, int groups) {
  typedef typename Mat<T>::V2 V2;
  constexpr int kLanes = DP / 4, kTeams = THREADS / (4 * kLanes);  // lanes of a row
  __shared__ F4 sums[kTeams][4 * kLanes];
  __shared__ float2 ml[kTeams][4];
  const int64_t block = first + blockIdx.x, unit = block / groups;
  const int item = (int)(unit / a.c.kv_heads), kvh = (int)(unit - (int64_t)item * a.c.kv_heads);
  const int2 u = a.units[unit];
  const CacheTile tile = a.c.tiles[item];
  if (u.y == 0) return;
  const int t = (int)threadIdx.x, team = t / (4 * kLanes), in = t % (4 * kLanes), row4 = in / kLanes, d = 4 * (in % kLanes);
  const int row = 4 * (int)(block - unit * groups) + row4;
  const bool there = row < tile.count && d < a.c.dim;
  // part p of the unit is its workgroup's last, but for the unit's last part
  auto place = [&](int p) { return (int64_t)(2 * (u.x + p) + (p + 1 < u.y)) * (16 * a.tiles) + row; };
  F4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
  float sum = 0.0f, m = kNever;
  if (there)
#pragma unroll 4
    for (int p = team; p < u.y; p += kTeams) {
      const float2 x = a.part_ml[place(p)];
      const F4 v = *reinterpret_cast<const F4*>(a.part_o + place(p) * DP + d);
      const float2 both[2] = {make_float2(m, sum), x};
      const Joined<2> joined(both);
      m = joined.m;
      sum = joined.sum;
      acc = acc * joined.weight[0] + v * joined.weight[1];
    }
  sums[team][in] = acc;
  if (d == 0) ml[team][row4] = make_float2(m, sum);
  __syncthreads();
  if (team > 0 || !there) return;
  float2 each[kTeams];
#pragma unroll
  for (int v = 0; v < kTeams; ++v) each[v] = ml[v][row4];
  const Joined<kTeams> joined(each);
  acc = F4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int v = 0; v < kTeams; ++v) acc += sums[v][in] * joined.weight[v];
  const float inv = joined.last();
  const int rr = tile.at + row, token = (int)((unsigned)rr / (unsigned)a.group);
  char* p = const_cast<char*>(a.o.data) + (tile.first + token) * a.o.row + (int64_t)(kvh * a.group + rr - token * a.group) * a.o.head;
  const F2 x = {acc.x * inv, acc.y * inv}, y = {acc.z * inv, acc.w * inv};
  const V2 f = __builtin_convertvector(x, V2), g = __builtin_convertvector(y, V2);
  *reinterpret_cast<uint2*>(p + 2 * d) = make_uint2(__builtin_bit_cast(uint32_t, f), __builtin_bit_cast(uint32_t, g));
}

template <typename T, int TYPE, int DP, int NR, int SHARE>
hipError_t run_rows(const CacheAttnArgs& a, hipStream_t stream) {
  const int64_t units = (int64_t)a.c.n_tiles * a.c.kv_heads;
  if (a.whole)
    return for_launches(units, 64 * kWaves, [&](int64_t first, unsigned blocks) {
      sfe_cache_attn_kernel<T, TYPE, DP, NR, SHARE, true><<<dim3(blocks), dim3(64 * kWaves), 0, stream>>>(a, first);
      return hipGetLastError();
    });
  sfe_cache_attn_kernel<T, TYPE, DP, NR, SHARE, false><<<dim3((unsigned)a.shares), dim3(64 * kWaves), 0, stream>>>(a, 0);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int groups = (a.rows + 3) / 4;
  // (a unit has about shares / units + 1 parts: few of them take half the waves.  256 units of 64 rows: 11.5 us with 512
  // threads, 9.0 with 256; 16 units in 34 parts: 4.7 and 5.0)
  const bool few = 4 * units >= a.shares;
  return for_launches(units * groups, 512, [&](int64_t first, unsigned blocks) {
    if (few) sfe_cache_attn_join_kernel<T, DP, 256><<<dim3(blocks), dim3(256), 0, stream>>>(a, first, groups);
    else sfe_cache_attn_join_kernel<T, DP, 512><<<dim3(blocks), dim3(512), 0, stream>>>(a, first, groups);
    return hipGetLastError();
  });
}

template <typename T, int TYPE, int DP>
hipError_t run_tiles(const CacheAttnArgs& a, hipStream_t stream) {
  switch (a.tiles) {
    case 1: return run_rows<T, TYPE, DP, 1, 1>(a, stream);
    case 2: return run_rows<T, TYPE, DP, 2, 1>(a, stream);
    case 4: return run_rows<T, TYPE, DP, 2, 2>(a, stream);
    default: return run_rows<T, TYPE, DP, 2, 4>(a, stream);
  }
}

template <typename T, int TYPE>
hipError_t run(const CacheAttnArgs& a, hipStream_t stream) {
  return a.c.dim <= 64 ? run_tiles<T, TYPE, 64>(a, stream) : run_tiles<T, TYPE, 128>(a, stream);
}

}  // namespace

hipError_t launch_cache_attn(const CacheAttnArgs& a, int type, int dtype, hipStream_t stream) {
  switch (type) {
    case kCacheBf16: return run<Bf, kCacheBf16>(a, stream);
    case kCacheF16: return run<Hf, kCacheF16>(a, stream);
    case kCacheE4m3: return dtype == kOpBf16 ? run<Bf, kCacheE4m3>(a, stream) : run<Hf, kCacheE4m3>(a, stream);
    default: return dtype == kOpBf16 ? run<Bf, kCacheInt8>(a, stream) : run<Hf, kCacheInt8>(a, stream);
  }
}

}  // namespace sfe
