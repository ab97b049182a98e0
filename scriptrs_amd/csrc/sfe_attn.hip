// Attention over packed sequences with grouped heads.
//
// For query i of a sequence of Lq queries and Lk keys, head h reading kv head
// h / group:  o_i = sum_j softmax_j(scale q_i . k_j) v_j over the keys j that i
// sees: i + Lk - Lq - left <= j <= i + Lk - Lq + right and not masked; zero if
// there is none.  One pass over the keys with a running reference exponent and
// sum: with x_j = scale log2(e) q_i . k_j and any reference m, the weights are
// 2^(x_j - m) / sum 2^(x_j - m).  m follows the running maximum only when that
// has risen by 8 since it last did, so most steps rescale nothing.  In f16 weights
// go from 2^7 of a new maximum up to 2^15 (it holds 65504), so that those down to 2^-17 of the
// largest keep all their bits; in bf16, which has the range anyway, from 2^-8 up to 1, so
// that no value that a mean of values can have is passed on the way to it.  Scores, m,
// sums and outputs are f32; a weight is rounded to the inputs' type for the
// product with v, since the matrix cores take both operands of one type: an error of up to 2^-9 of
// each term in bf16, as in v itself.  Against 64 bits, encoder chunks of 188 in bf16 are off by 0.0023
// in relative norm, with weights in 32 bits by 0.0017, the output's own rounding.
//
// Both products are matrix instructions on transposed tiles: S^T = K Q^T gives
// each lane the scores of one query, so the softmax is within lanes (but for
// one exchange when m moves), and S^T's register order is an operand order of
// the second product O^T = V^T P^T once V's rows are read in the same order
// (the transposing LDS read): the weights never leave their registers.
//
// K and V steps go from memory into LDS directly (buffer loads with an LDS
// destination) while the step before is computed on.  Rows past a sequence's
// end and hidden rows take an offset past the buffer's range, which the
// hardware answers with zeros: neither is read, so NaN or infinity there
// reaches nothing.  LDS rows hold their 16-byte chunks in an order permuted by
// the row (K: any chunk of 16 rows on distinct banks; V: 4 rows x 64 bytes).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "sfe_internal.hpp"
#include "sfe_ops.hpp"

namespace sfe {
namespace {

typedef __bf16 Bf;
typedef _Float16 Hf;
typedef float F2 __attribute__((ext_vector_type(2)));
typedef float F4 __attribute__((ext_vector_type(4)));
typedef float F16 __attribute__((ext_vector_type(16)));
typedef int I4 __attribute__((ext_vector_type(4)));
typedef short S4 __attribute__((ext_vector_type(4)));
typedef short S8 __attribute__((ext_vector_type(8)));

template <typename T>
struct Mat;
template <>
struct Mat<Bf> {
  typedef Bf V8 __attribute__((ext_vector_type(8)));
  typedef Bf V2 __attribute__((ext_vector_type(2)));
  static __device__ F16 m32(V8 a, V8 b, F16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
  static __device__ F4 m16(V8 a, V8 b, F4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
  static constexpr uint32_t kExp = 0x7f807f80, kCarry = 0x00800080, kOne = 0x3f80;
  // the reference moves when a score passes it by kRise, to kBelow below the maximum
  static constexpr float kRise = 0.0f, kBelow = -8.0f;
};
template <>
struct Mat<Hf> {
  typedef Hf V8 __attribute__((ext_vector_type(8)));
  typedef Hf V2 __attribute__((ext_vector_type(2)));
  static __device__ F16 m32(V8 a, V8 b, F16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
  static __device__ F4 m16(V8 a, V8 b, F4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }
  static constexpr uint32_t kExp = 0x7c007c00, kCarry = 0x04000400, kOne = 0x3c00;
  static constexpr float kRise = 15.0f, kBelow = 7.0f;
};

constexpr float kNever = -3e38f;  // reference exponent before the first visible key: below every score that counts
// Scores past this are scaled and rounded before the reference is taken off: the f32 reference of such
// a row is a rounded score itself, and exact products less it would be off by its rounding.
constexpr float kLarge = 1048576.0f;
constexpr uint32_t kOutside = 0x80000000u;  // an offset past every buffer's range
constexpr int kBufWord3 = 0x00020000;

__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) char*)p;
}

// The rows of a tensor's head as a raw buffer that moves along them: from row `row`, `rows`
// of them in reach (as far as 32-bit offsets go; the others read as zeros; without rows, none, whatever the
// stride: rows of one address, stride 0, too).
struct RowBuffer {
  uint64_t at;
  int64_t bytes;
  __device__ __forceinline__ RowBuffer(const AttnTensor& t, int64_t row, int64_t rows, int head, int dim_bytes)
      : at((uint64_t)(uintptr_t)t.data + (uint64_t)(row * t.row + (int64_t)head * t.head)),
        bytes(rows > 0 ? (rows - 1) * t.row + dim_bytes : 0) {}
  __device__ __forceinline__ void advance(int64_t by) {
    at += (uint64_t)by;
    bytes -= by;
  }
  __device__ __forceinline__ I4 words() const {
    I4 r;
    r.x = __builtin_amdgcn_readfirstlane((int)(uint32_t)at);
    r.y = __builtin_amdgcn_readfirstlane((int)((uint32_t)(at >> 32) & 0xffffu));
    r.z = __builtin_amdgcn_readfirstlane((int)(bytes < 0 ? 0 : (bytes < 0x7fffff00 ? bytes : 0x7fffff00)));
    r.w = kBufWord3;
    return r;
  }
};

// 16 bytes a lane from buffer offset `off` (a lane's own) into LDS at `lds` +
// 16 * lane.  Completion is waited for with vmcnt.
__device__ __forceinline__ void load_lds(I4 buf, uint32_t off, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(off), "s"(buf)
               : "memory");
}

template <typename T>
__device__ __forceinline__ typename Mat<T>::V8 read_k(uint32_t lds) {
  return __builtin_bit_cast(typename Mat<T>::V8, *(const __attribute__((address_space(3))) S8*)(uintptr_t)lds);
}
// Two transposed reads: 4 + 4 rows of V of this lane's column.
template <typename T>
__device__ __forceinline__ typename Mat<T>::V8 read_v(uint32_t lo, uint32_t hi) {
  typedef __attribute__((address_space(3))) S4* P;
  const S4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)lo);
  const S4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((P)(uintptr_t)hi);
  return __builtin_bit_cast(typename Mat<T>::V8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// s * c rounded, less m (never one fused operation).
__device__ __forceinline__ float scaled_less(float s, float c, float m) {
#pragma clang fp contract(off)
  const float x = s * c;
  return x - m;
}

// The larger (sum) of this lane's value and that of the lane 32 away.
__device__ __forceinline__ float max_halves(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float sum_halves(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}

// Keys that query `pos` of a sequence sees, [*lo, *hi] (empty: *hi < *lo).
__device__ __forceinline__ void visible(const AttnArgs& a, int pos, int lq, int lk, int* lo, int* hi) {
  const int64_t at = (int64_t)pos + lk - lq;
  const int64_t l = a.left == kAttnNoBound ? 0 : at - a.left, h = a.right == kAttnNoBound ? lk - 1 : at + a.right;
  *lo = (int)(l < 0 ? 0 : (l > lk ? lk : l));
  *hi = (int)(h < -1 ? -1 : (h > lk - 1 ? lk - 1 : h));
}

// Bits [lo, hi] of a word, both taken relative to its first key.
__device__ __forceinline__ uint64_t span_bits(int lo, int hi) {
  lo = lo < 0 ? 0 : lo;
  hi = hi > 63 ? 63 : hi;
  return hi < lo ? 0 : (~0ull >> (63 - hi)) & (~0ull << lo);
}

// Which unit a workgroup takes: consecutive workgroups go to the 8 XCDs in turn, each of which
// has a contiguous share of the units, of about equal work.
__device__ __forceinline__ int unit_of_block(const AttnArgs& a) {
  const int x = (int)(blockIdx.x % 8), u = a.share[x] + (int)(blockIdx.x / 8);
  return u < a.share[x + 1] ? u : -1;
}

// Unit u: units go kv head by kv head, so the tiles that read one sequence's keys find them in
// one L2.  (Sequence by sequence, the heads of a short one side by side, with shares of equal work as
// well: 280 sequences of 188 131-134 us against 131-132, causal prompts of 700-8192 in 32/8 heads of 128
// 942-948 us against 903-908.)
struct Unit {
  int64_t q_row, k_row;
  int lq, lk, kv0, kv1, row0, part, kvh, total;
};
__device__ __forceinline__ Unit unit_at(const AttnArgs& a, int u) {
  // (as constant memory: scalar loads, which no wait for vector memory is tied to)
  typedef const __attribute__((address_space(4))) AttnItem* Items;
  u = __builtin_amdgcn_readfirstlane(u);
  Unit r;
  r.kvh = (int)((unsigned)u / (unsigned)a.n_items);
  const Items it = (Items)(uintptr_t)a.items + (u - r.kvh * a.n_items);
  r.q_row = it->q_row;
  r.k_row = it->k_row;
  r.lq = it->lq;
  r.lk = it->lk;
  r.kv0 = it->kv0;
  r.kv1 = it->kv1;
  r.row0 = it->row0;
  r.part = it->part;
  r.total = it->lq * a.group;
  return r;
}

// The key mask of 64 keys from row `key` on, from its packed words (one more than the keys fill).
// (Read by the byte, each step's mask was one more trip to memory, waited for
// together with the loads into LDS.)
__device__ __forceinline__ uint64_t key_bits(const AttnArgs& a, int64_t key) {
  typedef const __attribute__((address_space(4))) uint64_t* Words;
  const Words w = (Words)(uintptr_t)a.mask + (key >> 6);
  const int shift = __builtin_amdgcn_readfirstlane((int)(key & 63));
  return shift ? w[0] >> shift | w[1] << (64 - shift) : w[0];
}

// Packs a key mask: bit i of word w is key 64 w + i.
__global__ __launch_bounds__(256) void sfe_attn_mask_kernel(const uint8_t* __restrict__ mask, int64_t keys, uint64_t* __restrict__ words,
                                                            int64_t n) {
  const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (w >= n) return;
  const int64_t key = 64 * w + (threadIdx.x & 63);
  const uint64_t bits = __ballot(key < keys && mask[key] != 0);
  if ((threadIdx.x & 63) == 0) words[w] = bits;
}

// Zeros chunk n of 16 bytes of the output's rows of no sequence: [0, first), then from `last` on.
__global__ __launch_bounds__(256) void sfe_attn_zero_kernel(AttnTensor out, int heads, int chunks, int64_t first, int64_t last,
                                                            int64_t n, int64_t total) {
  n += (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (n >= total) return;
  const int64_t r = n / (heads * chunks);
  const int c = (int)(n - r * (heads * chunks)), h = c / chunks;
  char* p = const_cast<char*>(out.data) + (r < first ? r : r - first + last) * out.row + h * out.head;
  *reinterpret_cast<uint4*>(p + 16 * (c - h * chunks)) = make_uint4(0, 0, 0, 0);
}

// Whether any of a V operand's 8 values is infinite or NaN.
template <typename T>
__device__ __forceinline__ uint32_t nonfinite(typename Mat<T>::V8 v) {
  const I4 w = __builtin_bit_cast(I4, v);
  uint32_t bad = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) bad |= ((uint32_t)w[i] & Mat<T>::kExp) + Mat<T>::kCarry;
  return bad & 0x80008000u;
}

// A V operand with infinite or NaN values, of keys that some queries see and
// others do not: *clean has zeros for them, *pos and *neg ones where a query that sees
// the key has to get +inf or -inf (both: NaN).
template <typename T>
__device__ __forceinline__ void split_nonfinite(S8 v, S8* clean, S8* pos, S8* neg) {
  constexpr uint32_t e = Mat<T>::kExp & 0xffff;
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t x = (uint16_t)v[j];
    const bool bad = (x & e) == e, nan = bad && (x & 0x7fff) != e;
    (*clean)[j] = bad ? 0 : v[j];
    (*pos)[j] = bad && (nan || !(x & 0x8000)) ? Mat<T>::kOne : 0;
    (*neg)[j] = bad && (nan || (x & 0x8000)) ? Mat<T>::kOne : 0;
  }
}

// o += V^T P^T of a step where values of V that are not finite are kept from the rows that do
// not see their key.  see: bit 32 h + 8 (i / 4) + i % 4, the lane's row sees that key; read(c, n):
// V operand of keys 16 c and channels 32 n.
template <typename T, int NT, class F>
__device__ __forceinline__ void careful_values(F16 (&o)[NT], const typename Mat<T>::V8 (&p)[4], uint64_t see, F&& read) {
  typedef typename Mat<T>::V8 V8;
#pragma unroll 1
  for (int c = 0; c < 4; ++c) {
    const V8 pc = c < 2 ? (c == 0 ? p[0] : p[1]) : (c == 2 ? p[2] : p[3]);
    S8 seen;
#pragma unroll
    for (int j = 0; j < 8; ++j) seen[j] = (see >> (16 * c + 8 * (j / 4) + j % 4)) & 1 ? Mat<T>::kOne : 0;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      V8 v = read(c, n);
      if (__any(nonfinite<T>(v) != 0)) {
        S8 clean, up, down;
        split_nonfinite<T>(__builtin_bit_cast(S8, v), &clean, &up, &down);
        F16 none;
#pragma unroll
        for (int i = 0; i < 16; ++i) none[i] = 0.0f;
        const F16 ups = Mat<T>::m32(__builtin_bit_cast(V8, up), __builtin_bit_cast(V8, seen), none);
        const F16 downs = Mat<T>::m32(__builtin_bit_cast(V8, down), __builtin_bit_cast(V8, seen), none);
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if (ups[i] > 0.0f) o[n][i] += INFINITY;
          if (downs[i] > 0.0f) o[n][i] -= INFINITY;
        }
        v = __builtin_bit_cast(V8, clean);
      }
      o[n] = Mat<T>::m32(v, pc, o[n]);
    }
  }
}

// ---- rows: 128 packed rows a workgroup ------------------------------------------------

template <int NT>
struct Geo {  // LDS rows of a step: 256 bytes (128 channels) or 128 (64)
  static constexpr int kPitch = NT > 2 ? 256 : 128;
  static constexpr int kChunks = kPitch / 16;
  static __device__ int k_swizzle(int row) { return NT > 2 ? row & 15 : (row >> 1) & 7; }
  static __device__ int v_swizzle(int row) { return NT > 2 ? 4 * (row & 3) : 4 * ((row >> 1) & 1); }
};

// Whether any of a lane's results is infinite or NaN: 0 times it is then NaN.
template <int NT>
__device__ __forceinline__ bool not_finite(const F16 (&o)[NT]) {
  float z[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i % 4] = __builtin_fmaf(o[n][i], 0.0f, z[i % 4]);
  return (z[0] + z[1]) + (z[2] + z[3]) != 0.0f;
}

// Whether a row's scores were too large for the loops without care.
__device__ __forceinline__ bool large(float m) { return fabsf(m) > kLarge && m != kNever; }

// Writes a wave's 32 rows.  The two lanes of a row hold 4 channels of every 8 each; an exchange
// gives either all 8 of every other chunk, 16 bytes a store.  (Through LDS, so that a store
// instruction wrote whole rows, the end of a workgroup took 1.5 us against 0.8.)
template <typename T, int NT>
__device__ __forceinline__ void store_rows(const AttnArgs& a, const F16 (&o)[NT], float l, int64_t q_row, int kvh, int row0,
                                           int total, int lane) {
  typedef typename Mat<T>::V2 V2;
  const int half = lane >> 5, r = row0 + (lane & 31);
  const float inv = l > 0.0f || l != l ? 1.0f / l : 0.0f;  // (a row that sees nothing is zero)
  const int rc = r < total ? r : total - 1;
  const int at = (int)((unsigned)rc / (unsigned)a.group);
  char* p = const_cast<char*>(a.o.data) + (q_row + at) * a.o.row + (int64_t)(kvh * a.group + rc - at * a.group) * a.o.head;
#pragma unroll
  for (int c = 0; c < 4 * NT; c += 2) {
    // chunks c and c + 1: registers 4 (c % 4) .. of tile c / 4
    const F16& x = o[c / 4];
    const int i = 4 * (c % 4);
    uint32_t e[2], f[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const F2 u = {x[i + 2 * j] * inv, x[i + 2 * j + 1] * inv}, w = {x[i + 4 + 2 * j] * inv, x[i + 5 + 2 * j] * inv};
      const auto y = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, __builtin_convertvector(u, V2)),
                                                      __builtin_bit_cast(uint32_t, __builtin_convertvector(w, V2)), false, false);
      e[j] = y[0];
      f[j] = y[1];
    }
    if (r < total && 16 * (c + half) < 2 * a.dim)
      *reinterpret_cast<uint4*>(p + 16 * (c + half)) = make_uint4(e[0], e[1], f[0], f[1]);
  }
}

// A workgroup: 4 waves of 32 packed rows, two workgroups a CU, over several units (tiles and kv
// heads) one after the other.  Short sequences spend their time waiting (for a
// unit's description, its queries, its first keys), so the last step of a unit has the next unit's first keys
// in flight and, once the scores are there, its queries.  (280 sequences of 188, 8 heads of 128:
// 128 us with a workgroup per unit.)  Units whose result is not finite are noted and done
// again at the end, CAREFUL: values of V that are not finite are kept from the rows that do not
// see their key (they would reach them as 0 * inf), and scores past 2^20 are rounded before their reference is
// taken off.  280 sequences of 188, 8 heads of 128: 119 us, 3.6 TB/s; 45,000
// rows that see 128 to either side 130 us, 2.8 TB/s; 256 of 13-251, 8 heads of 64, masked, 38 us, 2.2 TB/s.  Bound by the
// latency of a unit's few steps (its vector instructions take 36-44% of the time).
// Units of a workgroup at most.  (One after the other in 2 or 3 workgroups a CU for the whole
// call: the same on 280 sequences of 188, 117-122 us, and 51 us against 46 on 256 of 13-251, whose
// units are of unequal length.)
constexpr int kRowsUnits = 2;

// NT: head dim in units of 32 channels, rounded up.  MASKED: key mask.  stride: an XCD's workgroups.
template <typename T, int NT, bool MASKED>
__global__ __launch_bounds__(256, NT == 2 ? 3 : 2) void sfe_attn_rows_kernel(AttnArgs a) {
  typedef Geo<NT> G;
  typedef typename Mat<T>::V8 V8;
  typedef typename Mat<T>::V2 V2;
  constexpr int kStep = kAttnStepRows;
  constexpr int kBuf = kStep * G::kPitch;  // bytes of a step of K (or V)
  constexpr int kLoads = kBuf / 4096;      // load instructions of a wave for it
  constexpr int kRowsPerLoad = 4096 / G::kPitch;
  __shared__ __align__(1024) char lds[4 * kBuf];  // K, V of two steps
  __shared__ int again[kRowsUnits];               // the workgroup's unit is to be done with care
  const int stride = (int)(gridDim.x / 8), first = unit_of_block(a);
  if (first < 0) return;
  const int last = a.share[blockIdx.x % 8 + 1];
  const int t = (int)threadIdx.x, lane = t & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int dim_bytes = 2 * a.dim;
  const uint32_t base = lds_address(lds);
  if (t < kRowsUnits) again[t] = 0;

  // ---- addresses
  const int lrow = t / G::kChunks, lchunk = t % G::kChunks;
  const int kc = lchunk ^ G::k_swizzle(lrow), vc = lchunk ^ G::v_swizzle(lrow);
  const uint32_t k_off = 16 * kc < dim_bytes ? (uint32_t)(lrow * a.k.row) + 16 * kc : kOutside;
  const uint32_t v_off = 16 * vc < dim_bytes ? (uint32_t)(lrow * a.v.row) + 16 * vc : kOutside;
  const uint32_t k_next = (uint32_t)(kRowsPerLoad * a.k.row), v_next = (uint32_t)(kRowsPerLoad * a.v.row);
  const int64_t k_step = kStep * a.k.row, v_step = kStep * a.v.row;
  const uint32_t wave_base = __builtin_amdgcn_readfirstlane(base + 1024 * wave);
  uint32_t k_addr[2 * NT];
#pragma unroll
  for (int s = 0; s < 2 * NT; ++s)
    k_addr[s] = base + (lane & 31) * G::kPitch + 16 * ((2 * s + half) ^ G::k_swizzle(lane & 31));
  uint32_t v_addr[NT];
  {
    const int row = 4 * half + ((lane & 15) >> 2);
#pragma unroll
    for (int n = 0; n < NT; ++n)
      v_addr[n] = base + 2 * kBuf + row * G::kPitch +
                  16 * ((4 * n + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ G::v_swizzle(row)) + 8 * (lane & 1);
  }

  // ---- a unit's queries (operand B of the first product) and what they see
  V8 q[2 * NT];
  int lo = 0, hi = 0;
  auto load_queries = [&](const Unit& un) {
    const int r = un.row0 + 32 * wave + (lane & 31);
    const int rc = r < un.total ? r : un.total - 1;
    const int pos = (int)((unsigned)rc / (unsigned)a.group);
    visible(a, pos, un.lq, un.lk, &lo, &hi);
    const char* p = a.q.data + (un.q_row + pos) * a.q.row + (int64_t)(un.kvh * a.group + rc - pos * a.group) * a.q.head;
#pragma unroll
    for (int s = 0; s < 2 * NT; ++s) {
      const int c = 2 * s + half;
      S8 v = {0, 0, 0, 0, 0, 0, 0, 0};
      if (16 * c < dim_bytes) v = *reinterpret_cast<const S8*>(p + 16 * c);
      q[s] = __builtin_bit_cast(V8, v);
    }
  };
  // (waited for outside the steps: a wait within them would be one for the loads into LDS too)
  auto queries_there = [&]() {
#pragma unroll
    for (int s = 0; s < 2 * NT; ++s) asm volatile("" : "+v"(q[s]));
  };
  auto mask_bits = [&](const Unit& un, int kv) -> uint64_t { return MASKED ? key_bits(a, un.k_row + kv) : ~0ull; };
  auto load_step = [&](const RowBuffer& kr, const RowBuffer& vr, uint32_t buf, uint64_t bits) {
    const I4 kb = kr.words(), vb = vr.words();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint32_t ko = k_off == kOutside ? kOutside : k_off + i * k_next;
      uint32_t vo = v_off == kOutside ? kOutside : v_off + i * v_next;
      if (MASKED && !((bits >> (i * kRowsPerLoad + lrow)) & 1)) ko = vo = kOutside;
      load_lds(kb, ko, wave_base + buf + i * 4096);
      load_lds(vb, vo, wave_base + 2 * kBuf + buf + i * 4096);
    }
  };

  F16 o[NT];
  float m, l;
  uint32_t buf = 0;  // of the current step: 0 or kBuf
  bool stores = false;  // the last unit's end left exactly 2 NT stores behind its loads
  // Runs unit `un`, whose queries and first step have been asked for; `next`: the one after (if
  // `more`), whose queries and first step it asks for.  MASKED: bits of the first two steps.
  auto run = [&](auto careful, const Unit& un, const Unit& next, bool more, uint64_t& bits, uint64_t& bits_next) {
    constexpr bool kCareful = decltype(careful)::value;
    const int lo_all = __builtin_amdgcn_readlane(lo, 31), hi_all = __builtin_amdgcn_readlane(hi, 0);
    const int lo_any = __builtin_amdgcn_readlane(lo, 0), hi_any = __builtin_amdgcn_readlane(hi, 31);
    const int my_lo = lo, my_hi = hi;
    const bool idle = un.row0 + 32 * wave >= un.total;
    RowBuffer kr(a.k, un.k_row + un.kv0, un.kv1 - un.kv0, un.kvh, dim_bytes);
    RowBuffer vr(a.v, un.k_row + un.kv0, un.kv1 - un.kv0, un.kvh, dim_bytes);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[n][i] = 0.0f;
    m = kNever;
    l = 0.0f;
    // (a unit without keys goes through one step that nothing is seen in)
    for (int kv = un.kv0;; kv += kStep) {
      const bool final = kv + kStep >= un.kv1;
      // this step's keys have landed (the stores behind them need not), and every wave is done
      // with the step before
      if (stores)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * NT) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
      stores = false;
      uint64_t bits_after = ~0ull;
      if (!final) {
        kr.advance(k_step);
        vr.advance(v_step);
        load_step(kr, vr, buf ^ kBuf, bits_next);
        bits_after = mask_bits(un, kv + 2 * kStep);
      } else if (more) {
        bits_next = mask_bits(next, next.kv0);
        load_step(RowBuffer(a.k, next.k_row + next.kv0, next.kv1 - next.kv0, next.kvh, dim_bytes),
                  RowBuffer(a.v, next.k_row + next.kv0, next.kv1 - next.kv0, next.kvh, dim_bytes), buf ^ kBuf, bits_next);
        bits_after = mask_bits(next, next.kv0 + kStep);
      }
      const int end = un.kv1 < kv + kStep ? un.kv1 : kv + kStep;  // keys of the step: [kv, end)
      const bool seen = !idle && lo_any < end && hi_any >= kv;
      F16 s[2];
      constexpr int kK = 2 * NT, kV = 4 * NT, kAhead = 3;
      if (seen) {
        // (operands are read kAhead pairs ahead; see the tall kernel)
        V8 kf[kK][2];
        auto read_pair = [&](int c) {
          kf[c][0] = read_k<T>(k_addr[c] + buf);
          kf[c][1] = read_k<T>(k_addr[c] + buf + 32 * G::kPitch);
        };
#pragma unroll
        for (int c = 0; c < kAhead; ++c) read_pair(c);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[h][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < kK; ++c) {
          if (c + kAhead < kK) read_pair(c + kAhead);
          s[0] = Mat<T>::m32(kf[c][0], q[c], s[0]);
          s[1] = Mat<T>::m32(kf[c][1], q[c], s[1]);
          __builtin_amdgcn_sched_barrier(0);
        }
      }
      if (final && more) load_queries(next);
      if (seen) {
        const bool edge = lo_all > kv || hi_all < kv + kStep - 1 || end < kv + kStep;
        uint64_t see = ~0ull;
        if (edge || (MASKED && bits != ~0ull)) {
          // lane's keys are 32 h + 8 (i / 4) + 4 half + i % 4
          see = span_bits(my_lo - kv, (my_hi < end - 1 ? my_hi : end - 1) - kv);
          if (MASKED) see &= bits;
          see >>= 4 * half;
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 16; ++i)
              s[h][i] = (see >> (32 * h + 8 * (i / 4) + i % 4)) & 1 ? s[h][i] : -INFINITY;
        }
        float top = s[0][0];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) top = fmaxf(top, s[h][i]);
        if (__any(top * a.scale_log2 > m + Mat<T>::kRise)) {
          const float nm = fmaxf(m, scaled_less(max_halves(top), a.scale_log2, Mat<T>::kBelow));
          const float f = exp2_fast(m - nm);
          m = nm;
          l *= f;
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[n][i] *= f;
        }
        auto less = [&](float x) {
          return kCareful ? scaled_less(x, a.scale_log2, m) : __builtin_fmaf(x, a.scale_log2, -m);
        };
        float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        V8 p[4];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const F2 w = {exp2_fast(less(s[h][i])), exp2_fast(less(s[h][i + 1]))};
            sum[i % 4] += w.x;
            sum[i % 4 + 1] += w.y;
            const V2 c = __builtin_convertvector(w, V2);
            p[2 * h + i / 8][i % 8] = c.x;
            p[2 * h + i / 8][i % 8 + 1] = c.y;
          }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
        if constexpr (!kCareful) {
          V8 vf[kV];
          auto read_value = [&](int i) {
            const uint32_t at = v_addr[i % NT] + buf + 16 * (i / NT) * G::kPitch;
            vf[i] = read_v<T>(at, at + 8 * G::kPitch);
          };
#pragma unroll
          for (int i = 0; i < 2 * kAhead; ++i) read_value(i);
#pragma unroll
          for (int i = 0; i < kV; ++i) {
            if (i + 2 * kAhead < kV) read_value(i + 2 * kAhead);
            o[i % NT] = Mat<T>::m32(vf[i], p[i / NT], o[i % NT]);
            __builtin_amdgcn_sched_barrier(0);
          }
        } else {
          careful_values<T, NT>(o, p, see, [&](int c, int n) {
            const uint32_t at = v_addr[n] + buf + 16 * c * G::kPitch;
            return read_v<T>(at, at + 8 * G::kPitch);
          });
        }
      }
      buf ^= kBuf;
      bits = bits_next;
      bits_next = bits_after;
      if (final) break;
    }
    // (before the stores, which nothing then waits for)
    if (more) queries_there();
    l = sum_halves(l);
    if (un.part >= 0) {
      const int64_t at = ((int64_t)un.part * a.kv_heads + un.kvh) * kAttnTileRows + 32 * wave + (lane & 31);
      float* po = a.part_o + at * (32 * NT);
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; i += 4)
          *reinterpret_cast<F4*>(po + 32 * n + 2 * i + 4 * half) = F4{o[n][i], o[n][i + 1], o[n][i + 2], o[n][i + 3]};
      if (half == 0) a.part_ml[at] = make_float2(m, l);
    } else {
      store_rows<T, NT>(a, o, l, un.q_row, un.kvh, un.row0 + 32 * wave, un.total, lane);
      stores = !idle && dim_bytes == 64 * NT;
    }
  };

  auto begin = [&](const Unit& un, uint64_t& bits, uint64_t& bits_next) {
    load_queries(un);
    bits = mask_bits(un, un.kv0);
    bits_next = mask_bits(un, un.kv0 + kStep);
    load_step(RowBuffer(a.k, un.k_row + un.kv0, un.kv1 - un.kv0, un.kvh, dim_bytes),
              RowBuffer(a.v, un.k_row + un.kv0, un.kv1 - un.kv0, un.kvh, dim_bytes), buf, bits);
    queries_there();
  };
  Unit un = unit_at(a, first);
  uint64_t bits, bits_next;
  __syncthreads();  // (`again` is clear)
  begin(un, bits, bits_next);
  for (int u = first, k = 0; u < last; u += stride, ++k) {
    const bool more = u + stride < last;
    const Unit next = unit_at(a, more ? u + stride : u);
    run(std::false_type(), un, next, more, bits, bits_next);
    if (__any(not_finite(o) || large(m)) && lane == 0) again[k] = 1;
    un = next;
  }
  __syncthreads();
  for (int u = first, k = 0; u < last; u += stride, ++k) {
    if (!__builtin_amdgcn_readfirstlane(again[k])) continue;
    un = unit_at(a, u);
    buf = 0;
    begin(un, bits, bits_next);
    run(std::true_type(), un, un, false, bits, bits_next);
    __syncthreads();
  }
}

// ---- tall: 256 packed rows a workgroup ----------------------------------------------------

// One workgroup: 8 waves of 32 packed rows, two on each SIMD: waves 0-3 and 4-7 take turns at
// the matrix cores.  An interval is the time between two barriers; in it one half runs
// the products of a step (S of step j, then O of step j - 1) and the other the softmax of
// its step, so that on every SIMD matrix and vector instructions issue side by side.  (Left to
// themselves two waves of a SIMD overlapped little: causal prompts of up to 8192 took 2,660
// cycles a step and wave, its products 1,024 and its vector instructions 1,150.)
// K and V lie in 3 buffers each; the loads of K of step j + 2 and V of step j + 1 are issued
// in interval 2j, after the last read of the buffers' former steps, and waited for two
// intervals later by count, so every wave issues the same number in every step (steps past
// the end load nothing: all their offsets are outside).  8 causal prompts of 700-8192, 32/8 heads of 128:
// 1.12-1.15 ms, 1,030-1,060 TFLOP/s; bound by the vector instructions and the barriers between the
// halves' turns (the matrix cores run 54% of the time).
template <typename T, int NT, bool MASKED>
__global__ __launch_bounds__(512, 2) void sfe_attn_tall_kernel(AttnArgs a) {
  typedef Geo<NT> G;
  typedef typename Mat<T>::V8 V8;
  typedef typename Mat<T>::V2 V2;
  constexpr int kStep = kAttnStepRows;
  constexpr int kBuf = kStep * G::kPitch;  // bytes of a step of K (or V)
  constexpr int kLoads = kBuf / 8192;      // load instructions of a wave for it
  constexpr int kRowsPerLoad = 8192 / G::kPitch;
  __shared__ __align__(1024) char lds[6 * kBuf];  // 3 steps of K, 3 of V
  __shared__ int again[8];
  const int u = unit_of_block(a);
  if (u < 0) return;
  const Unit un = unit_at(a, u);
  const int lq = un.lq, lk = un.lk, kv0 = un.kv0, kv1 = un.kv1, row0 = un.row0, part = un.part, kvh = un.kvh;
  const int64_t q_row = un.q_row, k_row = un.k_row;
  const int total = un.total;
  const int t = (int)threadIdx.x, lane = t & 63, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
  const int dim_bytes = 2 * a.dim;
  const uint32_t base = lds_address(lds);

  // ---- addresses
  const int lrow = t / G::kChunks, lchunk = t % G::kChunks;
  const int kc = lchunk ^ G::k_swizzle(lrow), vc = lchunk ^ G::v_swizzle(lrow);
  const uint32_t k_off = 16 * kc < dim_bytes ? (uint32_t)(lrow * a.k.row) + 16 * kc : kOutside;
  const uint32_t v_off = 16 * vc < dim_bytes ? (uint32_t)(lrow * a.v.row) + 16 * vc : kOutside;
  const uint32_t k_next = (uint32_t)(kRowsPerLoad * a.k.row), v_next = (uint32_t)(kRowsPerLoad * a.v.row);
  const uint32_t wave_base = __builtin_amdgcn_readfirstlane(base + 1024 * wave);
  uint32_t k_addr[2 * NT];
#pragma unroll
  for (int s = 0; s < 2 * NT; ++s)
    k_addr[s] = base + (lane & 31) * G::kPitch + 16 * ((2 * s + half) ^ G::k_swizzle(lane & 31));
  uint32_t v_addr[NT];
  {
    const int row = 4 * half + ((lane & 15) >> 2);
#pragma unroll
    for (int n = 0; n < NT; ++n)
      v_addr[n] = base + 3 * kBuf + row * G::kPitch +
                  16 * ((4 * n + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ G::v_swizzle(row)) + 8 * (lane & 1);
  }

  auto mask_bits = [&](int kv) -> uint64_t { return MASKED ? key_bits(a, k_row + kv) : ~0ull; };
  // the next step's rows of K (or V) into LDS at dst
  auto load_rows = [&](const RowBuffer& x, uint32_t off, uint32_t next, uint32_t dst, uint64_t bits) {
    const I4 b = x.words();
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      uint32_t o = off == kOutside ? kOutside : off + i * next;
      if (MASKED && !((bits >> (i * kRowsPerLoad + lrow)) & 1)) o = kOutside;
      load_lds(b, o, wave_base + dst + i * 8192);
    }
  };
  const int64_t k_step = kStep * a.k.row, v_step = kStep * a.v.row;
  auto after = [](uint32_t slot) -> uint32_t { return slot == 2 * kBuf ? 0 : slot + kBuf; };

  // the first steps' loads, those of the queries behind them
  uint64_t bits0 = ~0ull, bits1 = ~0ull, bits2 = ~0ull;
  RowBuffer kr(a.k, 0, 0, 0, 0), vr = kr;
  auto begin = [&]() {
    bits0 = mask_bits(kv0), bits1 = mask_bits(kv0 + kStep), bits2 = mask_bits(kv0 + 2 * kStep);
    kr = RowBuffer(a.k, k_row + kv0, kv1 - kv0, kvh, dim_bytes);
    vr = RowBuffer(a.v, k_row + kv0, kv1 - kv0, kvh, dim_bytes);
    RowBuffer none = vr;
    none.bytes = 0;
    load_rows(none, v_off, v_next, 5 * kBuf, ~0ull);  // (zeros: the first step's weights of the step before are too)
    load_rows(kr, k_off, k_next, 0, bits0);
    load_rows(vr, v_off, v_next, 3 * kBuf, bits0);
    kr.advance(k_step);
    load_rows(kr, k_off, k_next, kBuf, bits1);
  };
  begin();

  // ---- queries: lane's row, operand B of the first product
  const int r = row0 + 32 * wave + (lane & 31);
  const int rc = r < total ? r : total - 1;
  const int pos = (int)((unsigned)rc / (unsigned)a.group);
  int lo, hi;
  visible(a, pos, lq, lk, &lo, &hi);
  V8 q[2 * NT];
  {
    const char* p = a.q.data + (q_row + pos) * a.q.row + (int64_t)(kvh * a.group + rc - pos * a.group) * a.q.head;
#pragma unroll
    for (int s = 0; s < 2 * NT; ++s) {
      const int c = 2 * s + half;
      S8 v = {0, 0, 0, 0, 0, 0, 0, 0};
      if (16 * c < dim_bytes) v = *reinterpret_cast<const S8*>(p + 16 * c);
      q[s] = __builtin_bit_cast(V8, v);
    }
    // (waited for here: a wait within the loop would be one for the loads into LDS too)
#pragma unroll
    for (int s = 0; s < 2 * NT; ++s) asm volatile("" : "+v"(q[s]));
  }
  const bool idle = row0 + 32 * wave >= total;  // none of the wave's rows exists
  const int lo_all = __builtin_amdgcn_readlane(lo, 31), hi_all = __builtin_amdgcn_readlane(hi, 0);
  const int lo_any = __builtin_amdgcn_readlane(lo, 0), hi_any = idle ? -1 : __builtin_amdgcn_readlane(hi, 31);

  F16 o[NT];
  float m, l;

  // Runs over the keys.  CAREFUL: values of V that are not finite are kept from the rows that
  // do not see their key (they would reach them as 0 * inf).
  auto run = [&](auto careful) {
    constexpr bool kCareful = decltype(careful)::value;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[n][i] = 0.0f;
    m = kNever;
    l = 0.0f;
    // (the first step; of the second, K is on its way)
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(kLoads) : "memory");
    uint32_t k2 = 2 * kBuf, v1 = kBuf;  // buffers of K of step j + 2 and V of step j + 1
    uint32_t kj = 0, vp = 2 * kBuf;     // ... of K of step j and V of step j - 1
    F16 s[2];
    V8 p[4];
    // weights of step j - 1, zero where the wave's rows saw none of it
#pragma unroll
    for (int c = 0; c < 4; ++c) p[c] = V8{0, 0, 0, 0, 0, 0, 0, 0};
    bool did = false;
    uint64_t see_before = 0;
    // the loads of interval 2j: K of step j + 2 and V of step j + 1
    auto loads = [&]() {
      kr.advance(k_step);
      vr.advance(v_step);
      load_rows(kr, k_off, k_next, k2, bits2);
      load_rows(vr, v_off, v_next, 3 * kBuf + v1, bits1);
      k2 = after(k2);
      v1 = after(v1);
    };
    auto products = [&](int kv) {
      const int end = kv1 < kv + kStep ? kv1 : kv + kStep;  // keys of the step: [kv, end)
      const bool now = kv < kv1 && lo_any < end && hi_any >= kv;
      if (now || did) {
        // Both products as one stream of matrix instructions, operands read kAhead pairs (K)
        // or fragments (V) ahead of their use; the fences keep the compiler from reading
        // each just before it (every product then waited for its read) or all at once.
        __builtin_amdgcn_s_setprio(1);  // (1,194 us without, on the same prompts)
        constexpr int kK = 2 * NT, kV = kCareful ? 0 : 4 * NT, kAhead = 3;
        V8 kf[kK][2], vf[4 * NT];
        auto read_pair = [&](int c) {
          kf[c][0] = read_k<T>(k_addr[c] + kj);
          kf[c][1] = read_k<T>(k_addr[c] + kj + 32 * G::kPitch);
        };
        auto read_value = [&](int i) {
          const uint32_t at = v_addr[i % NT] + vp + 16 * (i / NT) * G::kPitch;
          vf[i] = read_v<T>(at, at + 8 * G::kPitch);
        };
#pragma unroll
        for (int c = 0; c < kAhead; ++c) read_pair(c);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i) s[h][i] = 0.0f;
#pragma unroll
        for (int c = 0; c < kK; ++c) {
          if (c + kAhead < kK) {
            read_pair(c + kAhead);
          } else if (!kCareful) {
            read_value(2 * (c + kAhead - kK));
            read_value(2 * (c + kAhead - kK) + 1);
          }
          s[0] = Mat<T>::m32(kf[c][0], q[c], s[0]);
          s[1] = Mat<T>::m32(kf[c][1], q[c], s[1]);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < kV; ++i) {
          if (i + 2 * kAhead < kV) read_value(i + 2 * kAhead);
          o[i % NT] = Mat<T>::m32(vf[i], p[i / NT], o[i % NT]);
          __builtin_amdgcn_sched_barrier(0);
        }
        __builtin_amdgcn_s_setprio(0);
        if constexpr (kCareful)
          careful_values<T, NT>(o, p, see_before, [&](int c, int n) {
            const uint32_t at = v_addr[n] + vp + 16 * c * G::kPitch;
            return read_v<T>(at, at + 8 * G::kPitch);
          });
      }
      did = now;
      kj = after(kj);
      vp = after(vp);
    };
    auto softmax = [&](int kv, uint64_t bits) {
      if (!did) {
#pragma unroll
        for (int c = 0; c < 4; ++c) p[c] = V8{0, 0, 0, 0, 0, 0, 0, 0};
        see_before = 0;
        return;
      }
      const int end = kv1 < kv + kStep ? kv1 : kv + kStep;
      // keys that some of the wave's rows do not see
      const bool edge = lo_all > kv || hi_all < kv + kStep - 1 || end < kv + kStep;
      if (kCareful) see_before = ~0ull;
      if (edge || (MASKED && bits != ~0ull)) {
        // lane's keys are 32 h + 8 (i / 4) + 4 half + i % 4
        uint64_t see = span_bits(lo - kv, (hi < end - 1 ? hi : end - 1) - kv);
        if (MASKED) see &= bits;
        see >>= 4 * half;
        if (kCareful) see_before = see;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[h][i] = (see >> (32 * h + 8 * (i / 4) + i % 4)) & 1 ? s[h][i] : -INFINITY;
      }
      float top = s[0][0];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[h][i]);
      if (__any(top * a.scale_log2 > m + Mat<T>::kRise)) {
        const float nm = fmaxf(m, scaled_less(max_halves(top), a.scale_log2, Mat<T>::kBelow));
        const float f = exp2_fast(m - nm);
        m = nm;
        l *= f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 16; ++i) o[n][i] *= f;
      }
      auto less = [&](float x) {
        return kCareful ? scaled_less(x, a.scale_log2, m) : __builtin_fmaf(x, a.scale_log2, -m);
      };
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const F2 w = {exp2_fast(less(s[h][i])), exp2_fast(less(s[h][i + 1]))};
          sum[i % 4] += w.x;
          sum[i % 4 + 1] += w.y;
          const V2 c = __builtin_convertvector(w, V2);
          p[2 * h + i / 8][i % 8] = c.x;
          p[2 * h + i / 8][i % 8 + 1] = c.y;
        }
      l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };
    auto barrier = []() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
    // (after the loads of one more step have been issued, those of the step before are done)
    auto landed = []() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(2 * kLoads) : "memory"); };
    if (wave < 4) {
      for (int kv = kv0; kv < kv1; kv += kStep) {
        loads();
        products(kv);
        barrier();
        softmax(kv, bits0);
        bits0 = bits1, bits1 = bits2, bits2 = mask_bits(kv + 3 * kStep);
        landed();
      }
      products(kv1);
      barrier();
    } else {
      loads();
      barrier();
      for (int kv = kv0; kv < kv1; kv += kStep) {
        products(kv);
        const uint64_t bits = bits0;
        bits0 = bits1, bits1 = bits2, bits2 = mask_bits(kv + 3 * kStep);
        landed();
        loads();
        softmax(kv, bits);
        barrier();
      }
      products(kv1);
    }
    l = sum_halves(l);
  };
  run(std::false_type());
  // A result that is not finite may be a hidden value's, one of large scores off: then once more, with care
  const int flag = __any(not_finite(o) || large(m));
  if (lane == 0) again[wave] = flag;
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  if (__any(again[lane & 7])) {
    begin();
    run(std::true_type());
  }

  if (part >= 0) {
    const int64_t at = ((int64_t)part * a.kv_heads + kvh) * kAttnTileTall + 32 * wave + (lane & 31);
    float* po = a.part_o + at * (32 * NT);
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 16; i += 4)
        *reinterpret_cast<F4*>(po + 32 * n + 2 * i + 4 * half) = F4{o[n][i], o[n][i + 1], o[n][i + 2], o[n][i + 3]};
    if (half == 0) a.part_ml[at] = make_float2(m, l);
    return;
  }
  store_rows<T, NT>(a, o, l, q_row, kvh, row0 + 32 * wave, total, lane);
}

// ---- few: 16 packed rows a workgroup, its waves share the keys ---------------------------

// A workgroup: 4 waves over one tile of 16 packed rows, each taking every fourth step of 32 keys
// with its own buffers, running maximum and sum (no barrier in the loop), added up at the end.  A wave's
// first two steps are in flight before its queries are, since such calls are one
// trip through memory.  Bound by that trip and the bytes of K and V: one token of 4 beams of 64
// streams over 126-1500 keys, 16/4 heads of 128, 20 us, 3.7 TB/s; one token over 45,000 keys 25 us, 3.7 TB/s; one
// sequence of 126, 8 heads of 128, 7 us.
template <typename T, int NT, bool MASKED>
__global__ __launch_bounds__(64 * kAttnWavesFew, 1) void sfe_attn_few_kernel(AttnArgs a) {
  typedef Geo<NT> G;
  typedef typename Mat<T>::V8 V8;
  typedef typename Mat<T>::V2 V2;
  constexpr int kStep = kAttnStepFew, kWaves = kAttnWavesFew;
  constexpr int kBuf = kStep * G::kPitch;  // bytes of a wave's step of K (or V)
  constexpr int kLoads = kBuf / 1024;
  constexpr int kRowsPerLoad = 1024 / G::kPitch;
  constexpr int ND = 2 * NT;  // tiles of 16 channels
  __shared__ __align__(1024) char lds[kWaves * 4 * kBuf];
  const int u = unit_of_block(a);
  if (u < 0) return;
  const Unit un = unit_at(a, u);
  const int lq = un.lq, lk = un.lk, kv0 = un.kv0, kv1 = un.kv1, row0 = un.row0, part = un.part, kvh = un.kvh;
  const int64_t q_row = un.q_row, k_row = un.k_row;
  const int total = un.total;
  const int t = (int)threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), quarter = lane >> 4;
  const int dim_bytes = 2 * a.dim;
  const uint32_t base = lds_address(lds) + wave * 4 * kBuf;

  const int lrow = lane / G::kChunks, lchunk = lane % G::kChunks;
  uint32_t k_addr[NT], v_addr[ND];
#pragma unroll
  for (int s = 0; s < NT; ++s)
    k_addr[s] = base + (lane & 15) * G::kPitch + 16 * ((4 * s + quarter) ^ G::k_swizzle(lane & 15));
  {
    const int row = 4 * quarter + ((lane & 15) >> 2);
#pragma unroll
    for (int n = 0; n < ND; ++n)
      v_addr[n] = base + 2 * kBuf + row * G::kPitch + 16 * ((2 * n + ((lane & 3) >> 1)) ^ G::v_swizzle(row)) + 8 * (lane & 1);
  }
  const int first = kv0 + wave * kStep;
  RowBuffer kr(a.k, k_row + first, kv1 - first, kvh, dim_bytes), vr(a.v, k_row + first, kv1 - first, kvh, dim_bytes);
  const int64_t k_turn = kWaves * kStep * a.k.row, v_turn = kWaves * kStep * a.v.row;
  // the rows of the buffers' step; then they move on to the wave's next
  auto load_step = [&](int buf, uint32_t bits) {
    const I4 kb = kr.words(), vb = vr.words();
    kr.advance(k_turn);
    vr.advance(v_turn);
    const uint32_t dst = __builtin_amdgcn_readfirstlane(base + buf * kBuf);
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const int row = i * kRowsPerLoad + lrow;
      const int kc = 16 * (lchunk ^ G::k_swizzle(row)), vc = 16 * (lchunk ^ G::v_swizzle(row));
      uint32_t ko = kc < dim_bytes ? (uint32_t)(row * a.k.row) + kc : kOutside;
      uint32_t vo = vc < dim_bytes ? (uint32_t)(row * a.v.row) + vc : kOutside;
      if (MASKED && !((bits >> row) & 1)) ko = vo = kOutside;
      load_lds(kb, ko, dst + i * 1024);
      load_lds(vb, vo, dst + 2 * kBuf + i * 1024);
    }
  };

  // the first two steps' loads, those of the queries behind them
  constexpr int kTurn = kWaves * kStep;  // keys of all waves' steps
  uint32_t bits = ~0u, bits_next = ~0u;
  if (MASKED && first < kv1) bits = (uint32_t)key_bits(a, k_row + first);
  if (first < kv1) load_step(0, bits);
  if (MASKED && first + kTurn < kv1) bits_next = (uint32_t)key_bits(a, k_row + first + kTurn);
  if (first + kTurn < kv1) load_step(1, bits_next);
  const int r = row0 + (lane & 15);
  const int rc = r < total ? r : total - 1;
  const int pos = (int)((unsigned)rc / (unsigned)a.group);
  int lo, hi;
  visible(a, pos, lq, lk, &lo, &hi);
  V8 q[NT];
  {
    const char* p = a.q.data + (q_row + pos) * a.q.row + (int64_t)(kvh * a.group + rc - pos * a.group) * a.q.head;
#pragma unroll
    for (int s = 0; s < NT; ++s) {
      const int c = 4 * s + quarter;
      S8 v = {0, 0, 0, 0, 0, 0, 0, 0};
      if (16 * c < dim_bytes) v = *reinterpret_cast<const S8*>(p + 16 * c);
      q[s] = __builtin_bit_cast(V8, v);
    }
    // (waited for here: a wait within the loop would be one for the loads into LDS too)
#pragma unroll
    for (int s = 0; s < NT; ++s) asm volatile("" : "+v"(q[s]));
  }
  const int lo_all = __builtin_amdgcn_readlane(lo, 15), hi_all = __builtin_amdgcn_readlane(hi, 0);
  const bool overlaid = a.v.row < dim_bytes;

  F4 o[ND];
#pragma unroll
  for (int n = 0; n < ND; ++n) o[n] = F4{0.0f, 0.0f, 0.0f, 0.0f};
  float m = kNever, l = 0.0f;
  int buf = 0;
  for (int kv = first; kv < kv1; kv += kTurn, buf ^= 1) {
    // (a wave's LDS buffers are its own: its loads are waited for by count)
    if (kv + kTurn < kv1)
      asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kLoads) : "memory");
    else
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const int end = kv1 < kv + kStep ? kv1 : kv + kStep;
    const uint32_t kb = buf * kBuf;
    F4 s[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[h] = F4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int c = 0; c < NT; ++c)
        s[h] = Mat<T>::m16(read_k<T>(k_addr[c] + kb + h * 16 * G::kPitch), q[c], s[h]);
    }
    // keys that some rows do not see; rows past the last key read as values of it where v's rows lie over each other
    // (stride 0 for one value of all keys), and as zeros elsewhere
    const bool uneven = lo_all > kv || hi_all < (lk < kv + kStep ? lk : kv + kStep) - 1 || (overlaid && end < kv + kStep);
    const bool edge = uneven || end < kv + kStep;
    uint32_t see = ~0u;
    if (edge || (MASKED && bits != ~0u)) {
      // lane's keys are 16 h + 4 quarter + i
      see = (uint32_t)span_bits(lo - kv, (hi < end - 1 ? hi : end - 1) - kv);
      if (MASKED) see &= bits;
      see >>= 4 * quarter;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 4; ++i) s[h][i] = (see >> (16 * h + i)) & 1 ? s[h][i] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, s[h][i]);
    if (__any(top * a.scale_log2 > m + Mat<T>::kRise)) {
      top = fmaxf(top, __shfl_xor(top, 16));
      const float nm = fmaxf(m, scaled_less(max_halves(top), a.scale_log2, Mat<T>::kBelow));
      const float f = exp2_fast(m - nm);
      m = nm;
      l *= f;
#pragma unroll
      for (int n = 0; n < ND; ++n) o[n] *= f;
    }
    V8 p;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        const F2 w = {exp2_fast(scaled_less(s[h][i], a.scale_log2, m)),
                      exp2_fast(scaled_less(s[h][i + 1], a.scale_log2, m))};
        l += w.x + w.y;
        const V2 c = __builtin_convertvector(w, V2);
        p[4 * h + i] = c.x;
        p[4 * h + i + 1] = c.y;
      }
#pragma unroll
    for (int n = 0; n < ND; ++n) {
      V8 v = read_v<T>(v_addr[n] + kb, v_addr[n] + kb + 16 * G::kPitch);
      if (uneven && __any(nonfinite<T>(v) != 0)) {  // (see the rows kernel)
        S8 clean, up, down, seen;
        split_nonfinite<T>(__builtin_bit_cast(S8, v), &clean, &up, &down);
#pragma unroll
        for (int j = 0; j < 8; ++j) seen[j] = (see >> (16 * (j / 4) + j % 4)) & 1 ? Mat<T>::kOne : 0;
        const F4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        const F4 ups = Mat<T>::m16(__builtin_bit_cast(V8, up), __builtin_bit_cast(V8, seen), zero);
        const F4 downs = Mat<T>::m16(__builtin_bit_cast(V8, down), __builtin_bit_cast(V8, seen), zero);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (ups[i] > 0.0f) o[n][i] += INFINITY;
          if (downs[i] > 0.0f) o[n][i] -= INFINITY;
        }
        v = __builtin_bit_cast(V8, clean);
      }
      o[n] = Mat<T>::m16(v, p, o[n]);
    }
    bits = bits_next;
    if (kv + 2 * kTurn < kv1) {  // into the buffer just read
      if (MASKED) bits_next = (uint32_t)key_bits(a, k_row + kv + 2 * kTurn);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      load_step(buf, bits_next);
    }
  }
  l += __shfl_xor(l, 16);
  l = sum_halves(l);

  // ---- the waves' results, added up through LDS
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
  constexpr int kDim = 32 * NT, kRowF = kDim + 4;  // floats of a row (4 of padding)
  float* ow = reinterpret_cast<float*>(lds);                          // [wave][16][kRowF]
  float2* ml = reinterpret_cast<float2*>(ow + kWaves * 16 * kRowF);   // [wave][16]
  static_assert((kWaves * 16 * kRowF + 2 * kWaves * 16) * 4 <= (int)sizeof(lds), "results fit");
#pragma unroll
  for (int n = 0; n < ND; ++n)
    *reinterpret_cast<F4*>(ow + (wave * 16 + (lane & 15)) * kRowF + 16 * n + 4 * quarter) = o[n];
  if (quarter == 0) ml[wave * 16 + lane] = make_float2(m, l);
  __syncthreads();
  for (int e = t; e < 16 * (kDim / 4); e += 64 * kWaves) {
    const int row = e / (kDim / 4), d = 4 * (e % (kDim / 4));
    float mm = kNever;
    for (int w = 0; w < kWaves; ++w) mm = fmaxf(mm, ml[w * 16 + row].x);
    F4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    float sum = 0.0f;
    for (int w = 0; w < kWaves; ++w) {
      const float2 x = ml[w * 16 + row];
      if (x.x == kNever && x.y == 0.0f) continue;  // (saw nothing)
      const float f = exp2_fast(x.x - mm);
      sum += x.y * f;
      acc += *reinterpret_cast<const F4*>(ow + (w * 16 + row) * kRowF + d) * f;
    }
    const int rr = row0 + row;
    if (part >= 0) {
      const int64_t at = ((int64_t)part * a.kv_heads + kvh) * kAttnTileFew + row;
      *reinterpret_cast<F4*>(a.part_o + at * kDim + d) = acc;
      if (d == 0) a.part_ml[at] = make_float2(mm, sum);
    } else if (rr < total && d < a.dim) {
      const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
      const int at = (int)((unsigned)rr / (unsigned)a.group);
      char* p = const_cast<char*>(a.o.data) + (q_row + at) * a.o.row + (int64_t)(kvh * a.group + rr - at * a.group) * a.o.head;
      const F2 x = {acc.x * inv, acc.y * inv}, y = {acc.z * inv, acc.w * inv};
      const V2 c = __builtin_convertvector(x, V2), g = __builtin_convertvector(y, V2);
      *reinterpret_cast<uint2*>(p + 2 * d) = make_uint2(__builtin_bit_cast(uint32_t, c), __builtin_bit_cast(uint32_t, g));
    }
  }
}

// ---- pieces added up ---------------------------------------------------------------------

// A workgroup per packed row, 2 channels a lane: each wave adds every fourth piece up, relative
// to the row's largest reference exponent, and the first wave the four sums.  Bound by latency: 4 us for
// one token over 45,000 keys, 9 us for 300 queries (16/4 and 8 heads of 128).
template <typename T, int NT, int TILE>
__global__ __launch_bounds__(256) void sfe_attn_join_kernel(AttnArgs a) {
  typedef typename Mat<T>::V2 V2;
  constexpr int kDim = 32 * NT;
  __shared__ float2 part[4][64];
  __shared__ float sums[4];
  const int64_t jk = blockIdx.x / TILE;
  const int row = (int)(blockIdx.x % TILE), kvh = (int)(jk % a.kv_heads);
  const int lane = (int)(threadIdx.x & 63), wave = (int)(threadIdx.x >> 6);
  const AttnJoin j = a.joins[jk / a.kv_heads];
  const int rr = j.row0 + row;
  if (rr >= j.lq * a.group) return;
  // piece p of the row is at at0 + p * step
  const int64_t at0 = ((int64_t)j.part0 * a.kv_heads + kvh) * TILE + row, step = (int64_t)a.kv_heads * TILE;
  float m = kNever;
  for (int p = lane; p < j.parts; p += 64) m = fmaxf(m, a.part_ml[at0 + p * step].x);
  m = max_halves(m);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  float x = 0.0f, y = 0.0f, sum = 0.0f;
#pragma unroll 8
  for (int p = wave; p < j.parts; p += 4) {
    const int64_t at = at0 + p * step;
    const float2 ml = a.part_ml[at];
    // (a piece that saw nothing: all zeros)
    const float f = ml.x == kNever && ml.y == 0.0f ? 0.0f : exp2_fast(ml.x - m);
    sum += ml.y * f;
    float2 v = make_float2(0.0f, 0.0f);
    if (2 * lane < kDim) v = *reinterpret_cast<const float2*>(a.part_o + at * kDim + 2 * lane);
    x += v.x * f;
    y += v.y * f;
  }
  part[wave][lane] = make_float2(x, y);
  if (lane == 0) sums[wave] = sum;
  __syncthreads();
  if (wave > 0 || 2 * lane >= a.dim) return;
  x = (part[0][lane].x + part[1][lane].x) + (part[2][lane].x + part[3][lane].x);
  y = (part[0][lane].y + part[1][lane].y) + (part[2][lane].y + part[3][lane].y);
  sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
  const float inv = sum > 0.0f || sum != sum ? 1.0f / sum : 0.0f;
  const int at = (int)((unsigned)rr / (unsigned)a.group);
  char* p = const_cast<char*>(a.o.data) + (j.q_row + at) * a.o.row + (int64_t)(kvh * a.group + rr - at * a.group) * a.o.head;
  const F2 v = {x * inv, y * inv};
  *reinterpret_cast<V2*>(p + 4 * lane) = __builtin_convertvector(v, V2);
}

template <typename T, int NT, int FORM>
hipError_t run_form(const AttnArgs& a, int cus, hipStream_t stream) {
  int64_t per = 0;  // units of an XCD at most
  for (int x = 0; x < 8; ++x) per = std::max<int64_t>(per, a.share[x + 1] - a.share[x]);
  const dim3 blocks((unsigned)(8 * per));
  constexpr int kTile = FORM == kAttnTall ? kAttnTileTall : (FORM == kAttnRows ? kAttnTileRows : kAttnTileFew);
  if constexpr (FORM == kAttnTall) {
    if (a.mask)
      sfe_attn_tall_kernel<T, NT, true><<<blocks, dim3(512), 0, stream>>>(a);
    else
      sfe_attn_tall_kernel<T, NT, false><<<blocks, dim3(512), 0, stream>>>(a);
  } else if constexpr (FORM == kAttnRows) {
    const int64_t slots = cus / 8 * (NT == 2 ? 3 : 2), wgs = per <= 2 * slots ? per : (per + kRowsUnits - 1) / kRowsUnits;
    const dim3 few((unsigned)(8 * wgs));
    if (a.mask)
      sfe_attn_rows_kernel<T, NT, true><<<few, dim3(256), 0, stream>>>(a);
    else
      sfe_attn_rows_kernel<T, NT, false><<<few, dim3(256), 0, stream>>>(a);
  } else {
    if (a.mask)
      sfe_attn_few_kernel<T, NT, true><<<blocks, dim3(64 * kAttnWavesFew), 0, stream>>>(a);
    else
      sfe_attn_few_kernel<T, NT, false><<<blocks, dim3(64 * kAttnWavesFew), 0, stream>>>(a);
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.n_joins) return e;
  sfe_attn_join_kernel<T, NT, kTile>
      <<<dim3((unsigned)((int64_t)a.n_joins * a.kv_heads * kTile)), dim3(256), 0, stream>>>(a);
  return hipGetLastError();
}

template <typename T, int FORM>
hipError_t run_dim(const AttnArgs& a, int cus, hipStream_t stream) {
  switch (attn_padded_dim(a.dim)) {
    case 64:
      if constexpr (FORM == kAttnTall) return hipErrorInvalidValue;  // (the plan takes the rows form)
      else return run_form<T, 2, FORM>(a, cus, stream);
    case 96: return run_form<T, 3, FORM>(a, cus, stream);
    default: return run_form<T, 4, FORM>(a, cus, stream);
  }
}

template <typename T>
hipError_t run(const AttnArgs& a, int form, int cus, hipStream_t stream) {
  if (form == kAttnTall) return run_dim<T, kAttnTall>(a, cus, stream);
  return form == kAttnRows ? run_dim<T, kAttnRows>(a, cus, stream) : run_dim<T, kAttnFew>(a, cus, stream);
}

}  // namespace

hipError_t launch_attn_mask(const uint8_t* mask, int64_t keys, uint64_t* words, hipStream_t stream) {
  const int64_t n = attn_mask_words(keys);
  return for_launches((n + 3) / 4, 256, [&](int64_t first, unsigned blocks) {
    sfe_attn_mask_kernel<<<dim3(blocks), dim3(256), 0, stream>>>(mask + 256 * first, keys - 256 * first, words + 4 * first, n - 4 * first);
    return hipGetLastError();
  });
}

hipError_t launch_attn_zero(const AttnTensor& out, int heads, int dim, int64_t first, int64_t last, int64_t rows,
                            hipStream_t stream) {
  const int chunks = dim / 8;
  const int64_t total = (first + rows - last) * heads * chunks;
  return for_launches((total + 255) / 256, 256, [&](int64_t block, unsigned blocks) {
    sfe_attn_zero_kernel<<<dim3(blocks), dim3(256), 0, stream>>>(out, heads, chunks, first, last, 256 * block, total);
    return hipGetLastError();
  });
}

hipError_t launch_attn(const AttnArgs& a, int form, int type, int cus, hipStream_t stream) {
  return type == kOpBf16 ? run<Bf>(a, form, cus, stream) : run<Hf>(a, form, cus, stream);
}

}  // namespace sfe
