// A paged cache's write and read.
//
// New token i of n of a sequence of `length` tokens is at length - n + i, in the page that the sequence's
// table names; a record (one kv head of a page) holds its tokens' K rows, V rows and scales
// together (sfe_decode.hpp).
//
// Bound by memory: every element is read and written once, a workgroup's rows lie next to each other in both.  Written, 205,000
// tokens of 4 heads of 128 from bf16 to e4m3: 636 MB in 135 us (4.7 TB/s; bf16 to bf16 5.2), read back 128 (5.0; 5.4), 256 clips of 13-251 tokens of 8 heads
// of 64 in f16 18.5 us and read back 12.7 (5.7 and 8 TB/s, part of it in the last-level cache); 8 prompts of 700-8,192
// tokens in int8 read in 36 us (5.3 TB/s).  A thread keeps its place in four tokens (clips written and read 37 us with a
// token a thread, 31 with four and codes by one product).
//
// Codes are x M / a to the nearest, halves to the even one, a the row's largest magnitude.  Let x, a of 16 bits be
// whole numbers below 2^11 times powers of two.  A point p halfway between two codes (5 bits in e4m3, 8 in int8) differs from
// x M / a by nothing, or by 2^-19 of it at least: x M and p a are whole numbers below 2^19 times powers of two.  A product
// of x and M times a's reciprocal is off by 4 of 24 bits' last steps at most (reciprocal 2, two roundings 1 each): rounded to
// multiples of 16 of them it is p itself where it should be, and on the right side of p elsewhere (12 of
// them away at least).  For x of 32 bits the quotient is rounded correctly first: x M is exact up to its one
// rounding after a power of two is taken off a, and one division's remainder corrects it.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "sfe_cache.hpp"
#include "sfe_internal.hpp"

namespace sfe {
namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 4;  // of a thread

template <typename T>
struct alignas(16) Eight {
  T v[8];
};

template <int CTRL>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, 0xf, 0xf, true);
}
// The largest of `lanes` lanes (1, 2, 4, 8 or 16).
__device__ __forceinline__ uint32_t group_max(uint32_t x, int lanes) {
  if (lanes > 1) x = max(x, dpp<0xb1>(x));
  if (lanes > 2) x = max(x, dpp<0x4e>(x));
  if (lanes > 4) x = max(x, dpp<0x141>(x));
  if (lanes > 8) x = max(x, dpp<0x140>(x));
  return x;
}

// 8 codes of x, values of T; top the bits of the row's largest magnitude; *scale: the row's.
template <typename T, int TYPE>
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], uint32_t top, float* scale) {
  constexpr float M = Kept<TYPE>::kTop, kPart = 1.0f / M;
  if (top >= 0x7f800000u) {
    *scale = __uint_as_float(0x7fc00000u);
    return make_uint2(0, 0);
  }
  top = max(top, 0x0f800000u);  // 2^-96
  // (quotients by a reciprocal, corrected by their remainders)
  const float most = __uint_as_float(top), part = most * kPart;
  *scale = __builtin_fmaf(__builtin_fmaf(-part, M, most), kPart, part);
  // M over the power of two of the largest (from 2^-96 up: no more than 2^105, no less than 2^-121)
  const float c = __builtin_amdgcn_ldexpf(M, 127 - (int)(top >> 23));
  const float a = __uint_as_float((top & 0x7fffffu) | 0x3f800000u);
  float y[8];
  if constexpr (sizeof(T) == 2) {
    const float m = c * __builtin_amdgcn_rcpf(a);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = __uint_as_float((__float_as_uint(x[i] * m) + 8u) & ~15u);
  } else {
    const float r = 1.0f / a;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float n = x[i] * c;
      const float guess = n * r;
      y[i] = __builtin_fmaf(__builtin_fmaf(-guess, a, n), r, guess);
    }
  }
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (TYPE == kCacheE4m3) {
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i], y[4 * i + 1], 0, false);
      w[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[4 * i + 2], y[4 * i + 3], p, true);
    } else {
      // (1.5 * 2^23 more: the sum is rounded to a whole number, its low byte the code)
      uint32_t b[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) b[j] = __float_as_uint(y[4 * i + j] + 12582912.0f);
      w[i] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0c0c0400), __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400), 0x05040100);
    }
  }
  return make_uint2(w[0], w[1]);
}

// The bits of the largest magnitude of 8 values as f32 (magnitudes order as their bits do, infinity and NaN last).
template <typename T>
__device__ __forceinline__ uint32_t top_of(const Eight<T>& x) {
  if constexpr (sizeof(T) == 2) {
    typedef unsigned short Pair __attribute__((ext_vector_type(2)));
    const uint4 w = __builtin_bit_cast(uint4, x);
    auto bits = [](uint32_t v) { return __builtin_bit_cast(Pair, v & 0x7fff7fffu); };
    const Pair m = __builtin_elementwise_max(__builtin_elementwise_max(bits(w.x), bits(w.y)),
                                             __builtin_elementwise_max(bits(w.z), bits(w.w)));
    return max((uint32_t)m.x, (uint32_t)m.y);
  } else {
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x.v[e]) & 0x7fffffffu);
    return top;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t top_bits(uint32_t top) {
  if constexpr (sizeof(T) == 2) return __float_as_uint((float)__builtin_bit_cast(T, (unsigned short)top));
  else return top;
}

// Value of code i of 8.
template <int TYPE>
__device__ __forceinline__ float code_value(uint2 w, int i) {
  const uint32_t x = i < 4 ? w.x : w.y;
  if constexpr (TYPE == kCacheE4m3) {
    switch (i & 3) {
      case 0: return __builtin_amdgcn_cvt_f32_fp8((int)x, 0);
      case 1: return __builtin_amdgcn_cvt_f32_fp8((int)x, 1);
      case 2: return __builtin_amdgcn_cvt_f32_fp8((int)x, 2);
      default: return __builtin_amdgcn_cvt_f32_fp8((int)x, 3);
    }
  } else {
    return (float)(int8_t)(x >> (8 * (i & 3)));
  }
}

// A workgroup's part of a tile, and a thread's place in its tokens' rows: `lanes` lanes of 8 channels for each of the K and V
// heads, laid end to end.  A thread keeps its place in kTokens tokens, so that what depends on the place is
// computed once; where a tile's tokens lie (16 of them, in two pages at most) is scalar.
struct Shape {
  int places, lanes, per, by_place, by_token;  // per: tokens of a pass; by_...: workgroups of a tile
};
struct Part {
  CacheTile tile;
  int position;           // of the tile's first token
  int64_t page[2];        // that it is in, and the next
  char* record[2];        // of the thread's kv head in them
  int token, kvh, channel;
  bool value, in;         // V; whether the thread has channels
  __device__ __forceinline__ Part(const CacheArgs& c, const Shape& s, int64_t first_tile, uint32_t first) {
    typedef const __attribute__((address_space(4))) CacheTile* Tiles;
    const int of_tile = s.by_place * s.by_token, t = (int)threadIdx.x;
    const uint32_t block = first + blockIdx.x, at = block / (uint32_t)of_tile;
    const int rest = (int)(block - at * of_tile), chunk = (int)((uint32_t)rest / (uint32_t)s.by_token);
    const Tiles p = (Tiles)(uintptr_t)c.tiles + (first_tile + at);
    tile.first = p->first, tile.seq = p->seq, tile.n = p->n, tile.at = p->at, tile.count = p->count;
    const int length = c.lengths[tile.seq];
    position = __builtin_amdgcn_readfirstlane(max(length, 0) - tile.n + tile.at);
    const int pass = s.per > 1 ? (int)((unsigned)t / (unsigned)s.places) : 0;
    const int place = s.per > 1 ? t - pass * s.places : chunk * kThreads + t;
    token = (rest - chunk * s.by_token) * kTokens * s.per + pass;
    const int head = (int)((unsigned)place / (unsigned)s.lanes);
    channel = 8 * (place - head * s.lanes);
    value = head >= c.kv_heads;
    kvh = value ? head - c.kv_heads : head;
    in = place < s.places && pass < s.per && channel < c.dim;
  }
  __device__ __forceinline__ void look_up(const CacheArgs& c) {
    const int64_t from = (position >> c.shift) * ((int64_t)1 << c.shift);
    page[0] = page_of(c, tile.seq, position < 0 ? -1 : position);
    page[1] = page_of(c, tile.seq, from + (1 << c.shift));
    const int64_t in_page = kvh * c.record;
    for (int i = 0; i < 2; ++i) record[i] = c.data + page[i] * c.kv_heads * c.record + in_page;
  }
  // The codes of token i's place and its scale; null where the cache has none.
  template <int TYPE>
  __device__ __forceinline__ char* codes_at(const CacheArgs& c, int i, float** scale) const {
    const int at = (position & ((1 << c.shift) - 1)) + i, next = at >> c.shift;
    if ((next ? page[1] : page[0]) < 0) return nullptr;
    const int slot = at & ((1 << c.shift) - 1), part = Kept<TYPE>::kSize * c.dim << c.shift;
    char* in = next ? record[1] : record[0];
    *scale = reinterpret_cast<float*>(in + (uint32_t)(2 * part + (value ? 4 << c.shift : 0) + 4 * slot));
    return in + (uint32_t)((value ? part : 0) + Kept<TYPE>::kSize * (slot * c.dim + channel));
  }
};
template <typename T>
__device__ __forceinline__ const char* row_at(const Part& p, const AttnTensor& k, const AttnTensor& v, int64_t* row) {
  *row = p.value ? v.row : k.row;
  return (p.value ? v.data : k.data) + (p.tile.first + p.tile.at) * *row + p.kvh * (p.value ? v.head : k.head) + (int64_t)sizeof(T) * p.channel;
}

template <typename T, int TYPE>
__global__ __launch_bounds__(kThreads) void sfe_cache_write_kernel(CacheArgs c, AttnTensor k, AttnTensor v, int64_t first_tile, uint32_t first, Shape shape) {
  Part p(c, shape, first_tile, first);
  int64_t row;
  const char* from = row_at<T>(p, k, v, &row);
  Eight<T> x[kTokens];
#pragma unroll
  for (int j = 0; j < kTokens; ++j) {
    const int i = p.token + j * shape.per;
    x[j] = Eight<T>{};
    if (p.in && i < p.tile.count) x[j] = *reinterpret_cast<const Eight<T>*>(from + i * row);
  }
  p.look_up(c);
#pragma unroll
  for (int j = 0; j < kTokens; ++j) {
    const int i = p.token + j * shape.per;
    float f[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)x[j].v[e];
    float* scale;
    uint32_t top = 0;
    if constexpr (Kept<TYPE>::kSize == 1) top = top_bits<T>(group_max(top_of(x[j]), shape.lanes));
    if (!p.in || i >= p.tile.count) continue;
    char* to = p.codes_at<TYPE>(c, i, &scale);
    if (!to) continue;
    if constexpr (Kept<TYPE>::kSize == 1) {
      float s;
      *reinterpret_cast<uint2*>(to) = codes_of<T, TYPE>(f, top, &s);
      if (p.channel == 0) *scale = s;
    } else {
      typedef typename std::conditional<TYPE == kCacheBf16, __bf16, _Float16>::type O;
      Eight<O> y;
#pragma unroll
      for (int e = 0; e < 8; ++e) y.v[e] = (O)f[e];
      *reinterpret_cast<Eight<O>*>(to) = y;
    }
  }
}

template <typename T, int TYPE>
__global__ __launch_bounds__(kThreads) void sfe_cache_read_kernel(CacheArgs c, AttnTensor k, AttnTensor v, int64_t first_tile, uint32_t first, Shape shape) {
  Part p(c, shape, first_tile, first);
  p.look_up(c);
  int64_t row;
  char* to = const_cast<char*>(row_at<T>(p, k, v, &row));
  uint4 w[kTokens];
  float s[kTokens];
#pragma unroll
  for (int j = 0; j < kTokens; ++j) {
    const int i = p.token + j * shape.per;
    w[j] = make_uint4(0, 0, 0, 0);
    s[j] = 0.0f;
    if (!p.in || i >= p.tile.count) continue;
    float* scale;
    const char* from = p.codes_at<TYPE>(c, i, &scale);
    if (!from) continue;
    if constexpr (Kept<TYPE>::kSize == 1) {
      const uint2 x = *reinterpret_cast<const uint2*>(from);
      w[j].x = x.x, w[j].y = x.y;
      s[j] = *scale;
    } else {
      w[j] = *reinterpret_cast<const uint4*>(from);
    }
  }
#pragma unroll
  for (int j = 0; j < kTokens; ++j) {
    const int i = p.token + j * shape.per;
    if (!p.in || i >= p.tile.count) continue;
    Eight<T> y;
    if constexpr (Kept<TYPE>::kSize == 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y.v[e] = (T)(code_value<TYPE>(make_uint2(w[j].x, w[j].y), e) * s[j]);
    } else {
      typedef typename std::conditional<TYPE == kCacheBf16, __bf16, _Float16>::type O;
      const Eight<O> x = __builtin_bit_cast(Eight<O>, w[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) y.v[e] = (T)(float)x.v[e];
    }
    *reinterpret_cast<Eight<T>*>(to + i * row) = y;
  }
}

template <typename T, int TYPE, bool WRITE>
hipError_t run(const CacheArgs& c, const AttnTensor& k, const AttnTensor& v, hipStream_t stream) {
  Shape s;
  s.lanes = 2;
  while (8 * s.lanes < c.dim) s.lanes *= 2;
  s.places = 2 * c.kv_heads * s.lanes;
  s.by_place = (s.places + kThreads - 1) / kThreads;
  s.per = s.by_place > 1 ? 1 : kThreads / s.places;
  s.by_token = (c.most + kTokens * s.per - 1) / (kTokens * s.per);
  const int of_tile = s.by_place * s.by_token;
  return for_launches((int64_t)c.n_tiles * of_tile, kThreads, [&](int64_t at, unsigned blocks) {
    const int64_t tile = at / of_tile;
    const uint32_t first = (uint32_t)(at % of_tile);
    if (WRITE) sfe_cache_write_kernel<T, TYPE><<<dim3(blocks), dim3(kThreads), 0, stream>>>(c, k, v, tile, first, s);
    else sfe_cache_read_kernel<T, TYPE><<<dim3(blocks), dim3(kThreads), 0, stream>>>(c, k, v, tile, first, s);
    return hipGetLastError();
  });
}

template <typename T, bool WRITE>
hipError_t run_type(const CacheArgs& c, int type, const AttnTensor& k, const AttnTensor& v, hipStream_t stream) {
  switch (type) {
    case kCacheBf16: return run<T, kCacheBf16, WRITE>(c, k, v, stream);
    case kCacheF16: return run<T, kCacheF16, WRITE>(c, k, v, stream);
    case kCacheE4m3: return run<T, kCacheE4m3, WRITE>(c, k, v, stream);
    default: return run<T, kCacheInt8, WRITE>(c, k, v, stream);
  }
}

template <bool WRITE>
hipError_t run_dtype(const CacheArgs& c, int type, const AttnTensor& k, const AttnTensor& v, int dtype, hipStream_t stream) {
  if (dtype == kOpF32) return run_type<float, WRITE>(c, type, k, v, stream);
  if (dtype == kOpBf16) return run_type<__bf16, WRITE>(c, type, k, v, stream);
  return run_type<_Float16, WRITE>(c, type, k, v, stream);
}

}  // namespace

hipError_t launch_cache_write(const CacheArgs& c, int type, const AttnTensor& k, const AttnTensor& v, int dtype, hipStream_t stream) {
  return run_dtype<true>(c, type, k, v, dtype, stream);
}

hipError_t launch_cache_read(const CacheArgs& c, int type, const AttnTensor& k, const AttnTensor& v, int dtype, hipStream_t stream) {
  return run_dtype<false>(c, type, k, v, dtype, stream);
}

}  // namespace sfe
