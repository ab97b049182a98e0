// A paged cache's write and read.
//
// New token i of n of a sequence of `length` tokens is at length - n + i, in the page that the sequence's
// table names; a record (one kv head of a page) holds its tokens' K rows, V rows and scales
// together (sfe_decode.hpp).  The quotient x M / a is rounded correctly before it is rounded to a
// code (x M is exact for 16-bit x after a power of two is taken off a, one division's remainder
// corrects it), so that values halfway between two codes go to the even one.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "sfe_cache.hpp"
#include "sfe_internal.hpp"

namespace sfe {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;  // of a thread

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

// 8 codes of x, top the bits of the row's largest magnitude; *scale: the row's.
template <int TYPE>
__device__ __forceinline__ uint2 codes_of(const float (&x)[8], uint32_t top, float* scale) {
  constexpr float M = Kept<TYPE>::kTop;
  if (top >= 0x7f800000u) {
    *scale = __uint_as_float(0x7fc00000u);
    return make_uint2(0, 0);
  }
  top = max(top, 0x0f800000u);  // 2^-96
  *scale = __uint_as_float(top) / M;
  // M over the power of two of the largest (from 2^-96 up: no more than 2^105, no less than 2^-121)
  const float c = __builtin_amdgcn_ldexpf(M, 127 - (int)(top >> 23));
  const float a = __uint_as_float((top & 0x7fffffu) | 0x3f800000u), r = 1.0f / a;
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float n = x[i] * c;
    const float guess = n * r;
    y[i] = __builtin_fmaf(__builtin_fmaf(-guess, a, n), r, guess);
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

// What a thread does of a tile: a unit is a row of a token, one of K and V, and a kv head, of `lanes` lanes of 8
// channels each.
struct Place {
  int64_t row;      // packed
  int64_t token;    // of its sequence
  int64_t page;     // or -1
  int32_t slot, kvh;
  bool value, in;   // V; whether the lane has channels
};
__device__ __forceinline__ Place place_of(const CacheArgs& c, const CacheTile& tile, int unit, int channel, int length) {
  Place p;
  const int both = 2 * c.kv_heads;
  const int token = (int)((unsigned)unit / (unsigned)both), part = unit - token * both;
  p.value = part >= c.kv_heads;
  p.kvh = p.value ? part - c.kv_heads : part;
  p.in = token < tile.count && channel < c.dim;
  p.row = tile.first + tile.at + token;
  p.token = (int64_t)length - tile.n + tile.at + token;
  p.page = -1;
  p.slot = (int)(p.token & ((1 << c.shift) - 1));
  return p;
}
template <int TYPE>
__device__ __forceinline__ char* codes_at(const CacheArgs& c, const Place& p, int channel, float** scale) {
  char* record = c.data + (p.page * c.kv_heads + p.kvh) * c.record;
  const int64_t part = (int64_t)Kept<TYPE>::kSize * c.dim << c.shift;
  *scale = reinterpret_cast<float*>(record + 2 * part) + ((int64_t)p.value << c.shift) + p.slot;
  return record + (p.value ? part : 0) + (int64_t)Kept<TYPE>::kSize * (p.slot * c.dim + channel);
}

template <typename T, int TYPE>
__global__ __launch_bounds__(kThreads) void sfe_cache_write_kernel(CacheArgs c, AttnTensor k, AttnTensor v, int64_t first, int chunks,
                                                                   int lanes) {
  const int64_t block = first + blockIdx.x, at_tile = block / chunks;
  const CacheTile tile = c.tiles[at_tile];
  const int length = c.lengths[tile.seq];
  const int groups = kThreads / lanes, group = (int)threadIdx.x / lanes, channel = 8 * ((int)threadIdx.x - group * lanes);
  const int unit0 = (int)(block - at_tile * chunks) * kUnits * groups + group;
  Place p[kUnits];
  Eight<T> x[kUnits];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    p[j] = place_of(c, tile, unit0 + j * groups, channel, length);
    x[j] = Eight<T>{};
    const char* from = p[j].value ? v.data + p[j].row * v.row + p[j].kvh * v.head : k.data + p[j].row * k.row + p[j].kvh * k.head;
    if (p[j].in) x[j] = *reinterpret_cast<const Eight<T>*>(from + (int64_t)sizeof(T) * channel);
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j)
    if (p[j].in) p[j].page = page_of(c, tile.seq, p[j].token);
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    float f[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (float)x[j].v[i];
    float* scale;
    if constexpr (TYPE == kCacheE4m3 || TYPE == kCacheInt8) {
      uint32_t top = 0;  // (magnitudes order as their bits do, infinity and NaN last)
#pragma unroll
      for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(f[i]) & 0x7fffffffu);
      top = group_max(top, lanes);
      if (p[j].page < 0) continue;
      char* to = codes_at<TYPE>(c, p[j], channel, &scale);
      float s;
      *reinterpret_cast<uint2*>(to) = codes_of<TYPE>(f, top, &s);
      if (channel == 0) *scale = s;
    } else {
      if (p[j].page < 0) continue;
      char* to = codes_at<TYPE>(c, p[j], channel, &scale);
      typedef typename std::conditional<TYPE == kCacheBf16, __bf16, _Float16>::type O;
      Eight<O> y;
#pragma unroll
      for (int i = 0; i < 8; ++i) y.v[i] = (O)f[i];
      *reinterpret_cast<Eight<O>*>(to) = y;
    }
  }
}

template <typename T, int TYPE>
__global__ __launch_bounds__(kThreads) void sfe_cache_read_kernel(CacheArgs c, AttnTensor k, AttnTensor v, int64_t first, int chunks,
                                                                  int lanes) {
  const int64_t block = first + blockIdx.x, at_tile = block / chunks;
  const CacheTile tile = c.tiles[at_tile];
  const int length = c.lengths[tile.seq];
  const int groups = kThreads / lanes, group = (int)threadIdx.x / lanes, channel = 8 * ((int)threadIdx.x - group * lanes);
  const int unit0 = (int)(block - at_tile * chunks) * kUnits * groups + group;
  Place p[kUnits];
  uint4 w[kUnits];
  float s[kUnits];
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    p[j] = place_of(c, tile, unit0 + j * groups, channel, length);
    if (p[j].in) p[j].page = page_of(c, tile.seq, p[j].token);
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    w[j] = make_uint4(0, 0, 0, 0);
    s[j] = 0.0f;
    if (p[j].page < 0) continue;
    float* scale;
    const char* from = codes_at<TYPE>(c, p[j], channel, &scale);
    if constexpr (Kept<TYPE>::kSize == 1) {
      const uint2 x = *reinterpret_cast<const uint2*>(from);
      w[j].x = x.x, w[j].y = x.y;
      s[j] = *scale;
    } else {
      w[j] = *reinterpret_cast<const uint4*>(from);
    }
  }
#pragma unroll
  for (int j = 0; j < kUnits; ++j) {
    if (!p[j].in) continue;
    Eight<T> y;
    if constexpr (Kept<TYPE>::kSize == 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y.v[i] = (T)(code_value<TYPE>(make_uint2(w[j].x, w[j].y), i) * s[j]);
    } else {
      typedef typename std::conditional<TYPE == kCacheBf16, __bf16, _Float16>::type O;
      const Eight<O> x = __builtin_bit_cast(Eight<O>, w[j]);
#pragma unroll
      for (int i = 0; i < 8; ++i) y.v[i] = (T)(float)x.v[i];
    }
    const char* to = p[j].value ? v.data + p[j].row * v.row + p[j].kvh * v.head : k.data + p[j].row * k.row + p[j].kvh * k.head;
    *reinterpret_cast<Eight<T>*>(const_cast<char*>(to) + (int64_t)sizeof(T) * channel) = y;
  }
}

template <typename T, int TYPE, bool WRITE>
hipError_t run(const CacheArgs& c, const AttnTensor& k, const AttnTensor& v, hipStream_t stream) {
  int lanes = 2;
  while (8 * lanes < c.dim) lanes *= 2;
  const int units = kCacheTileTokens * 2 * c.kv_heads, each = kUnits * (kThreads / lanes);
  const int chunks = (units + each - 1) / each;
  return for_launches((int64_t)c.n_tiles * chunks, kThreads, [&](int64_t first, unsigned blocks) {
    if (WRITE) sfe_cache_write_kernel<T, TYPE><<<dim3(blocks), dim3(kThreads), 0, stream>>>(c, k, v, first, chunks, lanes);
    else sfe_cache_read_kernel<T, TYPE><<<dim3(blocks), dim3(kThreads), 0, stream>>>(c, k, v, first, chunks, lanes);
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
