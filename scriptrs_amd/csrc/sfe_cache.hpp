// Where a token lies in a paged cache, and how its values are kept (sfe_cache.hip, sfe_cache_attn.hip).
//
// Codes of 8 bits: with a the largest magnitude of a token's channels in one kv head (at least
// 2^-96) and M the largest code (448 in e4m3, 127 in int8), code = rne(x M / a) and
// scale = a / M; a code stands for code * scale.  A row that is not finite has the scale NaN: all of it reads
// as NaN.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "sfe_decode.hpp"

namespace sfe {

template <int TYPE>
struct Kept;  // element types of a cache
template <>
struct Kept<kCacheBf16> {
  static constexpr int kSize = 2;
};
template <>
struct Kept<kCacheF16> {
  static constexpr int kSize = 2;
};
template <>
struct Kept<kCacheE4m3> {
  static constexpr int kSize = 1;
  static constexpr float kTop = 448.0f;
};
template <>
struct Kept<kCacheInt8> {
  static constexpr int kSize = 1;
  static constexpr float kTop = 127.0f;
};

// The page of a sequence's token, or -1 where the cache has none: before its first, past the
// table, or in a page that is none of the cache's.
__host__ __device__ __forceinline__ int64_t page_of(const CacheArgs& c, int seq, int64_t token) {
  const int64_t column = token >> c.shift;
  if (token < 0 || column >= c.table_pages) return -1;
  const int32_t page = c.table[seq * c.table_row + column];
  return page < 0 || page >= c.pages ? -1 : page;
}

}  // namespace sfe
