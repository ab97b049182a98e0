// Operators of a decoder's step over a paged cache (head norms with rotary
// positions, the cache's write and read, attention of new tokens over it, and the steering of
// logits): what their entry points (sfe_decode.cpp) share with their kernels.
#pragma once

#include <algorithm>

#include "sfe_ops.hpp"

namespace sfe {

// ---- norms of heads and rotary positions in one pass (sfe_norm_rotary.hip) -----------
constexpr int kNormRotaryMaxDim = 256;
struct NormRotaryArgs {
  uint64_t step[kRotaryMaxPairs];  // turns a position, as a fraction of 2^64
  RotaryTensor t[2];
  const float* weight[2];  // [dim], or null
  const int32_t* positions;
  int64_t rows;
  int32_t dim, rotary;
  float magnitude, eps;
};
hipError_t launch_norm_rotary(const NormRotaryArgs& a, int type, bool interleaved, bool layer, int cus, hipStream_t stream);

// ---- the paged cache (sfe_cache.hip) ----------------------------------------------------
// Element types of a cache: sfe_dtype's 16-bit ones, then codes of 8 bits with an f32
// scale for each token and kv head.
enum CacheType { kCacheBf16 = 1, kCacheF16 = 2, kCacheE4m3 = 3, kCacheInt8 = 4 };
constexpr bool cache_coded(int type) { return type == kCacheE4m3 || type == kCacheInt8; }
constexpr int kCacheMaxDim = 128;
// A record, one kv head's part of a page: K [page][dim], V [page][dim], then for codes their
// scales, f32 K [page] and V [page].
inline int64_t cache_record(int page, int dim, int type) {
  return (int64_t)2 * page * dim * (cache_coded(type) ? 1 : 2) + (cache_coded(type) ? 8 * page : 0);
}

// Tokens of one sequence: its new tokens are the last n of `lengths[seq]`.
struct CacheTile {
  int64_t first;  // packed row of the sequence's first new token
  int32_t seq, n;
  int32_t at, count;  // write, read: tokens [at, at + count); attention: packed rows (token x head of a group) from `at` on
};
static_assert(sizeof(CacheTile) == 24, "layout shared with the kernels");
constexpr int kCacheTileTokens = 16;

struct CacheArgs {
  char* data;  // [pages][kv_heads][record]
  int64_t pages, record;
  const int32_t* table;  // [sequences][table_pages], rows table_row apart
  const int32_t* lengths;
  const CacheTile* tiles;
  int64_t table_row;
  int32_t n_tiles, most, table_pages, shift, kv_heads, dim;  // most: tokens of a tile; shift: log2 of the page's size
};
hipError_t launch_cache_write(const CacheArgs& c, int type, const AttnTensor& k, const AttnTensor& v, int dtype, hipStream_t stream);
hipError_t launch_cache_read(const CacheArgs& c, int type, const AttnTensor& k, const AttnTensor& v, int dtype, hipStream_t stream);

// ---- attention of new tokens over the cache (sfe_cache_attn.hip) ---------------------------
// A workgroup's waves, and the keys of a wave's step; tokens of a page table at most.
constexpr int kCacheAttnWaves = 4, kCacheAttnStep = 32;
constexpr int64_t kCacheAttnKeys = (int64_t)1 << 30;
// Tiles of 16 packed rows of a workgroup: 1 or 2 in each wave, all of whose waves take other keys; 4 and 8, of which two
// and four waves read the same keys.
inline int cache_attn_tiles(int64_t rows) { return rows <= 16 ? 1 : (rows <= 32 ? 2 : (rows <= 64 ? 4 : 8)); }
inline int cache_attn_round(int tiles) { return kCacheAttnStep * kCacheAttnWaves / (tiles <= 2 ? 1 : tiles / 2); }  // keys
// Whether each workgroup takes a whole unit (a tile and kv head), or an equal share of all units' rounds, which are then
// joined by a second launch.  A unit alone takes 0.9 us a round, 1.2 of shared steps; shares cost 5 us more, and divide what
// the device takes for all of it.  That is counted for a third of the table's tokens (`keys`), since lengths differ.  Measured (a
// call of ten in a graph), 16/4 heads of 128 in e4m3, one token of n sequences over l tokens, whole / shares: n 1, l 600
// 10.1 / 10.8 us, 1,200 15.2 / 12.6; n 32, 1,200 16.6 / 20.8, 4,800 46.2 / 37.9; n 64 of 600 to 4,800 47.1 / 41.6; n 128, 2,400
// 59.5 / 61.1, of 300 to 2,400 36.3 / 42.7; n 256 of 126 to 1,500 42.0 / 54.8.  16 tokens: n 1, 600 22.2 / 18.6; n 32, 600
// 23.7 / 34.9, 2,400 63.4 / 47.9; n 128, 2,400 98.5 / 100.2.  In bf16, one token: n 1, 600 10.0 / 10.0, 1,200 15.1 / 15.5; n 32, 1,200
// 18.1 / 28.5, 4,800 63.6 / 62.2; n 128, 2,400 114 / 118; n 256 of 126 to 1,500 82 / 92.
// Past 4,096 tokens one long sequence among short ones would keep the others waiting, but shares have every unit's length
// to look through: with thousands of units they are whole as long as that costs more than the longest unit alone can.
// Heads of 64: n 512 of 600 in a table of 5,000, 16 kv_heads 120 / 153, one of them of 60,000 tokens (and its table) 499 / 188; n
// 20,000 of 200 306 / 549; runs of new tokens: 64 of 1,024 over 6,000 6,265 / 9,309, one of 40,000 18,855 / 26,452, one of 16,384
// over 32,768 7,977 / 11,225 (4,096 units, which the rule shares).
inline bool cache_attn_whole(int64_t units, int64_t keys, int tiles, int esize) {
  const double rounds = (double)std::max<int64_t>(1, (keys + cache_attn_round(tiles) - 1) / cache_attn_round(tiles));
  const double alone = tiles <= 2 ? 0.92 : 1.24, all = std::max(0.0024 * esize, 0.002 * std::min(tiles, 4));
  if (keys > 4096) return units >= 8192 && alone * rounds <= 5.0 + (tiles <= 2 ? 0.0045 : 0.2) * (double)units;
  return alone * rounds <= 5.0 + all * (double)units * rounds;
}
inline int cache_attn_dim(int dim) { return dim <= 64 ? 64 : 128; }  // padded
inline int cache_attn_shares(int cus) { return 2 * ((cus + 7) / 8 * 8); }  // workgroups that share a call's rounds
struct CacheAttnArgs {
  CacheArgs c;  // tiles: of 16 * tiles packed rows (token x head of a group)
  AttnTensor q, o;
  const uint64_t* tree;  // bit j of a row: it sees new token j of its sequence; null: its own and those before
  float* part_o;    // [2 * shares][tile row][padded dim]
  float2* part_ml;  // [2 * shares][tile row]: (reference exponent, sum)
  int2* units;      // [tile][kv head]: the share of its first part, and its parts (0: not cut)
  int32_t group, tiles, rows, shares;  // rows: of a tile at most
  bool whole;       // a workgroup takes a whole unit
  float scale_log2;  // scale * log2(e)
};
hipError_t launch_cache_attn(const CacheAttnArgs& a, int type, int dtype, hipStream_t stream);

// ---- steering of logits (sfe_logits.hip) -----------------------------------------------------
// A row's tokens in spans, a workgroup each: vectors of n lie at multiples of their size, so that the first span
// begins `before` tokens (less than n) before the row.  There are as many spans as the row with the most before
// it needs: of another row the last one may begin at the vocabulary's end or past it, and has no tokens.
constexpr int logits_spans(int vocab, int n, int span) { return (int)(((int64_t)vocab + (n - 1) + span - 1) / span); }
struct LogitsSpan {
  int32_t first;    // token of its first place
  int32_t low;      // first token of the row that it has
  uint32_t tokens;  // that it has
  __host__ __device__ bool has(int32_t token) const { return (uint32_t)token - (uint32_t)low < tokens; }
  __host__ __device__ int32_t place(int32_t token) const { return token - first; }  // (of a token that it has)
};
__host__ __device__ inline LogitsSpan logits_span(int number, int span, int before, int vocab) {
  LogitsSpan s;
  s.first = number * span - before;
  s.low = s.first > 0 ? s.first : 0;
  const int end = s.first + span < vocab ? s.first + span : vocab;
  s.tokens = end > s.low ? (uint32_t)(end - s.low) : 0u;
  return s;
}
struct LogitsArgs {
  const char* in;
  char* out;
  int64_t in_row, out_row;  // strides in elements
  int32_t rows, vocab;
  const int32_t* history;  // or null
  const int32_t* lengths;  // or null: all of a row
  int64_t history_row;
  int32_t history_most;
  float repetition, presence, frequency;
  const float *repetitions, *presences, *frequencies;  // of each row, or null
  const float* bias;  // or null
  int64_t bias_row;
  const uint32_t* allowed;  // or null
  int64_t allowed_row;
  int32_t n_allowed;
  const int32_t* states;  // or null: row r takes mask r
};
hipError_t launch_logits(const LogitsArgs& a, int type, hipStream_t stream);

}  // namespace sfe
