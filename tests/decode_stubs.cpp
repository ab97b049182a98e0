// The launchers of a decoder's step (scriptrs_amd/csrc/sfe_decode.hpp), which launch nothing, and the cache's places on
// the host (sfe_cache.hpp): for tests without a GPU, linked with model_ops_stubs.cpp.
#include "sfe_cache.hpp"
#include "sfe_decode.hpp"

namespace sfe {
hipError_t launch_norm_rotary(const NormRotaryArgs&, int, bool, bool, int, hipStream_t) { return hipSuccess; }
hipError_t launch_cache_write(const CacheArgs&, int, const AttnTensor&, const AttnTensor&, int, hipStream_t) { return hipSuccess; }
hipError_t launch_cache_read(const CacheArgs&, int, const AttnTensor&, const AttnTensor&, int, hipStream_t) { return hipSuccess; }
hipError_t launch_cache_attn(const CacheAttnArgs&, int, int, hipStream_t) { return hipSuccess; }
hipError_t launch_logits(const LogitsArgs&, int, hipStream_t) { return hipSuccess; }
}  // namespace sfe

extern "C" int64_t stub_page_of(const int32_t* table, int64_t table_row, int32_t table_pages, int64_t pages, int32_t shift, int32_t seq,
                                int64_t token) {
  sfe::CacheArgs c{};
  c.table = table;
  c.table_row = table_row;
  c.table_pages = table_pages;
  c.pages = pages;
  c.shift = shift;
  return sfe::page_of(c, seq, token);
}
extern "C" int32_t stub_attn_tiles(int64_t rows) { return sfe::cache_attn_tiles(rows); }
extern "C" int32_t stub_attn_round(int32_t tiles) { return sfe::cache_attn_round(tiles); }
extern "C" int32_t stub_attn_whole(int64_t units, int64_t keys, int32_t tiles, int32_t esize) {
  return sfe::cache_attn_whole(units, keys, tiles, esize);
}
