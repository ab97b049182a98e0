// Entry points of a decoder's step over a paged cache (declared in include/scriptrs_fe.h):
// argument checks, the plan of new tokens, and the launches in their context's order.  All compute runs
// in sfe_norm_rotary.hip, sfe_cache.hip, sfe_cache_attn.hip and sfe_logits.hip.
#include <hip/hip_runtime.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <memory>
#include <vector>

#include "../../include/scriptrs_fe.h"
#include "sfe_checks.hpp"
#include "sfe_decode.hpp"

using sfe::apart;
using sfe::check_heads;
using sfe::guarded;
using sfe::known_dtype;
using sfe::kMaxStride;
using sfe::op_fail;
using sfe::Rows;
using sfe::rows_of;
using sfe::same_view;
using sfe::share;
using sfe::up;

struct sfe_cache_plan : sfe::OpPlan {
  ~sfe_cache_plan() { sfe::op_drop(this); }
  int32_t n = 0, heads = 0, kv_heads = 0, dim = 0;
  int64_t rows = 0, longest = 0;  // new tokens, and those of the sequence with the most
  int32_t n_tiles = 0, n_attn = 0, attn_tiles = 1;  // attn_tiles: tiles of 16 packed rows of an attention's tile
  size_t tiles = 0, attn = 0, part_o = 0, part_ml = 0, units = 0;  // offsets into buf
};

namespace {

int check_cache_shape(int32_t page_size, int32_t head_dim, int32_t type) {
  if (type < SFE_CACHE_BF16 || type > SFE_CACHE_INT8) return op_fail(SFE_INVALID_ARG, "unknown cache type");
  if (page_size < 16 || page_size > 1024 || (page_size & (page_size - 1)))
    return op_fail(SFE_INVALID_ARG, "page_size must be a power of two from 16 to 1024");
  if (head_dim <= 0 || head_dim % 16 != 0 || head_dim > sfe::kCacheMaxDim)
    return op_fail(SFE_INVALID_ARG, "head_dim must be a multiple of 16, at most 128");
  return SFE_OK;
}

// What a call over a cache has in common: the plan's and the cache's checks, and the kernels' arguments.
struct CacheCall {
  sfe::CacheArgs c{};
  Rows memory{"the cache", nullptr, 0, 0, 0}, table{"page_table", nullptr, 0, 0, 0}, lengths{"lengths", nullptr, 0, 0, 0};
};
int cache_call(sfe_cache_plan* plan, const sfe_cache* cache, const sfe_cache_tokens* tokens, CacheCall* out) {
  if (!plan || !cache || !tokens) return op_fail(SFE_INVALID_ARG, "null argument");
  if (!plan->ctx) return op_fail(SFE_INVALID_ARG, "the plan's context has been destroyed");
  int rc;
  if ((rc = check_cache_shape(cache->page_size, cache->head_dim, cache->type))) return rc;
  if (cache->kv_heads != plan->kv_heads || cache->head_dim != plan->dim)
    return op_fail(SFE_INVALID_ARG, "the cache's kv_heads and head_dim must be the plan's");
  if (cache->pages < 0 || cache->pages >= (int64_t)1 << 31) return op_fail(SFE_INVALID_ARG, "pages must be in [0, 2^31)");
  if (cache->pages > 0 && !cache->data) return op_fail(SFE_INVALID_ARG, "null cache data");
  if ((uintptr_t)cache->data % 16) return op_fail(SFE_INVALID_ARG, "cache data must be aligned to 16 bytes");
  if (tokens->table_pages < 0) return op_fail(SFE_INVALID_ARG, "negative table_pages");
  if (tokens->table_stride < 0 || tokens->table_stride >= kMaxStride)
    return op_fail(SFE_INVALID_ARG, "table_stride must be in [0, 2^40)");
  if (plan->rows > 0) {
    if (!tokens->lengths || (tokens->table_pages > 0 && !tokens->page_table)) return op_fail(SFE_INVALID_ARG, "null page_table or lengths");
    if ((uintptr_t)tokens->lengths % 4 || (uintptr_t)tokens->page_table % 4)
      return op_fail(SFE_INVALID_ARG, "page_table and lengths must be aligned");
  }
  sfe::CacheArgs& c = out->c;
  c.data = static_cast<char*>(cache->data);
  c.pages = cache->pages;
  c.record = sfe::cache_record(cache->page_size, cache->head_dim, cache->type);
  c.table = tokens->page_table;
  c.lengths = tokens->lengths;
  c.table_row = tokens->table_stride;
  c.table_pages = tokens->table_pages;
  c.kv_heads = cache->kv_heads;
  c.dim = cache->head_dim;
  c.shift = 0;
  while ((1 << c.shift) < cache->page_size) ++c.shift;
  out->memory = Rows("the cache", c.data, 1, 0, c.pages * c.kv_heads * c.record);
  out->table = Rows("page_table", c.table, plan->n, c.table_row * 4, (int64_t)c.table_pages * 4);
  out->lengths = Rows("lengths", c.lengths, 1, 0, (int64_t)plan->n * 4);
  return SFE_OK;
}

sfe::AttnTensor tensor_of(const sfe_heads* t, int esize) {
  return sfe::AttnTensor{static_cast<const char*>(t->data), t->row_stride * esize, t->head_stride * esize};
}

// sfe_cache_write and sfe_cache_read.
int move(sfe_cache_plan* plan, const sfe_cache* cache, const sfe_cache_tokens* tokens, int32_t dtype, const sfe_heads* k,
         const sfe_heads* v, bool write, void* stream) {
  if (!k || !v) return op_fail(SFE_INVALID_ARG, "null argument");
  if (!known_dtype(dtype)) return op_fail(SFE_INVALID_ARG, "dtype must be SFE_F32, SFE_BF16 or SFE_F16");
  CacheCall call;
  int rc;
  if ((rc = cache_call(plan, cache, tokens, &call))) return rc;
  if (plan->rows == 0) return SFE_OK;
  const int esize = sfe::op_size(dtype);
  const Rows both[] = {rows_of("k", *k, plan->rows, plan->kv_heads, plan->dim, esize),
                       rows_of("v", *v, plan->rows, plan->kv_heads, plan->dim, esize)};
  for (int i = 0; i < 2; ++i) {
    const sfe_heads& t = i ? *v : *k;
    if ((rc = check_heads(both[i].name, &t, plan->rows, esize, 16))) return rc;
    if (!write && !apart(t, plan->rows, plan->kv_heads, plan->dim))
      return op_fail(SFE_INVALID_ARG, std::string(both[i].name) + ": rows or heads overlap");
    if (share(both[i], call.memory)) return op_fail(SFE_INVALID_ARG, std::string(both[i].name) + " overlaps the cache");
    for (const Rows* o : {&call.table, &call.lengths})
      if (!write && share(both[i], *o)) return op_fail(SFE_INVALID_ARG, std::string(both[i].name) + " overlaps " + o->name);
  }
  if (!write && share(both[0], both[1])) return op_fail(SFE_INVALID_ARG, "k overlaps v");
  for (const Rows* o : {&call.table, &call.lengths})
    if (write && share(call.memory, *o)) return op_fail(SFE_INVALID_ARG, std::string("the cache overlaps ") + o->name);
  struct Call {
    sfe::CacheArgs c;
    const sfe_cache_plan* plan;
    sfe::AttnTensor k, v;
    int type, dtype;
    bool write;
    hipStream_t stream;
  } x{call.c, plan, tensor_of(k, esize), tensor_of(v, esize), cache->type, dtype, write, static_cast<hipStream_t>(stream)};
  return sfe::op_call(plan->ctx, x.stream, write ? "cache write" : "cache read", [](void* arg, int) -> hipError_t {
    Call& x = *static_cast<Call*>(arg);
    x.c.tiles = reinterpret_cast<const sfe::CacheTile*>(static_cast<char*>(x.plan->buf) + x.plan->tiles);
    x.c.n_tiles = x.plan->n_tiles;
    x.c.most = (int32_t)std::min<int64_t>(sfe::kCacheTileTokens, x.plan->longest);
    return x.write ? sfe::launch_cache_write(x.c, x.type, x.k, x.v, x.dtype, x.stream)
                   : sfe::launch_cache_read(x.c, x.type, x.k, x.v, x.dtype, x.stream);
  }, &x);
}

}  // namespace

extern "C" {

// ---- norms of heads and rotary positions -----------------------------------------------

int sfe_norm_rotary(sfe_ctx* ctx, const sfe_rotary_table* table, int32_t norm, float eps, int32_t dtype,
                    const int32_t* positions, int64_t rows, int32_t head_dim, int32_t q_heads, const float* q_weight,
                    const sfe_heads* q, const sfe_heads* q_out, int32_t k_heads, const float* k_weight,
                    const sfe_heads* k, const sfe_heads* k_out, void* stream) {
  return guarded([&]() -> int {
    if (!table) return op_fail(SFE_INVALID_ARG, "null table");
    if (norm != SFE_NORM_LAYER && norm != SFE_NORM_RMS) return op_fail(SFE_INVALID_ARG, "norm must be SFE_NORM_LAYER or SFE_NORM_RMS");
    if (!(eps >= 0.0f) || !isfinite(eps)) return op_fail(SFE_INVALID_ARG, "eps must be finite and not negative");
    if (!known_dtype(dtype)) return op_fail(SFE_INVALID_ARG, "dtype must be SFE_F32, SFE_BF16 or SFE_F16");
    if (rows < 0 || rows > (int64_t)1 << 40) return op_fail(SFE_INVALID_ARG, "rows must be in [0, 2^40]");
    if (table->rotary_dim <= 0 || table->rotary_dim % 2 || table->rotary_dim > 2 * sfe::kRotaryMaxPairs)
      return op_fail(SFE_INVALID_ARG, "table not initialised");
    if (head_dim < table->rotary_dim || head_dim > sfe::kNormRotaryMaxDim)
      return op_fail(SFE_INVALID_ARG, "head_dim must be at least the table's rotary_dim, at most 256");
    if (q_heads < 0 || k_heads < 0 || q_heads > 4096 || k_heads > 4096)
      return op_fail(SFE_INVALID_ARG, "heads must be in [0, 4096]");
    if (!ctx) return op_fail(SFE_INVALID_ARG, "null context");
    if (rows == 0 || q_heads + k_heads == 0) return SFE_OK;
    if (!positions) return op_fail(SFE_INVALID_ARG, "null positions");
    if ((uintptr_t)positions % 4) return op_fail(SFE_INVALID_ARG, "positions must be aligned");
    const int esize = sfe::op_size(dtype);
    struct Call {
      sfe::NormRotaryArgs a;
      int dtype;
      bool interleaved, layer;
      hipStream_t stream;
    } call{};
    const struct {
      const char *name, *out_name, *weight_name;
      int32_t heads;
      const float* weight;
      const sfe_heads *in, *out;
    } both[2] = {{"q", "q_out", "q_weight", q_heads, q_weight, q, q_out}, {"k", "k_out", "k_weight", k_heads, k_weight, k, k_out}};
    for (const auto& t : both) {
      if (!t.heads) continue;
      if (!t.in || !t.out) return op_fail(SFE_INVALID_ARG, std::string("null ") + t.name);
      int rc;
      if ((rc = check_heads(t.name, t.in, rows, esize, esize))) return rc;
      if ((rc = check_heads(t.out_name, t.out, rows, esize, esize))) return rc;
      if (!apart(*t.out, rows, t.heads, head_dim))
        return op_fail(SFE_INVALID_ARG, std::string(t.out_name) + ": rows or heads overlap");
      if ((uintptr_t)t.weight % 4) return op_fail(SFE_INVALID_ARG, std::string(t.weight_name) + " must be aligned");
    }
    // (a lane group reads a head before it writes it: an output may be its input's own view, and
    // of nothing that other groups read)
    auto view = [&](int i, bool out) {
      const auto& t = both[i];
      return rows_of(out ? t.out_name : t.name, out ? *t.out : *t.in, rows, t.heads, head_dim, esize);
    };
    for (int i = 0; i < 2; ++i) {
      if (!both[i].heads) continue;
      const Rows o = view(i, true);
      for (int j = 0; j < 2; ++j) {
        if (!both[j].heads) continue;
        const Rows x = view(j, false);
        if (share(o, x) && !(i == j && same_view(o, x) && (both[i].heads == 1 || both[i].in->head_stride == both[i].out->head_stride)))
          return op_fail(SFE_INVALID_ARG, std::string(o.name) + " overlaps " + x.name);
        if (i < j && share(o, view(j, true))) return op_fail(SFE_INVALID_ARG, "q_out overlaps k_out");
        const Rows w(both[j].weight_name, both[j].weight, both[j].weight ? 1 : 0, 0, (int64_t)head_dim * 4);
        if (share(o, w)) return op_fail(SFE_INVALID_ARG, std::string(o.name) + " overlaps " + w.name);
      }
      if (share(o, Rows("positions", positions, 1, 0, rows * 4)))
        return op_fail(SFE_INVALID_ARG, std::string(o.name) + " overlaps positions");
      call.a.t[i] = sfe::RotaryTensor{static_cast<const char*>(both[i].in->data), static_cast<char*>(both[i].out->data),
                                      both[i].in->row_stride, both[i].in->head_stride, both[i].out->row_stride,
                                      both[i].out->head_stride, both[i].heads};
      call.a.weight[i] = both[i].weight;
    }
    memcpy(call.a.step, table->step, sizeof(call.a.step));
    call.a.positions = positions;
    call.a.rows = rows;
    call.a.dim = head_dim;
    call.a.rotary = table->rotary_dim;
    call.a.magnitude = table->magnitude;
    call.a.eps = eps;
    call.dtype = dtype;
    call.interleaved = table->layout == SFE_ROTARY_INTERLEAVED;
    call.layer = norm == SFE_NORM_LAYER;
    call.stream = static_cast<hipStream_t>(stream);
    return sfe::op_call(ctx, call.stream, "norm and rotary", [](void* arg, int cus) -> hipError_t {
      Call& c = *static_cast<Call*>(arg);
      return sfe::launch_norm_rotary(c.a, c.dtype, c.interleaved, c.layer, cus, c.stream);
    }, &call);
  });
}

// ---- the paged cache ---------------------------------------------------------------------

int64_t sfe_cache_record(int32_t page_size, int32_t head_dim, int32_t type) {
  int64_t bytes = 0;
  (void)guarded([&]() -> int {
    const int rc = check_cache_shape(page_size, head_dim, type);
    if (!rc) bytes = sfe::cache_record(page_size, head_dim, type);
    return rc;
  });
  return bytes;
}

int sfe_cache_plan_make(sfe_ctx* ctx, const int64_t* offsets, int32_t n, int32_t heads, int32_t kv_heads,
                        int32_t head_dim, void* stream, sfe_cache_plan** out) {
  return guarded([&]() -> int {
    if (!out) return op_fail(SFE_INVALID_ARG, "null argument");
    *out = nullptr;
    if (!offsets) return op_fail(SFE_INVALID_ARG, "null offsets");
    if (n < 0 || n > 1 << 20) return op_fail(SFE_INVALID_ARG, "sequences must be in [0, 2^20]");
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0)
      return op_fail(SFE_INVALID_ARG, "heads must be a positive multiple of kv_heads");
    if (heads > 1024) return op_fail(SFE_INVALID_ARG, "more than 1024 heads");
    if (head_dim <= 0 || head_dim % 16 != 0 || head_dim > sfe::kCacheMaxDim)
      return op_fail(SFE_INVALID_ARG, "head_dim must be a multiple of 16, at most 128");
    int rc;
    if ((rc = sfe::check_offsets("offsets", offsets, n))) return rc;
    if (offsets[0] != 0) return op_fail(SFE_INVALID_ARG, "offsets must begin at 0");
    if (offsets[n] > 1 << 24) return op_fail(SFE_INVALID_ARG, "more than 2^24 new tokens");
    if (offsets[n] * (heads / kv_heads) > 1 << 28) return op_fail(SFE_INVALID_ARG, "more than 2^28 new tokens of grouped heads");
    if (!ctx) return op_fail(SFE_INVALID_ARG, "null context");
    auto plan = std::make_unique<sfe_cache_plan>();
    if ((rc = sfe::op_adopt(ctx, plan.get()))) return rc;
    plan->n = n;
    plan->heads = heads;
    plan->kv_heads = kv_heads;
    plan->dim = head_dim;
    plan->rows = offsets[n];
    for (int32_t s = 0; s < n; ++s) plan->longest = std::max(plan->longest, offsets[s + 1] - offsets[s]);
    if (plan->rows == 0) {
      *out = plan.release();
      return SFE_OK;
    }
    const int group = heads / kv_heads;
    plan->attn_tiles = sfe::cache_attn_tiles(plan->longest * group);
    const int rows = 16 * plan->attn_tiles;
    std::vector<sfe::CacheTile> tiles, attn;
    for (int32_t s = 0; s < n; ++s) {
      const int32_t m = (int32_t)(offsets[s + 1] - offsets[s]);
      for (int32_t at = 0; at < m; at += sfe::kCacheTileTokens)
        tiles.push_back({offsets[s], s, m, at, std::min(sfe::kCacheTileTokens, m - at)});
      for (int64_t at = 0; at < (int64_t)m * group; at += rows)
        attn.push_back({offsets[s], s, m, (int32_t)at, (int32_t)std::min<int64_t>(rows, (int64_t)m * group - at)});
    }
    plan->n_tiles = (int32_t)tiles.size();
    plan->n_attn = (int32_t)attn.size();
    plan->attn = up(tiles.size() * sizeof(sfe::CacheTile));
    std::vector<char> table(plan->attn + attn.size() * sizeof(sfe::CacheTile));
    memcpy(table.data(), tiles.data(), tiles.size() * sizeof(sfe::CacheTile));
    memcpy(table.data() + plan->attn, attn.data(), attn.size() * sizeof(sfe::CacheTile));
    const size_t shares = (size_t)sfe::cache_attn_shares(sfe::op_cus(ctx));
    plan->part_o = up(table.size());
    plan->part_ml = plan->part_o + up(2 * shares * rows * sfe::cache_attn_dim(head_dim) * sizeof(float));
    plan->units = plan->part_ml + up(2 * shares * rows * sizeof(float2));
    const size_t room = plan->units + up(attn.size() * kv_heads * sizeof(int2));
    if ((rc = sfe::op_upload(plan.get(), table.data(), table.size(), room, static_cast<hipStream_t>(stream)))) return rc;
    *out = plan.release();
    return SFE_OK;
  });
}

void sfe_cache_plan_free(sfe_cache_plan* plan) { delete plan; }

int sfe_cache_write(sfe_cache_plan* plan, const sfe_cache* cache, const sfe_cache_tokens* tokens, int32_t dtype,
                    const sfe_heads* k, const sfe_heads* v, void* stream) {
  return guarded([&]() -> int { return move(plan, cache, tokens, dtype, k, v, true, stream); });
}

int sfe_cache_read(sfe_cache_plan* plan, const sfe_cache* cache, const sfe_cache_tokens* tokens, int32_t dtype,
                   const sfe_heads* k, const sfe_heads* v, void* stream) {
  return guarded([&]() -> int { return move(plan, cache, tokens, dtype, k, v, false, stream); });
}

int sfe_cache_attention(sfe_cache_plan* plan, const sfe_cache* cache, const sfe_cache_tokens* tokens, int32_t dtype,
                        const sfe_heads* q, const uint64_t* tree, float scale, const sfe_heads* out, int64_t rows,
                        void* stream) {
  return guarded([&]() -> int {
    if (!q || !out) return op_fail(SFE_INVALID_ARG, "null argument");
    if (dtype != SFE_BF16 && dtype != SFE_F16) return op_fail(SFE_INVALID_ARG, "dtype must be SFE_BF16 or SFE_F16");
    CacheCall call;
    int rc;
    if ((rc = cache_call(plan, cache, tokens, &call))) return rc;
    if (!sfe::cache_coded(cache->type) && cache->type != dtype)
      return op_fail(SFE_INVALID_ARG, "a cache of 16 bits must have the queries' dtype");
    if (!(scale > 0.0f) || scale > 1e30f) return op_fail(SFE_INVALID_ARG, "scale must be positive and finite");
    if (rows < plan->rows || rows > (int64_t)1 << 40) return op_fail(SFE_INVALID_ARG, "rows must be in [offsets[n], 2^40]");
    if (tree && plan->longest > 64) return op_fail(SFE_INVALID_ARG, "a tree has at most 64 new tokens");
    if ((uintptr_t)tree % 8) return op_fail(SFE_INVALID_ARG, "tree must be aligned to 8 bytes");
    if (rows == 0) return SFE_OK;
    const int64_t keys = (int64_t)tokens->table_pages * cache->page_size;
    if (keys > sfe::kCacheAttnKeys) return op_fail(SFE_INVALID_ARG, "a page table of more than 2^30 tokens");
    const int64_t rounds = std::max<int64_t>(1, (keys + sfe::cache_attn_round(plan->attn_tiles) - 1) / sfe::cache_attn_round(plan->attn_tiles));
    const int64_t units = (int64_t)plan->n_attn * plan->kv_heads;
    const bool whole = sfe::cache_attn_whole(units, keys, plan->attn_tiles, sfe::cache_coded(cache->type) ? 1 : 2);
    if (!whole && units * rounds > (int64_t)1 << 30)
      return op_fail(SFE_INVALID_ARG, "batch too large: tiles of new tokens x kv_heads x tokens of a page table must be below 2^35");
    if ((rc = check_heads("q", q, plan->rows, 2, 16))) return rc;
    if ((rc = check_heads("out", out, rows, 2, 16))) return rc;
    if (!apart(*out, rows, plan->heads, plan->dim)) return op_fail(SFE_INVALID_ARG, "out: rows or heads overlap");
    const Rows mine = rows_of("out", *out, rows, plan->heads, plan->dim, 2);
    const Rows others[] = {rows_of("q", *q, plan->rows, plan->heads, plan->dim, 2), call.memory, call.table, call.lengths,
                           Rows("tree", tree, tree ? 1 : 0, 0, plan->rows * 8)};
    for (const Rows& o : others)
      if (share(mine, o)) return op_fail(SFE_INVALID_ARG, std::string("out overlaps ") + o.name);
    struct Call {
      sfe::CacheAttnArgs a;
      const sfe_cache_plan* plan;
      int type, dtype;
      int64_t rows;
      hipStream_t stream;
    } x{};
    x.a.c = call.c;
    x.a.q = tensor_of(q, 2);
    x.a.o = tensor_of(out, 2);
    x.a.tree = tree;
    x.a.group = plan->heads / plan->kv_heads;
    x.a.tiles = plan->attn_tiles;
    x.a.rows = (int32_t)std::min<int64_t>(16 * plan->attn_tiles, plan->longest * x.a.group);
    x.a.whole = whole;
    x.a.scale_log2 = (float)((double)scale * 1.4426950408889634);
    x.plan = plan;
    x.type = cache->type;
    x.dtype = dtype;
    x.rows = rows;
    x.stream = static_cast<hipStream_t>(stream);
    return sfe::op_call(plan->ctx, x.stream, "cache attention", [](void* arg, int cus) -> hipError_t {
      Call& x = *static_cast<Call*>(arg);
      if (x.rows > x.plan->rows) {
        const hipError_t e = sfe::launch_attn_zero(x.a.o, x.plan->heads, x.plan->dim, 0, x.plan->rows, x.rows, x.stream);
        if (e != hipSuccess) return e;
      }
      if (x.plan->rows == 0) return hipSuccess;
      char* base = static_cast<char*>(x.plan->buf);
      x.a.c.tiles = reinterpret_cast<const sfe::CacheTile*>(base + x.plan->attn);
      x.a.c.n_tiles = x.plan->n_attn;
      x.a.part_o = reinterpret_cast<float*>(base + x.plan->part_o);
      x.a.part_ml = reinterpret_cast<float2*>(base + x.plan->part_ml);
      x.a.units = reinterpret_cast<int2*>(base + x.plan->units);
      x.a.shares = sfe::cache_attn_shares(cus);
      return sfe::launch_cache_attn(x.a, x.type, x.dtype, x.stream);
    }, &x);
  });
}

// ---- steering of logits --------------------------------------------------------------------

int sfe_adjust_logits(sfe_ctx* ctx, const sfe_logits* l, void* stream) {
  return guarded([&]() -> int {
    if (!l) return op_fail(SFE_INVALID_ARG, "null argument");
    if (!known_dtype(l->dtype)) return op_fail(SFE_INVALID_ARG, "dtype must be SFE_F32, SFE_BF16 or SFE_F16");
    if (l->rows < 0) return op_fail(SFE_INVALID_ARG, "negative number of rows");
    if (l->vocab <= 0 || l->vocab > (1 << 24)) return op_fail(SFE_INVALID_ARG, "vocab must be in [1, 2^24]");
    if (l->history && (l->history_most < 0 || l->history_most > 1 << 30))
      return op_fail(SFE_INVALID_ARG, "history_most must be in [0, 2^30]");
    if (!l->history && l->lengths) return op_fail(SFE_INVALID_ARG, "lengths without a history");
    // (below f32's normal numbers its reciprocal, which quotients are products with, is infinite)
    if (!l->repetitions && (!(l->repetition >= 0x1p-126f) || !isfinite(l->repetition)))
      return op_fail(SFE_INVALID_ARG, "repetition must be finite and at least 2^-126");
    if ((!l->presences && !isfinite(l->presence)) || (!l->frequencies && !isfinite(l->frequency)))
      return op_fail(SFE_INVALID_ARG, "presence and frequency must be finite");
    if (l->allowed && l->n_allowed < 0) return op_fail(SFE_INVALID_ARG, "negative n_allowed");
    if (!l->allowed && l->states) return op_fail(SFE_INVALID_ARG, "states without masks");
    for (const int64_t stride : {l->logits_row, l->out_row, l->history ? l->history_row : 0, l->bias ? l->bias_row : 0,
                                 l->allowed ? l->allowed_row : 0})
      if (stride < 0 || stride >= kMaxStride) return op_fail(SFE_INVALID_ARG, "strides must be in [0, 2^40)");
    if (!ctx) return op_fail(SFE_INVALID_ARG, "null context");
    if (l->rows == 0) return SFE_OK;
    if (!l->logits || !l->out) return op_fail(SFE_INVALID_ARG, "null logits or out");
    const int esize = sfe::op_size(l->dtype);
    if ((uintptr_t)l->logits % esize || (uintptr_t)l->out % esize)
      return op_fail(SFE_INVALID_ARG, "logits and out must be aligned to their element size");
    if (l->rows > 1 && l->out_row < l->vocab) return op_fail(SFE_INVALID_ARG, "out: rows overlap");
    const int64_t rows = l->rows, words = ((int64_t)l->vocab + 31) / 32;
    const Rows out("out", l->out, rows, l->out_row * esize, (int64_t)l->vocab * esize);
    const Rows in("logits", l->logits, rows, l->logits_row * esize, (int64_t)l->vocab * esize);
    // (a thread reads what it writes before it does: out may be the logits' own view)
    if (share(out, in) && !same_view(out, in)) return op_fail(SFE_INVALID_ARG, "out overlaps logits");
    const Rows others[] = {Rows("history", l->history, l->history ? rows : 0, l->history_row * 4, (int64_t)l->history_most * 4),
                           Rows("lengths", l->lengths, l->lengths ? 1 : 0, 0, rows * 4),
                           Rows("repetition", l->repetitions, l->repetitions ? 1 : 0, 0, rows * 4),
                           Rows("presence", l->presences, l->presences ? 1 : 0, 0, rows * 4),
                           Rows("frequency", l->frequencies, l->frequencies ? 1 : 0, 0, rows * 4),
                           Rows("bias", l->bias, l->bias ? rows : 0, l->bias_row * 4, (int64_t)l->vocab * 4),
                           Rows("allowed", l->allowed, l->allowed ? l->n_allowed : 0, l->allowed_row * 4, words * 4),
                           Rows("states", l->states, l->states ? 1 : 0, 0, rows * 4)};
    for (const Rows& o : others) {
      if ((uintptr_t)o.p % 4) return op_fail(SFE_INVALID_ARG, std::string(o.name) + " must be aligned to 4 bytes");
      if (share(out, o)) return op_fail(SFE_INVALID_ARG, std::string("out overlaps ") + o.name);
    }
    struct Call {
      sfe::LogitsArgs a;
      int dtype;
      hipStream_t stream;
    } call{};
    sfe::LogitsArgs& a = call.a;
    a.in = static_cast<const char*>(l->logits);
    a.out = static_cast<char*>(l->out);
    a.in_row = l->logits_row;
    a.out_row = l->out_row;
    a.rows = l->rows;
    a.vocab = l->vocab;
    a.history = l->history;
    a.lengths = l->lengths;
    a.history_row = l->history_row;
    a.history_most = l->history_most;
    a.repetition = l->repetition;
    a.presence = l->presence;
    a.frequency = l->frequency;
    a.repetitions = l->repetitions;
    a.presences = l->presences;
    a.frequencies = l->frequencies;
    a.bias = l->bias;
    a.bias_row = l->bias_row;
    a.allowed = l->allowed;
    a.allowed_row = l->allowed_row;
    a.n_allowed = l->n_allowed;
    a.states = l->states;
    call.dtype = l->dtype;
    call.stream = static_cast<hipStream_t>(stream);
    return sfe::op_call(ctx, call.stream, "logits", [](void* arg, int) -> hipError_t {
      Call& c = *static_cast<Call*>(arg);
      return sfe::launch_logits(c.a, c.dtype, c.stream);
    }, &call);
  });
}

}  // extern "C"
