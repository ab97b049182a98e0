// Entry points of the model operators (declared in include/scriptrs_fe.h):
// argument checks, the attention's plans, and the launches in their context's
// order.  All compute runs in sfe_attn.hip, sfe_rotary.hip, sfe_residual.hip and
// sfe_beam.hip.
#include <hip/hip_runtime.h>
#include <math.h>
#include <string.h>

#include <algorithm>
#include <exception>
#include <memory>
#include <new>
#include <numeric>

#include "../../include/scriptrs_fe.h"
#include "sfe_ops.hpp"

using sfe::op_fail;

struct sfe_attn_plan : sfe::OpPlan {
  ~sfe_attn_plan() { sfe::op_drop(this); }
  int32_t heads = 0, kv_heads = 0, dim = 0, left = 0, right = 0;
  struct Form {
    int32_t n_items = 0, n_joins = 0;
    int32_t share[9] = {0};
    size_t items = 0, joins = 0, part_o = 0, part_ml = 0;  // offsets into buf
  } form[sfe::kAttnForms];
  bool empty = true;  // no queries
  size_t mask = 0;    // packed key mask
  int64_t first_q = 0, total_q = 0, total_k = 0;
};

namespace {

// Turns a C++ exception into a status: none crosses the C ABI.
template <class F>
int guarded(F&& body) {
  try {
    return body();
  } catch (const std::exception& e) {
    try {
      return op_fail(SFE_HIP_ERROR, std::string("host error: ") + e.what());
    } catch (...) {
      return SFE_HIP_ERROR;
    }
  } catch (...) {
    return SFE_HIP_ERROR;
  }
}

bool known_dtype(int32_t d) { return d == SFE_F32 || d == SFE_BF16 || d == SFE_F16; }

// A tensor's rows: n of len bytes, row bytes apart; each of `heads` pieces of `piece` bytes, head bytes apart.
struct Rows {
  const char* name;
  const void* p;
  int64_t n, row, len;
  int64_t heads, head, piece;
  Rows(const char* name_, const void* p_, int64_t n_, int64_t row_, int64_t len_)
      : Rows(name_, p_, n_, row_, 1, 0, len_) {}
  Rows(const char* name_, const void* p_, int64_t n_, int64_t row_, int64_t heads_, int64_t head_, int64_t piece_)
      : name(name_), p(p_), n(n_), row(row_), len((heads_ - 1) * head_ + piece_), heads(heads_), head(head_), piece(piece_) {}
  int64_t extent() const { return n <= 0 ? 0 : (n - 1) * row + len; }
  int64_t row_pitch() const { return n > 1 ? row : 0; }
  int64_t head_pitch() const { return heads > 1 ? head : 0; }
};
// Whether two tensors may share memory.  Views of one buffer lie between each other: where all parts of
// both (whole rows, single pieces, or a head's pieces of all rows) begin at multiples of one pitch from their
// first, their places within the pitch tell; otherwise whole extents do.
bool share(const Rows& a, const Rows& b) {
  const uintptr_t x = (uintptr_t)a.p, y = (uintptr_t)b.p;
  if (a.extent() == 0 || b.extent() == 0 || x >= y + (uintptr_t)b.extent() || y >= x + (uintptr_t)a.extent()) return false;
  auto between = [&](int64_t pitch, int64_t mine, int64_t other) {
    if (pitch == 0) return false;
    const int64_t d = ((int64_t)(y - x) % pitch + pitch) % pitch;
    return d >= mine && d + other <= pitch;
  };
  const int64_t rows = std::gcd(a.row_pitch(), b.row_pitch()), heads = std::gcd(a.head_pitch(), b.head_pitch());
  return !between(rows, a.len, b.len) && !between(std::gcd(rows, heads), a.piece, b.piece) &&
         !between(heads, (a.n - 1) * a.row + a.piece, (b.n - 1) * b.row + b.piece);
}
// An output that is an input's own view.
bool same_view(const Rows& a, const Rows& b) {
  return a.p == b.p && a.n == b.n && a.len == b.len && (a.n <= 1 || a.row == b.row);
}

// Bytes that a call reads or writes as a whole.
struct Span {
  uintptr_t begin, end;
  bool out;
  const char* name;
  int32_t number;  // of the tensors of the name, or -1
  Span(const void* p, int64_t bytes, bool out_, const char* name_, int32_t number_ = -1)
      : begin((uintptr_t)p), end((uintptr_t)p + (uintptr_t)bytes), out(out_), name(name_), number(number_) {}
};
// Refuses outputs that share memory with any other span.
int check_apart(Span* spans, size_t n) {
  std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
  uintptr_t any = 0, out = 0;  // ends of what begins at or before the span looked at, and of the outputs among it
  for (size_t i = 0; i < n; ++i) {
    const Span& s = spans[i];
    if (s.begin < (s.out ? any : out))
      return op_fail(SFE_INVALID_ARG, std::string(s.name) + (s.number < 0 ? "" : " " + std::to_string(s.number)) +
                                          " overlaps another tensor of the call");
    any = std::max(any, s.end);
    if (s.out) out = std::max(out, s.end);
  }
  return SFE_OK;
}

constexpr int64_t kMaxStride = (int64_t)1 << 40;  // elements: keeps 64-bit offsets far from their end

int check_heads(const char* name, const sfe_heads* t, int64_t rows, int esize, int align) {
  if (rows > 0 && !t->data) return op_fail(SFE_INVALID_ARG, std::string("null ") + name);
  if ((uintptr_t)t->data % align || t->row_stride * esize % align || t->head_stride * esize % align)
    return op_fail(SFE_INVALID_ARG, std::string(name) + ": data and strides must be aligned to " + std::to_string(align) +
                                        " bytes");
  if (t->row_stride < 0 || t->head_stride < 0 || t->row_stride >= kMaxStride || t->head_stride >= kMaxStride)
    return op_fail(SFE_INVALID_ARG, std::string(name) + ": strides must be in [0, 2^40)");
  return SFE_OK;
}

// Rows and heads of an output must be apart, in one of the two orders.
bool apart(const sfe_heads& t, int64_t rows, int heads, int dim) {
  const int64_t r = t.row_stride, h = t.head_stride;
  if (heads > 1 && h < dim) return false;
  if (rows > 1 && r < dim) return false;
  return rows <= 1 || heads <= 1 || r >= (heads - 1) * h + dim || h >= (rows - 1) * r + dim;
}
Rows rows_of(const char* name, const sfe_heads& t, int64_t rows, int heads, int dim, int esize) {
  return Rows(name, t.data, rows, t.row_stride * esize, heads, t.head_stride * esize, (int64_t)dim * esize);
}

int check_offsets(const char* name, const int64_t* off, int32_t n) {
  if (off[0] < 0) return op_fail(SFE_INVALID_ARG, std::string(name) + " must not be negative");
  for (int32_t i = 0; i < n; ++i) {
    if (off[i + 1] < off[i]) return op_fail(SFE_INVALID_ARG, std::string(name) + " must be non-decreasing");
    if (off[i + 1] - off[i] > (1 << 30)) return op_fail(SFE_INVALID_ARG, std::string(name) + ": sequence longer than 2^30");
  }
  if (off[n] > (int64_t)1 << 40) return op_fail(SFE_INVALID_ARG, std::string(name) + ": more than 2^40 rows");
  return SFE_OK;
}

size_t up(size_t x) { return (x + 255) / 256 * 256; }

// sfe_attention, and sfe_attention_rows where all_rows is given.
int attention(sfe_attn_plan* plan, int32_t dtype, const sfe_heads* q, const sfe_heads* k, const sfe_heads* v,
              const uint8_t* key_mask, float scale, const sfe_heads* out, const int64_t* all_rows, void* stream) {
  if (!plan || !q || !k || !v || !out) return op_fail(SFE_INVALID_ARG, "null argument");
  if (dtype != SFE_BF16 && dtype != SFE_F16) return op_fail(SFE_INVALID_ARG, "dtype must be SFE_BF16 or SFE_F16");
  if (!plan->ctx) return op_fail(SFE_INVALID_ARG, "the plan's context has been destroyed");
  if (!(scale > 0.0f) || scale > 1e30f) return op_fail(SFE_INVALID_ARG, "scale must be positive and finite");
  if (all_rows && (*all_rows < plan->total_q || *all_rows > (int64_t)1 << 40))
    return op_fail(SFE_INVALID_ARG, "rows must be in [q_offsets[n], 2^40]");
  const int64_t rows = all_rows ? *all_rows : plan->total_q;
  const bool outside = all_rows && (plan->first_q > 0 || rows > plan->total_q);
  if (plan->empty && !outside) return SFE_OK;  // no queries
  int rc;
  const struct {
    const char* name;
    const sfe_heads* t;
  } all[] = {{"q", q}, {"k", k}, {"v", v}, {"out", out}};
  for (const auto& x : all) {
    if (plan->empty && x.t != out) continue;  // (not read)
    // (k and v of sequences without keys are not read)
    if ((rc = check_heads(x.name, x.t, x.t == q || x.t == out ? 1 : 0, 2, 16))) return rc;
    if (x.t->row_stride >= (1 << 23))
      return op_fail(SFE_INVALID_ARG, std::string(x.name) + ": rows more than 2^23 elements apart");
  }
  if (!apart(*out, rows, plan->heads, plan->dim))
    return op_fail(SFE_INVALID_ARG, "out: rows or heads overlap");
  const Rows mine = rows_of("out", *out, rows, plan->heads, plan->dim, 2);
  for (const Rows& o : {rows_of("q", *q, plan->total_q, plan->heads, plan->dim, 2),
                        rows_of("k", *k, plan->total_k, plan->kv_heads, plan->dim, 2),
                        rows_of("v", *v, plan->total_k, plan->kv_heads, plan->dim, 2)})
    if (!plan->empty && share(mine, o)) return op_fail(SFE_INVALID_ARG, std::string("out overlaps ") + o.name);
  if (!plan->empty && plan->total_k > 0 && (!k->data || !v->data)) return op_fail(SFE_INVALID_ARG, "null k or v");
  auto tensor = [](const sfe_heads* t) {
    return sfe::AttnTensor{static_cast<const char*>(t->data), t->row_stride * 2, t->head_stride * 2};
  };
  sfe::AttnArgs a{};
  a.q = tensor(q);
  a.k = tensor(k);
  a.v = tensor(v);
  a.o = tensor(out);
  a.kv_heads = plan->kv_heads;
  a.group = plan->heads / plan->kv_heads;
  a.dim = plan->dim;
  a.left = plan->left;
  a.right = plan->right;
  a.scale_log2 = (float)((double)scale * 1.4426950408889634);
  struct Call {
    sfe::AttnArgs a;
    const sfe_attn_plan* plan;
    const uint8_t* key_mask;
    int dtype;
    int64_t rows;  // with those of no sequence to be zeroed, or 0
    hipStream_t stream;
  } call{a, plan, key_mask, dtype, outside ? rows : 0, static_cast<hipStream_t>(stream)};
  return sfe::op_call(plan->ctx, call.stream, "attention", [](void* arg, int cus) -> hipError_t {
    Call& c = *static_cast<Call*>(arg);
    char* base = static_cast<char*>(c.plan->buf);
    if (c.rows) {
      const hipError_t e = sfe::launch_attn_zero(c.a.o, c.plan->heads, c.plan->dim, c.plan->first_q, c.plan->total_q, c.rows,
                                                 c.stream);
      if (e != hipSuccess) return e;
    }
    if (c.plan->empty) return hipSuccess;
    if (c.key_mask) {
      uint64_t* words = reinterpret_cast<uint64_t*>(base + c.plan->mask);
      const hipError_t e = sfe::launch_attn_mask(c.key_mask, c.plan->total_k, words, c.stream);
      if (e != hipSuccess) return e;
      c.a.mask = words;
    }
    for (int i = 0; i < sfe::kAttnForms; ++i) {
      const auto& f = c.plan->form[i];
      if (!f.n_items) continue;
      c.a.n_items = f.n_items;
      memcpy(c.a.share, f.share, sizeof(f.share));
      c.a.items = reinterpret_cast<const sfe::AttnItem*>(base + f.items);
      c.a.n_joins = f.n_joins;
      c.a.joins = reinterpret_cast<const sfe::AttnJoin*>(base + f.joins);
      c.a.part_o = reinterpret_cast<float*>(base + f.part_o);
      c.a.part_ml = reinterpret_cast<float2*>(base + f.part_ml);
      const hipError_t e = sfe::launch_attn(c.a, i, c.dtype, cus, c.stream);
      if (e != hipSuccess) return e;
    }
    return hipSuccess;
  }, &call);
}

}  // namespace

extern "C" {

// ---- attention ---------------------------------------------------------------------

int sfe_attention_plan(sfe_ctx* ctx, const int64_t* q_offsets, const int64_t* k_offsets, int32_t n, int32_t heads,
                       int32_t kv_heads, int32_t head_dim, int64_t left, int64_t right, void* stream,
                       sfe_attn_plan** out) {
  return guarded([&]() -> int {
    if (!out) return op_fail(SFE_INVALID_ARG, "null argument");
    *out = nullptr;
    if (!q_offsets || !k_offsets) return op_fail(SFE_INVALID_ARG, "null offsets");
    if (n < 0) return op_fail(SFE_INVALID_ARG, "negative number of sequences");
    if (kv_heads <= 0 || heads <= 0 || heads % kv_heads != 0)
      return op_fail(SFE_INVALID_ARG, "heads must be a positive multiple of kv_heads");
    if (heads > 1024) return op_fail(SFE_INVALID_ARG, "more than 1024 heads");
    if (head_dim <= 0 || head_dim % 8 != 0 || head_dim > sfe::kAttnMaxDim)
      return op_fail(SFE_INVALID_ARG, "head_dim must be a multiple of 8, at most 128");
    int rc;
    if ((rc = check_offsets("q_offsets", q_offsets, n))) return rc;
    if ((rc = check_offsets("k_offsets", k_offsets, n))) return rc;
    const int group = heads / kv_heads;
    for (int32_t i = 0; i < n; ++i)
      if ((q_offsets[i + 1] - q_offsets[i]) * group > (1 << 30))
        return op_fail(SFE_INVALID_ARG, "a sequence has more than 2^30 queries of grouped heads");
    if (!ctx) return op_fail(SFE_INVALID_ARG, "null context");
    auto plan = std::make_unique<sfe_attn_plan>();
    if ((rc = sfe::op_adopt(ctx, plan.get()))) return rc;
    plan->heads = heads;
    plan->kv_heads = kv_heads;
    plan->dim = head_dim;
    plan->left = left < 0 || left >= sfe::kAttnNoBound ? sfe::kAttnNoBound : (int32_t)left;
    plan->right = right < 0 || right >= sfe::kAttnNoBound ? sfe::kAttnNoBound : (int32_t)right;
    plan->first_q = q_offsets[0];
    plan->total_q = q_offsets[n];
    plan->total_k = n ? k_offsets[n] : 0;
    sfe::AttnPlanHost h;
    sfe::attn_plan(q_offsets, k_offsets, n, group, kv_heads, head_dim, plan->left, plan->right, sfe::op_cus(ctx), &h);
    // (a launch holds fewer than 2^32 threads: 512 for each of 8 shares of at most all units)
    for (const auto& f : h.form) {
      if ((int64_t)f.items.size() * kv_heads > 1000000) return op_fail(SFE_INVALID_ARG, "batch too large for one launch");
      if (!f.items.empty()) plan->empty = false;
    }
    if (plan->empty) {
      *out = plan.release();
      return SFE_OK;
    }
    size_t at = 0;
    auto place = [&](size_t bytes) {
      const size_t o = at;
      at += up(bytes);
      return o;
    };
    for (int i = 0; i < sfe::kAttnForms; ++i) {
      plan->form[i].n_items = (int32_t)h.form[i].items.size();
      plan->form[i].n_joins = (int32_t)h.form[i].joins.size();
      memcpy(plan->form[i].share, h.form[i].share, sizeof(h.form[i].share));
      plan->form[i].items = place(h.form[i].items.size() * sizeof(sfe::AttnItem));
      plan->form[i].joins = place(h.form[i].joins.size() * sizeof(sfe::AttnJoin));
    }
    const size_t bytes = at;
    plan->mask = place((size_t)sfe::attn_mask_words(plan->total_k) * sizeof(uint64_t));
    std::vector<char> table(bytes);
    auto put = [&](size_t o, const void* p, size_t size) {
      if (size) memcpy(table.data() + o, p, size);
    };
    for (int i = 0; i < sfe::kAttnForms; ++i) {
      put(plan->form[i].items, h.form[i].items.data(), h.form[i].items.size() * sizeof(sfe::AttnItem));
      put(plan->form[i].joins, h.form[i].joins.data(), h.form[i].joins.size() * sizeof(sfe::AttnJoin));
      const size_t rows = (size_t)h.form[i].parts * kv_heads * sfe::attn_tile(i);
      plan->form[i].part_o = place(rows * sfe::attn_padded_dim(head_dim) * sizeof(float));
      plan->form[i].part_ml = place(rows * sizeof(float2));
    }
    if ((rc = sfe::op_upload(plan.get(), table.data(), bytes, at, static_cast<hipStream_t>(stream)))) return rc;
    *out = plan.release();
    return SFE_OK;
  });
}

void sfe_attention_plan_free(sfe_attn_plan* plan) { delete plan; }

int sfe_attention(sfe_attn_plan* plan, int32_t dtype, const sfe_heads* q, const sfe_heads* k, const sfe_heads* v,
                  const uint8_t* key_mask, float scale, const sfe_heads* out, void* stream) {
  return guarded([&]() -> int { return attention(plan, dtype, q, k, v, key_mask, scale, out, nullptr, stream); });
}

int sfe_attention_rows(sfe_attn_plan* plan, int32_t dtype, const sfe_heads* q, const sfe_heads* k, const sfe_heads* v,
                       const uint8_t* key_mask, float scale, const sfe_heads* out, int64_t rows, void* stream) {
  return guarded([&]() -> int { return attention(plan, dtype, q, k, v, key_mask, scale, out, &rows, stream); });
}

// ---- rotary ---------------------------------------------------------------------------

int sfe_rotary_init(sfe_rotary_table* table, int32_t rotary_dim, int32_t layout, double base, int32_t scaling,
                    double factor, double original_length, double low, double high, double magnitude) {
  return guarded([&]() -> int {
    if (!table) return op_fail(SFE_INVALID_ARG, "null argument");
    if (rotary_dim <= 0 || rotary_dim % 2 != 0 || rotary_dim > 2 * sfe::kRotaryMaxPairs)
      return op_fail(SFE_INVALID_ARG, "rotary_dim must be even, at most 256");
    if (layout != SFE_ROTARY_HALF && layout != SFE_ROTARY_INTERLEAVED)
      return op_fail(SFE_INVALID_ARG, "layout must be SFE_ROTARY_HALF or SFE_ROTARY_INTERLEAVED");
    if (!(base >= 1.0) || !isfinite(base)) return op_fail(SFE_INVALID_ARG, "base must be at least 1");
    if (scaling < SFE_ROTARY_UNSCALED || scaling > SFE_ROTARY_PARTS)
      return op_fail(SFE_INVALID_ARG, "unknown rotary scaling");
    if (scaling != SFE_ROTARY_UNSCALED && (!(factor >= 1.0) || !isfinite(factor)))
      return op_fail(SFE_INVALID_ARG, "factor must be at least 1");
    if (scaling == SFE_ROTARY_BASE && rotary_dim < 4)
      return op_fail(SFE_INVALID_ARG, "scaling the base needs at least 2 pairs");
    if (scaling == SFE_ROTARY_PARTS && (!(original_length > 0.0) || !isfinite(original_length) || !isfinite(low) ||
                                        !isfinite(high) || !(high > low)))
      return op_fail(SFE_INVALID_ARG, "original_length must be positive and low below high");
    if (!isfinite(magnitude)) return op_fail(SFE_INVALID_ARG, "magnitude must be finite");
    memset(table, 0, sizeof(*table));
    table->rotary_dim = rotary_dim;
    table->layout = layout;
    table->magnitude = (float)magnitude;
    // (64 bits of mantissa: a double's 53 are off by 2^-25 of a turn and more at the farthest positions)
    typedef long double Real;
    const Real R = rotary_dim, two_pi = 6.28318530717958647692528676655900577L;
    const Real b = scaling == SFE_ROTARY_BASE ? base * powl(factor, R / (R - 2)) : (Real)base;
    for (int p = 0; p < rotary_dim / 2; ++p) {
      Real f = powl(b, -2 * p / R);
      if (scaling == SFE_ROTARY_LINEAR) f /= factor;
      if (scaling == SFE_ROTARY_PARTS) {
        const Real turns = original_length * f / two_pi;
        const Real keep = std::min<Real>(1, std::max<Real>(0, (turns - low) / ((Real)high - low)));
        f *= (1 - keep) / factor + keep;
      }
      // at most 1 radian a position: below a turn
      table->step[p] = (uint64_t)rintl(f / two_pi * 18446744073709551616.0L);
    }
    return SFE_OK;
  });
}

int sfe_rotary(sfe_ctx* ctx, const sfe_rotary_table* table, int32_t inverse, int32_t dtype, const int32_t* positions,
               int64_t rows, int32_t head_dim, int32_t q_heads, const sfe_heads* q, const sfe_heads* q_out,
               int32_t k_heads, const sfe_heads* k, const sfe_heads* k_out, void* stream) {
  return guarded([&]() -> int {
    if (!table) return op_fail(SFE_INVALID_ARG, "null table");
    if (!known_dtype(dtype)) return op_fail(SFE_INVALID_ARG, "dtype must be SFE_F32, SFE_BF16 or SFE_F16");
    if (rows < 0 || rows > (int64_t)1 << 40) return op_fail(SFE_INVALID_ARG, "rows must be in [0, 2^40]");
    if (table->rotary_dim <= 0 || table->rotary_dim % 2 || table->rotary_dim > 2 * sfe::kRotaryMaxPairs)
      return op_fail(SFE_INVALID_ARG, "table not initialised");
    if (head_dim < table->rotary_dim || head_dim > 4096)
      return op_fail(SFE_INVALID_ARG, "head_dim must be at least the table's rotary_dim, at most 4096");
    if (q_heads < 0 || k_heads < 0 || q_heads > 4096 || k_heads > 4096)
      return op_fail(SFE_INVALID_ARG, "heads must be in [0, 4096]");
    if (!ctx) return op_fail(SFE_INVALID_ARG, "null context");
    if (rows == 0 || q_heads + k_heads == 0) return SFE_OK;
    if (!positions) return op_fail(SFE_INVALID_ARG, "null positions");
    const int esize = sfe::op_size(dtype);
    struct Call {
      sfe::RotaryArgs a;
      int dtype;
      bool interleaved;
      hipStream_t stream;
    } call{};
    const struct {
      const char *name, *out_name;
      int32_t heads;
      const sfe_heads *in, *out;
    } both[2] = {{"q", "q_out", q_heads, q, q_out}, {"k", "k_out", k_heads, k, k_out}};
    for (int i = 0; i < 2; ++i) {
      const auto& t = both[i];
      if (!t.heads) continue;
      if (!t.in || !t.out) return op_fail(SFE_INVALID_ARG, std::string("null ") + t.name);
      int rc;
      if ((rc = check_heads(t.name, t.in, rows, esize, esize))) return rc;
      if ((rc = check_heads(t.out_name, t.out, rows, esize, esize))) return rc;
      if (!apart(*t.out, rows, t.heads, head_dim))
        return op_fail(SFE_INVALID_ARG, std::string(t.out_name) + ": rows or heads overlap");
    }
    // (a thread reads a pair of every head before it writes it: an output may be its
    // input's own view)
    auto view = [&](int i, bool out) {
      const auto& t = both[i];
      return rows_of(out ? t.out_name : t.name, out ? *t.out : *t.in, rows, t.heads, head_dim, esize);
    };
    for (int i = 0; i < 2; ++i)
      for (int j = 0; j < 2; ++j) {
        if (!both[i].heads || !both[j].heads) continue;
        const Rows o = view(i, true), x = view(j, false);
        if (share(o, x) && !(i == j && same_view(o, x) && (both[i].heads == 1 || both[i].in->head_stride == both[i].out->head_stride)))
          return op_fail(SFE_INVALID_ARG, std::string(o.name) + " overlaps " + x.name);
        if (i < j && share(o, view(j, true))) return op_fail(SFE_INVALID_ARG, "q_out overlaps k_out");
      }
    memcpy(call.a.step, table->step, sizeof(call.a.step));
    for (int i = 0; i < 2; ++i) {
      const auto& t = both[i];
      if (!t.heads) continue;
      call.a.t[i] = sfe::RotaryTensor{static_cast<const char*>(t.in->data), static_cast<char*>(t.out->data),
                                      t.in->row_stride, t.in->head_stride, t.out->row_stride, t.out->head_stride, t.heads};
    }
    call.a.positions = positions;
    call.a.rows = rows;
    call.a.dim = head_dim;
    call.a.rotary = table->rotary_dim;
    call.a.inverse = inverse ? 1 : 0;
    call.a.magnitude = table->magnitude;
    call.dtype = dtype;
    call.interleaved = table->layout == SFE_ROTARY_INTERLEAVED;
    call.stream = static_cast<hipStream_t>(stream);
    return sfe::op_call(ctx, call.stream, "rotary", [](void* arg, int cus) -> hipError_t {
      Call& c = *static_cast<Call*>(arg);
      return sfe::launch_rotary(c.a, c.dtype, c.interleaved, cus, c.stream);
    }, &call);
  });
}

// ---- norms around a block ----------------------------------------------------------------

int sfe_residual_norm(sfe_ctx* ctx, const sfe_residual* r, void* stream) {
  return guarded([&]() -> int {
    if (!r) return op_fail(SFE_INVALID_ARG, "null argument");
    if (!known_dtype(r->stream_dtype) || !known_dtype(r->block_dtype))
      return op_fail(SFE_INVALID_ARG, "dtypes must be SFE_F32, SFE_BF16 or SFE_F16");
    if (r->stream_dtype != SFE_F32 && r->stream_dtype != r->block_dtype)
      return op_fail(SFE_INVALID_ARG, "stream_dtype must be SFE_F32 or block_dtype");
    if (r->rows < 0 || r->rows > (int64_t)1 << 40) return op_fail(SFE_INVALID_ARG, "rows must be in [0, 2^40]");
    if (r->width <= 0 || r->width > sfe::kResidualMaxWidth)
      return op_fail(SFE_INVALID_ARG, "width must be in [1, " + std::to_string(sfe::kResidualMaxWidth) + "]");
    const struct {
      const char* name;
      int32_t kind;
      const float *w, *b;
    } norms[] = {{"post", r->post, r->post_weight, r->post_bias}, {"pre", r->pre, r->pre_weight, r->pre_bias}};
    for (const auto& n : norms) {
      if (n.kind < SFE_NORM_NONE || n.kind > SFE_NORM_RMS) return op_fail(SFE_INVALID_ARG, std::string("unknown ") + n.name + " norm");
      if (n.kind != SFE_NORM_NONE && !n.w) return op_fail(SFE_INVALID_ARG, std::string(n.name) + " norm without weight");
      if (n.kind == SFE_NORM_RMS && n.b) return op_fail(SFE_INVALID_ARG, std::string(n.name) + ": an rms norm has no bias");
      if ((uintptr_t)n.w % 4 || (uintptr_t)n.b % 4) return op_fail(SFE_INVALID_ARG, std::string(n.name) + ": weights must be aligned");
    }
    if (!(r->eps >= 0.0f) || !isfinite(r->eps)) return op_fail(SFE_INVALID_ARG, "eps must be finite and not negative");
    if (!isfinite(r->scale)) return op_fail(SFE_INVALID_ARG, "scale must be finite");
    if (!ctx) return op_fail(SFE_INVALID_ARG, "null context");
    if (r->rows == 0) return SFE_OK;
    if (!r->residual || !r->block || !r->residual_out) return op_fail(SFE_INVALID_ARG, "null residual, block or residual_out");
    if (r->pre != SFE_NORM_NONE && !r->norm_out) return op_fail(SFE_INVALID_ARG, "null norm_out");
    const int xs = sfe::op_size(r->stream_dtype), ys = sfe::op_size(r->block_dtype);
    const struct {
      Rows r;
      int size;
      bool out;
    } all[] = {{{"residual", r->residual, r->rows, r->residual_row, r->width}, xs, false},
               {{"block", r->block, r->rows, r->block_row, r->width}, ys, false},
               {{"gate", r->gate, r->gate_row ? r->rows : 1, r->gate_row, r->width}, ys, false},
               {{"residual_out", r->residual_out, r->rows, r->residual_out_row, r->width}, xs, true},
               {{"norm_out", r->pre != SFE_NORM_NONE ? r->norm_out : nullptr, r->rows, r->norm_out_row, r->width}, ys, true}};
    auto in_bytes = [](Rows x, int size) {
      return Rows(x.name, x.p, x.n, x.row * size, x.len * size);
    };
    for (const auto& t : all) {
      if (!t.r.p) continue;
      if ((uintptr_t)t.r.p % t.size) return op_fail(SFE_INVALID_ARG, std::string(t.r.name) + " is not aligned to its element size");
      if (t.r.row < 0 || t.r.row >= kMaxStride)
        return op_fail(SFE_INVALID_ARG, std::string(t.r.name) + ": row stride must be in [0, 2^40)");
      if (t.out && r->rows > 1 && t.r.row < r->width) return op_fail(SFE_INVALID_ARG, std::string(t.r.name) + ": rows overlap");
    }
    // (a thread reads its channels of a row before it writes them: an output may be
    // an input's own view)
    for (const auto& t : all)
      for (const auto& o : all) {
        if (!t.out || !t.r.p || !o.r.p || &t == &o) continue;
        const Rows x = in_bytes(t.r, t.size), y = in_bytes(o.r, o.size);
        if (share(x, y) && !(same_view(x, y) && !o.out))
          return op_fail(SFE_INVALID_ARG, std::string(t.r.name) + " overlaps " + o.r.name);
      }
    struct Call {
      sfe::ResidualArgs a;
      int xt, yt;
      hipStream_t stream;
    } call{};
    sfe::ResidualArgs& a = call.a;
    a.x = static_cast<const char*>(r->residual);
    a.y = static_cast<const char*>(r->block);
    a.gate = static_cast<const char*>(r->gate);
    a.xo = static_cast<char*>(r->residual_out);
    a.z = static_cast<char*>(r->norm_out);
    a.post_w = r->post_weight;
    a.post_b = r->post_bias;
    a.pre_w = r->pre_weight;
    a.pre_b = r->pre_bias;
    a.x_row = r->residual_row;
    a.y_row = r->block_row;
    a.gate_row = r->gate_row;
    a.xo_row = r->residual_out_row;
    a.z_row = r->norm_out_row;
    a.rows = r->rows;
    a.width = r->width;
    a.post = r->post;
    a.pre = r->pre;
    a.sigmoid = r->gate_sigmoid ? 1 : 0;
    a.scale = r->scale;
    a.eps = r->eps;
    call.xt = r->stream_dtype;
    call.yt = r->block_dtype;
    call.stream = static_cast<hipStream_t>(stream);
    return sfe::op_call(ctx, call.stream, "residual norm", [](void* arg, int) -> hipError_t {
      Call& c = *static_cast<Call*>(arg);
      return sfe::launch_residual(c.a, c.xt, c.yt, c.stream);
    }, &call);
  });
}

// ---- beam search -------------------------------------------------------------------------

int sfe_beam_select(sfe_ctx* ctx, int32_t dtype, const void* logits, int64_t row_stride, int32_t streams, int32_t beams,
                    int32_t vocab, const float* scores, const uint8_t* finished, int32_t end_token, float* out_scores,
                    int32_t* parents, int32_t* tokens, uint8_t* out_finished, void* stream) {
  return guarded([&]() -> int {
    if (!known_dtype(dtype)) return op_fail(SFE_INVALID_ARG, "dtype must be SFE_F32, SFE_BF16 or SFE_F16");
    if (streams < 0) return op_fail(SFE_INVALID_ARG, "negative number of streams");
    if (beams <= 0 || beams > sfe::kMaxBeams) return op_fail(SFE_INVALID_ARG, "beams must be in [1, 32]");
    if (vocab <= 0 || vocab > (1 << 24)) return op_fail(SFE_INVALID_ARG, "vocab must be in [1, 2^24]");
    if (end_token < -1 || end_token >= vocab) return op_fail(SFE_INVALID_ARG, "end_token must be a token, or -1");
    if (finished && end_token < 0) return op_fail(SFE_INVALID_ARG, "finished beams need an end_token");
    if (!ctx) return op_fail(SFE_INVALID_ARG, "null context");
    if (streams == 0) return SFE_OK;
    if (!logits || !scores || !out_scores || !parents || !tokens) return op_fail(SFE_INVALID_ARG, "null argument");
    if ((uintptr_t)logits % sfe::op_size(dtype)) return op_fail(SFE_INVALID_ARG, "logits are not aligned to their element size");
    if (row_stride < 0 || row_stride >= kMaxStride) return op_fail(SFE_INVALID_ARG, "row_stride must be in [0, 2^40)");
    // a launch holds fewer than 2^32 threads, of up to 64 a beam and up to 2 workgroups of
    // 256 a row (more only where the rows alone do not fill the device)
    if ((int64_t)streams * beams > (1 << 22)) return op_fail(SFE_INVALID_ARG, "batch too large for one launch");
    const int64_t rows = (int64_t)streams * beams;
    Span spans[] = {{scores, 4 * rows, false, "scores"},
                    {finished, finished ? rows : 0, false, "finished"},
                    {out_scores, 4 * rows, true, "out_scores"},
                    {parents, 4 * rows, true, "parents"},
                    {tokens, 4 * rows, true, "tokens"},
                    {out_finished, out_finished ? rows : 0, true, "out_finished"}};
    if (const int rc = check_apart(spans, sizeof(spans) / sizeof(*spans))) return rc;
    const int esize = sfe::op_size(dtype);
    for (const Span& s : spans)
      if (s.out && share(Rows("logits", logits, rows, row_stride * esize, (int64_t)vocab * esize),
                         Rows(s.name, (const void*)s.begin, 1, 0, (int64_t)(s.end - s.begin))))
        return op_fail(SFE_INVALID_ARG, std::string(s.name) + " overlaps logits");
    struct Call {
      sfe::BeamArgs a;
      int dtype;
      hipStream_t stream;
    } call{};
    call.stream = static_cast<hipStream_t>(stream);
    call.dtype = dtype;
    void* scratch = nullptr;
    const size_t room = sfe::beam_scratch_bytes(streams, beams, vocab, sfe::op_cus(ctx));
    const int rc = room ? sfe::op_scratch(ctx, room, call.stream, &scratch) : SFE_OK;
    if (rc) return rc;
    call.a = sfe::BeamArgs{static_cast<const char*>(logits), row_stride, streams, beams, vocab, end_token, scores, finished,
                           out_scores, parents, tokens, out_finished, static_cast<char*>(scratch)};
    return sfe::op_call(ctx, call.stream, "beam select", [](void* arg, int cus) -> hipError_t {
      Call& c = *static_cast<Call*>(arg);
      return sfe::launch_beam_select(c.a, c.dtype, cus, c.stream);
    }, &call);
  });
}

int sfe_beam_reorder(sfe_ctx* ctx, const int32_t* parents, int32_t streams, int32_t beams, const sfe_beam_state* states,
                     int32_t n, void* stream) {
  return guarded([&]() -> int {
    if (n < 0 || streams < 0) return op_fail(SFE_INVALID_ARG, "negative count");
    if (beams <= 0 || beams > sfe::kMaxBeams) return op_fail(SFE_INVALID_ARG, "beams must be in [1, 32]");
    if (!ctx) return op_fail(SFE_INVALID_ARG, "null context");
    if (n == 0 || streams == 0) return SFE_OK;
    if (!parents || !states) return op_fail(SFE_INVALID_ARG, "null argument");
    struct Call {
      std::vector<sfe::ReorderArgs> launches;
      hipStream_t stream;
    } call;
    call.stream = static_cast<hipStream_t>(stream);
    // What the launch reads and writes (all states at once): an output may share memory with nothing but its own
    // input, in place.
    std::vector<Span> used;
    used.reserve(2 * (size_t)n + 1);
    used.emplace_back(parents, (int64_t)streams * beams * 4, false, "parents");
    for (int32_t i = 0; i < n; ++i) {
      const sfe_beam_state& s = states[i];
      const std::string name = "state " + std::to_string(i);
      if (s.outer < 0 || s.inner_bytes < 0) return op_fail(SFE_INVALID_ARG, name + ": negative size");
      if (s.outer > (int64_t)1 << 40 || s.inner_bytes >= (int64_t)1 << 31 ||
          (double)s.outer * (double)s.inner_bytes * streams * beams > 1e12)
        return op_fail(SFE_INVALID_ARG, name + " is too large");
      const int64_t bytes = s.outer * streams * beams * s.inner_bytes;
      if (bytes == 0) continue;
      if (!s.in || !s.out) return op_fail(SFE_INVALID_ARG, name + " is null");
      used.emplace_back(s.out, bytes, true, "state", i);
      if (s.in != s.out) used.emplace_back(s.in, bytes, false, "state", i);
      if (call.launches.empty() || call.launches.back().n == sfe::kReorderStates) {
        call.launches.emplace_back();
        memset(&call.launches.back(), 0, sizeof(sfe::ReorderArgs));
        call.launches.back().streams = streams;
        call.launches.back().beams = beams;
        call.launches.back().parents = parents;
      }
      sfe::ReorderArgs& l = call.launches.back();
      l.s[l.n++] = sfe::BeamState{static_cast<const char*>(s.in), static_cast<char*>(s.out), s.outer, s.inner_bytes};
    }
    if (call.launches.empty()) return SFE_OK;
    if (const int rc = check_apart(used.data(), used.size())) return rc;
    return sfe::op_call(ctx, call.stream, "beam reorder", [](void* arg, int) -> hipError_t {
      Call& c = *static_cast<Call*>(arg);
      for (const sfe::ReorderArgs& l : c.launches) {
        const hipError_t e = sfe::launch_beam_reorder(l, c.stream);
        if (e != hipSuccess) return e;
      }
      return hipSuccess;
    }, &call);
  });
}

}  // extern "C"
