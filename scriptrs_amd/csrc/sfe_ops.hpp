// The model operators behind the features (attention over packed sequences,
// rotary positions, norms around a block, beam search): what their entry
// points (sfe_ops.cpp) share with the context (sfe_capi.cpp), and their
// kernels' launchers.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <string>
#include <utility>
#include <vector>

struct sfe_ctx;

namespace sfe {

// ---- the context's part (sfe_capi.cpp) ----------------------------------------

// Sets the calling thread's message and returns code.
int op_fail(int code, const std::string& msg);
int op_hip_fail(hipError_t e, const char* what);

// Queues an operator on `stream` in the context's order: the device is made
// current, the context locked, the stream ordered after the context's earlier
// calls, body(arg, compute units) run, and the call's end marked.  On a stream
// that is being captured the order is the caller's graph's: nothing is waited
// for or marked.
int op_call(sfe_ctx* ctx, hipStream_t stream, const char* what, hipError_t (*body)(void* arg, int cus), void* arg);

// A plan's part that its context knows: which context it is of, until that is destroyed, and its
// device buffer.
struct OpPlan {
  sfe_ctx* ctx = nullptr;
  void* buf = nullptr;
  size_t cap = 0;
};
// The plans of a context and the buffers of freed ones, which the next plans take.  A context that is destroyed takes
// its plans' buffers along; what is left of such a plan is only good for freeing.
class OpPlans {
 public:
  void adopt(OpPlan* p, sfe_ctx* ctx) {
    live_.reserve(live_.size() + 1);
    free_.reserve(free_.size() + live_.size() + 1);  // (so that drop and give cannot throw)
    live_.push_back(p);
    p->ctx = ctx;
  }
  void drop(OpPlan* p) noexcept {
    live_.erase(std::find(live_.begin(), live_.end(), p));
    if (p->buf) give(p->buf, p->cap);
    *p = OpPlan{};
  }
  // The smallest freed buffer that is large enough and not far too large.
  bool take(size_t room, void** buf, size_t* cap) noexcept {
    size_t best = free_.size();
    for (size_t i = 0; i < free_.size(); ++i) {
      const size_t c = free_[i].second;
      if (c >= room && c / 8 <= room + 65536 && (best == free_.size() || c < free_[best].second)) best = i;
    }
    if (best == free_.size()) return false;
    *buf = free_[best].first;
    *cap = free_[best].second;
    free_.erase(free_.begin() + (std::ptrdiff_t)best);
    return true;
  }
  // A buffer of an adopted plan that has none, back.
  void give(void* buf, size_t cap) noexcept { free_.emplace_back(buf, cap); }
  template <class F>
  void close(F&& free_buffer) noexcept {
    for (OpPlan* p : live_) {
      if (p->buf) free_buffer(p->buf);
      *p = OpPlan{};
    }
    for (auto& b : free_) free_buffer(b.first);
    live_.clear();
    free_.clear();
  }

 private:
  std::vector<OpPlan*> live_;
  std::vector<std::pair<void*, size_t>> free_;
};

// Enters a plan into its context; it stays there until op_drop (which does nothing for a plan of no context).
int op_adopt(sfe_ctx* ctx, OpPlan* plan);
void op_drop(OpPlan* plan) noexcept;
// Memory of an adopted plan: the first `bytes` of a device buffer of at least `room`
// bytes are filled from `table` on `stream` (through the context's pinned
// staging).  The buffer comes from the context's freed ones where one fits: the
// upload is ordered after every earlier call that read it.  Refused while `stream` is being captured.
int op_upload(OpPlan* plan, const void* table, size_t bytes, size_t room, hipStream_t stream);
int op_cus(sfe_ctx* ctx);  // compute units of the context's device

// Scratch of at least `bytes` for the calls of a context, which are ordered after
// each other.  Outgrown buffers live as long as the context (a captured graph
// may hold their addresses).  Growing while `stream` is captured fails.
int op_scratch(sfe_ctx* ctx, size_t bytes, hipStream_t stream, void** out);

// ---- element types ---------------------------------------------------------------
enum OpType { kOpF32 = 0, kOpBf16 = 1, kOpF16 = 2 };  // sfe_dtype
inline int op_size(int type) { return type == kOpF32 ? 4 : 2; }

// ---- attention over packed sequences (sfe_attn.hip, sfe_attn_plan.cpp) -------------

// A tile's piece: `rows` packed rows of one sequence (row = query * group +
// head within the group: the queries of the heads that share a kv head) against
// the keys [kv0, kv1).
struct AttnItem {
  int64_t q_row, k_row;  // first query and key row of the sequence
  int32_t lq, lk;        // its queries and keys
  int32_t row0;          // first packed row of the tile
  int32_t kv0, kv1;
  int32_t part;          // piece number among the partial results, or -1: the whole result
  int32_t pad[2];
};
static_assert(sizeof(AttnItem) == 48, "layout shared with the kernels");
// Pieces of one tile to be added up.
struct AttnJoin {
  int64_t q_row;
  int32_t lq, row0, part0, parts;
};
static_assert(sizeof(AttnJoin) == 24, "layout shared with the kernels");

// Kernel forms, packed rows of their tiles and keys of their steps: `tall` (8 waves of 32 rows
// share a step's keys, in two halves that take turns at the matrix cores), `rows` (4 waves of
// 32 rows) and `few` (16 rows, each of 4 waves takes every fourth step).
enum AttnKernel { kAttnTall = 0, kAttnRows = 1, kAttnFew = 2, kAttnForms = 3 };
constexpr int kAttnTileTall = 256, kAttnTileRows = 128, kAttnStepRows = 64;
constexpr int kAttnTileFew = 16, kAttnStepFew = 32, kAttnWavesFew = 4;
constexpr int kAttnMaxDim = 128;
constexpr int32_t kAttnNoBound = 0x7fffffff;
inline int attn_tile(int form) { return form == kAttnTall ? kAttnTileTall : (form == kAttnRows ? kAttnTileRows : kAttnTileFew); }

struct AttnForm {
  std::vector<AttnItem> items;
  std::vector<AttnJoin> joins;
  int32_t parts = 0;  // pieces with a partial result
  int32_t share[9];   // units of XCD x: [share[x], share[x + 1])
};
struct AttnPlanHost {
  AttnForm form[kAttnForms];
};
// Lays the tiles of n sequences out (host only).  left, right: the window, or
// kAttnNoBound.
void attn_plan(const int64_t* q_offsets, const int64_t* k_offsets, int n, int group, int kv_heads, int head_dim,
               int32_t left, int32_t right, int cus, AttnPlanHost* out);

struct AttnTensor {
  const char* data;
  int64_t row, head;  // strides in bytes
};
struct AttnArgs {
  AttnTensor q, k, v, o;
  const uint64_t* mask;  // packed, or null
  const AttnItem* items;
  const AttnJoin* joins;
  float* part_o;    // [piece][kv head][tile row][padded head dim]
  float2* part_ml;  // [piece][kv head][tile row]: (reference exponent, sum)
  int32_t n_items, n_joins, kv_heads, group, dim;
  int32_t share[9];  // units of XCD x: [share[x], share[x + 1])
  int32_t left, right;
  float scale_log2;  // scale * log2(e)
};
inline int attn_padded_dim(int dim) { return dim <= 64 ? 64 : (dim <= 96 ? 96 : 128); }
// Words of a packed key mask: the masks of up to 3 steps past the last key are looked at, any
// of them across two words.
inline int64_t attn_mask_words(int64_t keys) { return (keys + 63) / 64 + 3 * kAttnStepRows / 64 + 2; }
hipError_t launch_attn_mask(const uint8_t* mask, int64_t keys, uint64_t* words, hipStream_t stream);
// Zeros the rows [0, first) and [last, rows) of `out` of heads x dim.
hipError_t launch_attn_zero(const AttnTensor& out, int heads, int dim, int64_t first, int64_t last, int64_t rows,
                            hipStream_t stream);
hipError_t launch_attn(const AttnArgs& a, int form, int type, int cus, hipStream_t stream);

// ---- rotary positions (sfe_rotary.hip) ----------------------------------------------
constexpr int kRotaryMaxPairs = 128;
struct RotaryTensor {
  const char* x;
  char* y;
  int64_t x_row, x_head, y_row, y_head;  // strides in elements
  int32_t heads;
};
struct RotaryArgs {
  uint64_t step[kRotaryMaxPairs];  // turns a position, as a fraction of 2^64
  RotaryTensor t[2];
  const int32_t* positions;
  int64_t rows;
  int32_t dim, rotary, inverse;
  float magnitude;
};
hipError_t launch_rotary(const RotaryArgs& a, int type, bool interleaved, int cus, hipStream_t stream);

// ---- norms around a block (sfe_residual.hip) ------------------------------------------
enum NormKind { kNormNone = 0, kNormLayer = 1, kNormRms = 2 };
struct ResidualArgs {
  const char *x, *y, *gate;  // residual stream, block output, gate (or null)
  char *xo, *z;              // new residual stream, its norm (or null)
  const float *post_w, *post_b, *pre_w, *pre_b;
  int64_t x_row, y_row, gate_row, xo_row, z_row;  // strides in elements
  int64_t rows;
  int32_t width, post, pre, sigmoid;
  float scale, eps;
};
constexpr int kResidualMaxWidth = 16384;
hipError_t launch_residual(const ResidualArgs& a, int stream_type, int block_type, hipStream_t stream);

// ---- beam search (sfe_beam.hip) ----------------------------------------------------------
constexpr int kMaxBeams = 32;
struct BeamArgs {
  const char* logits;
  int64_t row;  // stride in elements
  int32_t streams, beams, vocab, end;
  const float* scores;
  const uint8_t* finished;  // or null
  float* out_scores;
  int32_t *parents, *tokens;
  uint8_t* out_finished;  // or null
  char* scratch;
};
size_t beam_scratch_bytes(int streams, int beams, int vocab, int cus);
hipError_t launch_beam_select(const BeamArgs& a, int type, int cus, hipStream_t stream);

struct BeamState {
  const char* in;
  char* out;
  int64_t outer, inner;  // [outer][streams * beams][inner bytes]
};
constexpr int kReorderStates = 8;  // of one launch
struct ReorderArgs {
  BeamState s[kReorderStates];
  int32_t n, streams, beams;
  const int32_t* parents;
};
hipError_t launch_beam_reorder(const ReorderArgs& a, hipStream_t stream);

}  // namespace sfe
