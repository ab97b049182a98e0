// Checks of arguments that the model operators' entry points (sfe_ops.cpp, sfe_decode.cpp) share.
#pragma once

#include <stdint.h>

#include <algorithm>
#include <exception>
#include <numeric>
#include <string>

#include "../../include/scriptrs_fe.h"
#include "sfe_ops.hpp"

namespace sfe {

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

inline bool known_dtype(int32_t d) { return d == SFE_F32 || d == SFE_BF16 || d == SFE_F16; }

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
inline bool share(const Rows& a, const Rows& b) {
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
inline bool same_view(const Rows& a, const Rows& b) {
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
inline int check_apart(Span* spans, size_t n) {
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

inline int check_heads(const char* name, const sfe_heads* t, int64_t rows, int esize, int align) {
  if (rows > 0 && !t->data) return op_fail(SFE_INVALID_ARG, std::string("null ") + name);
  if ((uintptr_t)t->data % align || t->row_stride * esize % align || t->head_stride * esize % align)
    return op_fail(SFE_INVALID_ARG, std::string(name) + ": data and strides must be aligned to " + std::to_string(align) +
                                        " bytes");
  if (t->row_stride < 0 || t->head_stride < 0 || t->row_stride >= kMaxStride || t->head_stride >= kMaxStride)
    return op_fail(SFE_INVALID_ARG, std::string(name) + ": strides must be in [0, 2^40)");
  return SFE_OK;
}

// Rows and heads of an output must be apart, in one of the two orders.
inline bool apart(const sfe_heads& t, int64_t rows, int heads, int dim) {
  const int64_t r = t.row_stride, h = t.head_stride;
  if (heads > 1 && h < dim) return false;
  if (rows > 1 && r < dim) return false;
  return rows <= 1 || heads <= 1 || r >= (heads - 1) * h + dim || h >= (rows - 1) * r + dim;
}
inline Rows rows_of(const char* name, const sfe_heads& t, int64_t rows, int heads, int dim, int esize) {
  return Rows(name, t.data, rows, t.row_stride * esize, heads, t.head_stride * esize, (int64_t)dim * esize);
}

inline int check_offsets(const char* name, const int64_t* off, int32_t n) {
  if (off[0] < 0) return op_fail(SFE_INVALID_ARG, std::string(name) + " must not be negative");
  for (int32_t i = 0; i < n; ++i) {
    if (off[i + 1] < off[i]) return op_fail(SFE_INVALID_ARG, std::string(name) + " must be non-decreasing");
    if (off[i + 1] - off[i] > (1 << 30)) return op_fail(SFE_INVALID_ARG, std::string(name) + ": sequence longer than 2^30");
  }
  if (off[n] > (int64_t)1 << 40) return op_fail(SFE_INVALID_ARG, std::string(name) + ": more than 2^40 rows");
  return SFE_OK;
}

inline size_t up(size_t x) { return (x + 255) / 256 * 256; }

}  // namespace sfe
