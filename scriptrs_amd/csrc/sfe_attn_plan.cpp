// Host planner of the packed attention: which tile of which sequence takes
// which keys, in which kernel form, and which tiles are cut along their keys.
#include <algorithm>

#include "sfe_ops.hpp"

namespace sfe {
namespace {

// Keys that queries [i0, i1] of a sequence can see: [*lo, *hi).
void key_range(int64_t lq, int64_t lk, int64_t i0, int64_t i1, int32_t left, int32_t right, int64_t* lo, int64_t* hi) {
  const int64_t c = lk - lq;
  *lo = left == kAttnNoBound ? 0 : std::max<int64_t>(0, i0 + c - left);
  *hi = right == kAttnNoBound ? lk : std::min<int64_t>(lk, i1 + c + right + 1);
  if (*hi < *lo) *hi = *lo;
}

struct Tile {
  int64_t q_row, k_row;
  int32_t lq, lk, row0, kv0, kv1;
};

// Cuts each tile's keys into pieces of at most `most` keys (a multiple of
// `unit`), equal within a unit.
void cut(const std::vector<Tile>& tiles, int64_t most, int unit, AttnForm* f) {
  for (const Tile& t : tiles) {
    const int64_t keys = t.kv1 - t.kv0;
    const int64_t n = keys > most ? (keys + most - 1) / most : 1;
    AttnItem it{t.q_row, t.k_row, t.lq, t.lk, t.row0, t.kv0, t.kv1, -1, {0, 0}};
    if (n == 1) {
      f->items.push_back(it);
      continue;
    }
    const int64_t units = (keys + unit - 1) / unit;
    f->joins.push_back(AttnJoin{t.q_row, t.lq, t.row0, f->parts, (int32_t)n});
    for (int64_t p = 0; p < n; ++p) {
      it.kv0 = (int32_t)(t.kv0 + units * p / n * unit);
      it.kv1 = (int32_t)std::min<int64_t>(t.kv1, t.kv0 + units * (p + 1) / n * unit);
      it.part = f->parts++;
      f->items.push_back(it);
    }
  }
}

// The longest piece for which the tiles' pieces fill `slots` workgroups about
// once (no cut where the tiles alone do), at least `least` keys.
int64_t piece_keys(const std::vector<Tile>& tiles, int kv_heads, int64_t slots, int64_t least) {
  int64_t total = 0, longest = 0;
  for (const Tile& t : tiles) {
    total += t.kv1 - t.kv0;
    longest = std::max<int64_t>(longest, t.kv1 - t.kv0);
  }
  total *= kv_heads;
  return std::max(least, std::min(longest, (total + slots - 1) / slots));
}

}  // namespace

void attn_plan(const int64_t* q_offsets, const int64_t* k_offsets, int n, int group, int kv_heads, int head_dim,
               int32_t left, int32_t right, int cus, AttnPlanHost* out) {
  (void)head_dim;
  std::vector<Tile> tiles[kAttnForms];
  for (int s = 0; s < n; ++s) {
    const int64_t lq = q_offsets[s + 1] - q_offsets[s], lk = k_offsets[s + 1] - k_offsets[s];
    const int64_t total = lq * group;
    const int form = total <= kAttnTileFew ? kAttnFew : (total <= kAttnTileRows ? kAttnRows : kAttnTall);
    const int tile = attn_tile(form);
    // (the last tiles of a causal sequence see the most keys: they go first)
    for (int64_t t = (total + tile - 1) / tile - 1; t >= 0; --t) {
      int64_t lo, hi;
      key_range(lq, lk, t * tile / group, (std::min(total, (t + 1) * tile) - 1) / group, left, right, &lo, &hi);
      tiles[form].push_back(
          Tile{q_offsets[s], k_offsets[s], (int32_t)lq, (int32_t)lk, (int32_t)(t * tile), (int32_t)lo, (int32_t)hi});
    }
  }
  for (int form = 0; form < kAttnForms; ++form) {
    const int unit = form == kAttnFew ? kAttnWavesFew * kAttnStepFew : kAttnStepRows;
    const int64_t slots = form == kAttnRows ? 2 * cus : cus;
    cut(tiles[form], piece_keys(tiles[form], kv_heads, slots, form == kAttnFew ? 2 * unit : 4 * unit), unit, &out->form[form]);
  }
}

}  // namespace sfe
