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

// The longest piece for which the tiles' pieces fill `slots` workgroups about once, at least
// `least` keys; tiles of up to `whole` keys are not cut (adding the pieces up is one more launch).
int64_t piece_keys(const std::vector<Tile>& tiles, int kv_heads, int64_t slots, int64_t least, int64_t whole) {
  int64_t total = 0, longest = 0;
  for (const Tile& t : tiles) {
    total += t.kv1 - t.kv0;
    longest = std::max<int64_t>(longest, t.kv1 - t.kv0);
  }
  if (longest <= whole) return std::max(least, longest);
  total *= kv_heads;
  return std::max(least, std::min(longest, (total + slots - 1) / slots));
}

// Time of a sequence's tiles in a form, in microseconds of a CU: steps and a fixed part a tile,
// fitted to 40,000 rows of 8 heads of 128 (steps of 2.03 us for 256 rows, 1.31 for 128).  Measured
// on both sides (rows / tall, us; such a call fills the chip):
//   full attention of 188, 260, 384, 512, 1024, 4096 keys
//     heads of 128   96 / 107, 130 / 177, 122 / 140, 147 / 131, 238 / 197, 757 / 600
//     heads of 96    72 / 87, 100 / 140, 85 / 109, 102 / 104, 175 / 158, 628 / 502
//     heads of 80    75 / 85, 99 / 137, 84 / 106, 104 / 100, 174 / 153, 626 / 488
//   causal 384, 512, 768, 4096
//     heads of 128   101 / 120, 132 / 122, 146 / 128, 397 / 356
//     heads of 96    74 / 96, 97 / 100, 113 / 102, 334 / 302
//     heads of 80    73 / 93, 97 / 98, 112 / 99, 326 / 293
//   windows of 64, 256, 512, 1024 to either side
//     heads of 128   94 / 110, 150 / 158, 236 / 224, 406 / 377
//     heads of 96    77 / 95, 129 / 133, 200 / 191, 345 / 311
//     heads of 80    77 / 93, 126 / 131, 197 / 187, 337 / 301
// It chooses the shorter one in all of them but causal 512 in heads of 80 and 96 and full 512 in
// heads of 96 (1-3% longer).  Heads of 64 channels and less leave room for 3 workgroups of the rows
// form on a CU, which is then faster everywhere (4096 keys 695 / 727 us, 512 119 / 145).
// A call that leaves CUs empty is not what was fitted: one sequence of 700 rows in 8 heads of 128
// takes 25 (rows) / 29 (tall, as chosen), of 2000 51 / 50, of 4000 107 / 102.
double tile_costs(int form, int64_t lq, int64_t lk, int group, int32_t left, int32_t right) {
  const bool causal = left == kAttnNoBound && right == 0;
  const double step = form == kAttnTall ? 2.03 : 1.31, fixed = form == kAttnTall ? (causal ? 10.0 : 13.0) : 5.2;
  const int64_t tile = attn_tile(form), total = lq * group;
  double cost = 0.0;
  for (int64_t t = 0; t * tile < total; ++t) {
    int64_t lo, hi;
    key_range(lq, lk, t * tile / group, (std::min(total, (t + 1) * tile) - 1) / group, left, right, &lo, &hi);
    cost += fixed + step * (double)((hi - lo + kAttnStepRows - 1) / kAttnStepRows);
    if (t == 4096) return cost * ((double)total / (double)((t + 1) * tile));  // (long enough to tell)
  }
  return cost;
}

// Whether the few form takes the whole call: only sequences of up to 16 packed rows, or so few
// tiles of 16 that they get a CU each and not many keys, so that the whole call is one trip
// through memory.  One sequence of 250, 500, 700, 1125, 2000, 4000 rows in 8 heads, in this form / the
// faster of the others: heads of 128 9.1 / 13.3 us, 11.9 / 21.4, 23.9 / 25.3, 42.6 / 37.6, 83.5 / 50.2, 283 / 102; of 64
// 7.2 / 11.0, 8.7 / 17.8, 11.2 / 20.4, 20.7 / 30.0, 32.8 / 41.7, 104 / 82.  (The bound of 5 tiles to 4 CUs, up to 640
// rows here, fits heads of 128; heads of 64 would go on to about 2000.)
bool whole_call_few(const int64_t* q_offsets, const int64_t* k_offsets, int n, int group, int kv_heads, int cus) {
  int64_t units = 0, rows = 0, keys = 0;
  for (int s = 0; s < n; ++s) {
    const int64_t total = (q_offsets[s + 1] - q_offsets[s]) * group;
    units += (total + kAttnTileFew - 1) / kAttnTileFew * kv_heads;
    rows = std::max(rows, total);
    keys = std::max(keys, k_offsets[s + 1] - k_offsets[s]);
  }
  return rows <= kAttnTileFew || (units <= cus * 5 / 4 && keys <= 2048);
}

// The form of a sequence of a call that does not take the few form as a whole: few for up to 16 packed rows
// over many keys (a launch of its own for a few short ones would cost more than their place
// among the rows: 256 clips of 13-251 frames 51 us with it, 46 without).
int form_of(int64_t lq, int64_t lk, int group, int head_dim, int32_t left, int32_t right, bool all_few) {
  const int64_t total = lq * group;
  if (all_few || (total <= kAttnTileFew && lk >= 1024)) return kAttnFew;
  if (total <= kAttnTileRows || attn_padded_dim(head_dim) <= 64) return kAttnRows;
  return tile_costs(kAttnTall, lq, lk, group, left, right) < tile_costs(kAttnRows, lq, lk, group, left, right) ? kAttnTall
                                                                                                              : kAttnRows;
}

// Cuts the units (kv head by kv head, in a head the items in order) into 8 shares of about equal
// work, one an XCD.
void share_out(int kv_heads, AttnForm* f) {
  const int64_t n = (int64_t)f->items.size();
  std::fill(f->share, f->share + 9, 0);
  if (n == 0) return;  // (no work to have a part of)
  std::vector<double> sum((size_t)n + 1, 0.0);
  for (int64_t i = 0; i < n; ++i) {
    const AttnItem& it = f->items[(size_t)i];
    sum[(size_t)i + 1] = sum[(size_t)i] + 4.0 + (double)((it.kv1 - it.kv0 + kAttnStepRows - 1) / kAttnStepRows);
  }
  for (int x = 1; x < 8; ++x) {
    const double at = sum[(size_t)n] * kv_heads * x / 8.0;
    const int64_t head = std::min<int64_t>(kv_heads - 1, (int64_t)(at / sum[(size_t)n]));
    const double rest = at - (double)head * sum[(size_t)n];
    const int64_t i = std::lower_bound(sum.begin(), sum.end(), rest - 1e-6 * sum[(size_t)n]) - sum.begin();
    f->share[x] = std::max<int32_t>(f->share[x - 1], (int32_t)std::min<int64_t>(head * n + i, n * kv_heads));
  }
  f->share[8] = (int32_t)(n * kv_heads);
}

}  // namespace

void attn_plan(const int64_t* q_offsets, const int64_t* k_offsets, int n, int group, int kv_heads, int head_dim,
               int32_t left, int32_t right, int cus, AttnPlanHost* out) {
  const bool all_few = whole_call_few(q_offsets, k_offsets, n, group, kv_heads, cus);
  std::vector<Tile> tiles[kAttnForms];
  for (int s = 0; s < n; ++s) {
    const int64_t lq = q_offsets[s + 1] - q_offsets[s], lk = k_offsets[s + 1] - k_offsets[s];
    const int64_t total = lq * group;
    const int form = form_of(lq, lk, group, head_dim, left, right, all_few);
    const int tile = attn_tile(form);
    // (the last tiles of a causal sequence see the most keys: they go first)
    for (int64_t t = (total + tile - 1) / tile - 1; t >= 0; --t) {
      int64_t lo, hi;
      key_range(lq, lk, t * tile / group, (std::min(total, (t + 1) * tile) - 1) / group, left, right, &lo, &hi);
      tiles[form].push_back(
          Tile{q_offsets[s], k_offsets[s], (int32_t)lq, (int32_t)lk, (int32_t)(t * tile), (int32_t)lo, (int32_t)hi});
    }
  }
  // (64 single-token steps of 4 beams over 126-1500 keys, 4 kv heads: 27 us cut to 256 workgroups' worth,
  // 21 whole; 4 over 2000 keys 22.6 whole)
  const int unit_few = kAttnWavesFew * kAttnStepFew;
  auto lay = [&](int form, int unit, int64_t slots, int64_t least, int64_t whole) {
    cut(tiles[form], piece_keys(tiles[form], kv_heads, slots, least, whole), unit, &out->form[form]);
    share_out(kv_heads, &out->form[form]);
  };
  lay(kAttnTall, kAttnStepRows, cus, 4 * kAttnStepRows, 0);
  lay(kAttnRows, kAttnStepRows, 2 * cus, 4 * kAttnStepRows, 0);
  lay(kAttnFew, unit_few, cus, 4 * unit_few, 2 * (int64_t)tiles[kAttnFew].size() * kv_heads >= cus ? 2048 : 768);
}

}  // namespace sfe
