// Host run of the attention's planner (scriptrs_amd/csrc/sfe_attn_plan.cpp): for random batches,
// windows and head groups, every (packed row, visible key) pair must lie in exactly one
// piece, pieces of a tile must be joined once, and the XCDs' shares must cover the units.  Argument: seed.
// Prints "bad N".
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>

#include "sfe_ops.hpp"

int main(int argc, char** argv) {
  std::mt19937 rng((unsigned)(argc > 1 ? atoi(argv[1]) : 1));
  auto pick = [&](int lo, int hi) { return (int)(lo + rng() % (unsigned)(hi - lo + 1)); };
  int64_t bad = 0;
  for (int trial = 0; trial < 200; ++trial) {
    const int n = pick(0, 6), group = 1 << pick(0, 3), kv_heads = pick(1, 8), dim = 8 * pick(1, 16);
    const int most = trial % 4 == 0 ? 3000 : 300;
    const int32_t left = pick(0, 2) ? sfe::kAttnNoBound : pick(0, 400), right = pick(0, 1) ? sfe::kAttnNoBound : pick(0, 40);
    std::vector<int64_t> q(1, 0), k(1, 0);
    const int kind = pick(0, 2);
    for (int s = 0; s < n; ++s) {
      const int lk = pick(0, most), lq = kind == 0 ? lk : (kind == 1 ? pick(0, 4) : pick(0, most));
      q.push_back(q.back() + lq);
      k.push_back(k.back() + lk);
    }
    sfe::AttnPlanHost plan;
    sfe::attn_plan(q.data(), k.data(), n, group, kv_heads, dim, left, right, 256, &plan);
    std::map<int64_t, std::vector<int64_t>> seen;  // first query row -> keys seen by each packed row
    for (int s = 0; s < n; ++s)
      if (q[s + 1] > q[s]) seen[q[s]].assign((size_t)((q[s + 1] - q[s]) * group), 0);
    std::map<int64_t, int64_t> keys_of;
    for (int s = 0; s < n; ++s)
      if (q[s + 1] > q[s]) keys_of[q[s]] = k[s];
    for (int form = 0; form < sfe::kAttnForms; ++form) {
      const sfe::AttnForm& f = plan.form[form];
      const int tile = sfe::attn_tile(form);
      std::vector<int> part_joined((size_t)f.parts, 0), part_made((size_t)f.parts, 0);
      std::map<int32_t, const sfe::AttnJoin*> join_of;
      for (const sfe::AttnJoin& j : f.joins)
        for (int p = 0; p < j.parts; ++p) {
          if (j.part0 + p >= f.parts) { ++bad; continue; }
          ++part_joined[(size_t)(j.part0 + p)];
          join_of[j.part0 + p] = &j;
        }
      for (const sfe::AttnItem& it : f.items) {
        auto at = seen.find(it.q_row);
        if (at == seen.end() || keys_of[it.q_row] != it.k_row || it.kv0 < 0 || it.kv1 > it.lk || it.kv1 < it.kv0) { ++bad; continue; }
        if (it.part >= 0) {
          if (it.part >= f.parts || !join_of.count(it.part)) { ++bad; continue; }
          ++part_made[(size_t)it.part];
          const sfe::AttnJoin* j = join_of[it.part];
          if (j->q_row != it.q_row || j->row0 != it.row0 || j->lq != it.lq) ++bad;
        }
        for (int64_t r = it.row0; r < it.row0 + tile && r < (int64_t)it.lq * group; ++r) {
          const int64_t i = r / group + it.lk - it.lq;
          const int64_t lo = left == sfe::kAttnNoBound ? 0 : std::max<int64_t>(0, i - left);
          const int64_t hi = right == sfe::kAttnNoBound ? it.lk - 1 : std::min<int64_t>(it.lk - 1, i + right);
          const int64_t a = std::max<int64_t>(lo, it.kv0), b = std::min<int64_t>(hi, it.kv1 - 1);
          if (b >= a) at->second[(size_t)r] += b - a + 1;
        }
      }
      for (int32_t p = 0; p < f.parts; ++p) bad += part_joined[(size_t)p] != 1 || part_made[(size_t)p] != 1;
      if (f.share[0] != 0 || f.share[8] != (int64_t)f.items.size() * kv_heads) ++bad;
      for (int x = 0; x < 8; ++x) bad += f.share[x + 1] < f.share[x];
    }
    for (int s = 0; s < n; ++s)
      for (int64_t r = 0; r < (q[s + 1] - q[s]) * group; ++r) {
        const int64_t lq = q[s + 1] - q[s], lk = k[s + 1] - k[s], i = r / group + lk - lq;
        const int64_t lo = left == sfe::kAttnNoBound ? 0 : std::max<int64_t>(0, i - left);
        const int64_t hi = right == sfe::kAttnNoBound ? lk - 1 : std::min<int64_t>(lk - 1, i + right);
        // (pieces do not overlap if every row counts each of its keys once: counted from disjoint ranges below)
        if (seen[q[s]][(size_t)r] != std::max<int64_t>(0, hi - lo + 1)) ++bad;
      }
    // ranges of one tile do not overlap
    for (int form = 0; form < sfe::kAttnForms; ++form) {
      std::map<std::pair<int64_t, int32_t>, int32_t> end;
      for (const sfe::AttnItem& it : plan.form[form].items) {
        auto key = std::make_pair(it.q_row, it.row0);
        if (end.count(key) && it.kv0 < end[key]) ++bad;
        end[key] = it.kv1;
      }
    }
  }
  printf("bad %lld\n", (long long)bad);
  return 0;
}
