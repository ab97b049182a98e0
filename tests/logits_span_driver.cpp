// Checks the spans of a row's logits (scriptrs_amd/csrc/sfe_decode.hpp) on the host: every token of the row lies in one
// span, and no token, of the row or not, has a place outside its span's counts.
#include <cstdio>

#include "sfe_decode.hpp"

namespace {

// Tokens next to a span's and a row's ends, and those of other spans.
int check(int vocab, int n, int span, int before) {
  const int spans = sfe::logits_spans(vocab, n, span);
  int64_t there = 0;
  for (int i = 0; i < spans; ++i) {
    const sfe::LogitsSpan s = sfe::logits_span(i, span, before, vocab);
    if (s.tokens > (uint32_t)span) {
      std::printf("vocab %d, vectors of %d, span %d of %d, %d before: %u tokens\n", vocab, n, i, span, before, s.tokens);
      return 1;
    }
    there += s.tokens;
    const int64_t near[] = {-2147483647 - 1, -1, 0, 1, vocab - 1, vocab, s.first, s.first + span, (int64_t)s.first + 2 * span, s.first - span, 2147483647};
    for (int64_t around : near)
      for (int64_t token = around - 9; token <= around + 9; ++token) {
        if (token < -2147483647 - 1 || token > 2147483647) continue;
        const int at = s.has((int32_t)token) ? s.place((int32_t)token) : -1;
        const bool mine = token >= 0 && token < vocab && token >= s.first && token < (int64_t)s.first + span;
        if (at != (mine ? (int)(token - s.first) : -1)) {
          std::printf("vocab %d, vectors of %d, span %d of %d, %d before: token %lld at %d\n", vocab, n, i, span, before, (long long)token, at);
          return 1;
        }
      }
  }
  if (there != vocab) std::printf("vocab %d, vectors of %d, spans of %d, %d before: %lld tokens\n", vocab, n, span, before, (long long)there);
  return there != vocab;
}

}  // namespace

int main() {
  const int forms[][2] = {{1, 1024}, {4, 4096}, {4, 8192}, {8, 4096}, {8, 8192}};
  for (const auto& f : forms)
    for (int before = 0; before < f[0]; ++before) {
      for (int vocab = 1; vocab <= 40; ++vocab)
        if (check(vocab, f[0], f[1], before)) return 1;
      for (int k = 1; k <= 16; ++k)
        for (int vocab = 1024 * k - 12; vocab <= 1024 * k + 12; ++vocab)
          if (check(vocab, f[0], f[1], before)) return 1;
      for (int vocab = (1 << 24) - 12; vocab <= 1 << 24; ++vocab)
        if (check(vocab, f[0], f[1], before)) return 1;
    }
  std::puts("ok");
  return 0;
}
