// csrc/sequence_search.h on the CPU. A line "SEQUENCES ROW LENGTHS SIDE" on stdin asks for the
// sequence that a row lies in, among the starts 0, 3, 3, 6, 6, 9, ... (LENGTHS 1:
// with lengths, 100 + b). The starts and lengths lie at the beginning (SIDE 0) or the
// end (SIDE 1) of memory that nothing around may be read of.
#include "wave_shim.h"

#include "sequence_search.h"

int main() {
  int n, with_lengths, side;
  long long row;
  while (std::scanf("%d %lld %d %d", &n, &row, &with_lengths, &side) == 4) {
    int32_t* starts = guarded(n + 1, side);
    int32_t* lengths = with_lengths ? guarded(std::max(n, 1), side) : nullptr;
    for (int b = 0; b <= n; ++b) starts[b] = (b + 1) / 2 * 3;
    for (int b = 0; with_lengths && b < n; ++b) lengths[b] = 100 + b;
    w8a8::SequenceRow r[64];
    wave([&](int lane) { r[lane] = w8a8::sequence_of(starts, n, row, lengths); });
    for (int i = 1; i < 64; ++i)
      if (r[i].b != r[0].b || r[i].first != r[0].first || r[i].last != r[0].last || r[i].length != r[0].length) return 2;
    std::printf("%d %d %d %d\n", r[0].b, r[0].first, r[0].last, r[0].length);
    std::fflush(stdout);
  }
}
