// csrc/packed_tiles.h on the CPU. A line "ROWS KEYS SEQUENCES GROUP SIDE", with the
// starts and the keys' starts behind it, asks for the tiles of a key head as a call
// launches them: each as "b first n row0 key0 nk", b -1 where there is none.
#include "wave_shim.h"

#include "packed_tiles.h"

struct Params {
  const int32_t* starts;
  const int32_t* k_starts;
  int rows, keys, sequences, group;
};

int main() {
  Params p;
  int side;
  while (std::scanf("%d %d %d %d %d", &p.rows, &p.keys, &p.sequences, &p.group, &side) == 5) {
    int32_t* at[2] = {guarded(p.sequences + 1, side), guarded(p.sequences + 1, side)};
    for (int32_t* x : at)
      for (int b = 0; b <= p.sequences; ++b)
        if (std::scanf("%d", x + b) != 1) return 3;
    p.starts = at[0];
    p.k_starts = at[1];
    const int tiles = (int)((int64_t)p.rows * p.group / w8a8::kPackQ) + p.sequences + 1;
    std::vector<w8a8::PackedTile> found[64];
    wave([&](int lane) {
      for (int t = 0; t < tiles; ++t) found[lane].push_back(w8a8::packed_find(p, t));
    });
    std::printf("%d\n", tiles);
    for (int t = 0; t < tiles; ++t) {
      const w8a8::PackedTile r = found[0][t];
      for (int i = 1; i < 64; ++i) {
        const w8a8::PackedTile o = found[i][t];
        if (o.b != r.b || o.first != r.first || o.n != r.n || o.row0 != r.row0 || o.key0 != r.key0 || o.nk != r.nk) return 2;
      }
      std::printf("%d %d %d %d %d %d\n", r.b, r.first, r.n, r.row0, r.key0, r.nk);
    }
    std::fflush(stdout);
  }
}
