// The tiles that packed sequences are cut into, found by a wave. Apart from the
// other device code, so that a CPU build can run it lane by lane.
#pragma once

#include "sequence_search.h"

namespace w8a8 {

constexpr int kPackWaves = 4;
constexpr int kPackQ = 32 * kPackWaves;

__device__ __forceinline__ int clamp_to(int v, int lo, int hi) { return min(max(v, lo), hi); }

// The sequence and the tile of key head's tile t. A tile's rows are a sequence's
// queries with the heads of the group, query by query: short sequences fill it,
// and a causal one's tile spans few queries. The tiles of a sequence come from its
// last (of causal ones the longest) to its first, and of fewer than kPackSearch
// sequences those with the most keys come first, so that what is left at the end
// is short (five images, 21591 rows, 662 -> 642 us; of ten prompts and
// more the order costs more than it gives: 101 us against 94). Behind the
// sequences come the tiles of the rows behind them, as a sequence without keys.
struct PackedTile {
  int b, first, n;     // first row of the tile in its sequence, the sequence's rows
  int row0, key0, nk;  // the sequence's first query, first key and keys
};
constexpr PackedTile kNoTile = {-1, 0, 0, 0, 0, 0};
constexpr int kPackSearch = 8;

// More sequences: sequence b has the tiles from start_b / kPackQ + b on (start_b
// times the group), at least as many as it fills, and of these at most one more.
// That needs no sums over the sequences before it, and 64 of them are looked at
// at once (300 prompts of 8 rows 71 -> 38 us, 4096 of 4 rows 2394 -> 439).
template <typename Params>
__device__ __forceinline__ PackedTile packed_search(const Params& p, int t) {
  const int lane = threadIdx.x & 63;
  auto place = [&](int b) { return clamp_to(p.starts[b], 0, p.rows) * p.group / kPackQ + b; };
  int b = 0;
  for (int size = p.sequences + 1; size > 1;) {
    const int step = (size + 63) / 64, at = lane * step;
    const int skip = last_lane(at < size && place(b + min(at, size - 1)) <= t) * step;
    b += skip;
    size = min(step, size - skip);
  }
  PackedTile r;
  const bool behind = b == p.sequences;
  r.b = b;
  r.row0 = clamp_to(scalar_int(p.starts, b), 0, p.rows);
  r.n = ((behind ? p.rows : clamp_to(scalar_int(p.starts, b + 1), r.row0, p.rows)) - r.row0) * p.group;
  r.key0 = behind ? 0 : clamp_to(scalar_int(p.k_starts, b), 0, p.keys);
  r.nk = behind ? 0 : clamp_to(scalar_int(p.k_starts, b + 1), r.key0, p.keys) - r.key0;
  const int tiles = (r.n + kPackQ - 1) / kPackQ, i = t - (r.row0 * p.group / kPackQ + b);
  if (i < 0 || i >= tiles) return kNoTile;
  r.first = (tiles - 1 - i) * kPackQ;
  return r;
}

template <typename Params>
__device__ __forceinline__ PackedTile packed_find(const Params& p, int t) {
  if (p.sequences >= kPackSearch) return packed_search(p, t);
  const int b = threadIdx.x & 63;
  int lo = 0, n = 0, key0 = 0, nk = -1;
  if (b <= p.sequences) {
    lo = clamp_to(p.starts[b], 0, p.rows);
    n = (clamp_to(b < p.sequences ? p.starts[b + 1] : p.rows, lo, p.rows) - lo) * p.group;
    if (b < p.sequences) {
      key0 = clamp_to(p.k_starts[b], 0, p.keys);
      nk = clamp_to(p.k_starts[b + 1], key0, p.keys) - key0;
    }
  }
  const int tiles = (n + kPackQ - 1) / kPackQ;
  int before = 0;   // tiles of the sequences that come first
  for (int j = 0; j <= p.sequences; ++j) {
    const int other = __builtin_amdgcn_readlane(nk, j), theirs = __builtin_amdgcn_readlane(tiles, j);
    if (other > nk || (other == nk && j < b)) before += theirs;
  }
  const uint64_t here = __builtin_amdgcn_ballot_w64(b <= p.sequences && before <= t && t < before + tiles);
  if (here == 0) return kNoTile;
  const int at = __builtin_ctzll(here);
  PackedTile r;
  r.b = at;
  r.row0 = __builtin_amdgcn_readlane(lo, at);
  r.n = __builtin_amdgcn_readlane(n, at);
  r.key0 = __builtin_amdgcn_readlane(key0, at);
  r.nk = max(__builtin_amdgcn_readlane(nk, at), 0);
  r.first = (__builtin_amdgcn_readlane(before + tiles, at) - 1 - t) * kPackQ;
  return r;
}

}  // namespace w8a8
