// The search for a packed row's sequence, by a wave. Apart from the other device
// code, so that a CPU build can run it lane by lane.
#pragma once

#include <stdint.h>

namespace w8a8 {

// The last of the lanes with x (0 if there is none).
__device__ __forceinline__ int last_lane(bool x) {
  const uint64_t m = __builtin_amdgcn_ballot_w64(x);
  return m ? 63 - __builtin_clzll(m) : 0;
}

// The sequence b in [0, n) with starts[b] <= row < starts[b + 1], or n, with its
// two starts and its length, if lengths are given (a wave works together; the
// row is the wave's). The lanes look at 64 sequences at once, where there are more
// first at the starts of 64 ranges of them (16384 rows of 4096 sequences written
// as codes 42.7 -> 25.7 us, against all in turn; 20000 of one row 162 -> 34).
struct SequenceRow {
  int b, first, last, length;
};
// The first of 64 sequences or fewer among which the row's lies, if there is one.
__device__ __forceinline__ int sequence_window(const int32_t* starts, int n, int64_t row) {
  const int lane = threadIdx.x & 63;
  int b = 0, size = n;
  while (size > 64) {
    const int step = (size + 63) / 64, at = lane * step;
    const int skip = last_lane(at < size && starts[b + min(at, size - 1)] <= row) * step;
    b += skip;
    size = min(step, size - skip);
  }
  return b;
}
__device__ __forceinline__ SequenceRow sequence_of(const int32_t* starts, int n, int64_t row, const int32_t* lengths) {
  if (n <= 0) return {n, 0, 0, 0};   // (the starts are one, and no sequence has a start and an end)
  const int lane = threadIdx.x & 63, b = sequence_window(starts, n, row);
  const int i = min(b + lane, n - 1);
  const int first = starts[i], last = starts[i + 1], length = lengths ? lengths[i] : 0;
  const uint64_t in = __builtin_amdgcn_ballot_w64(b + lane < n && first <= row && row < last);
  if (in == 0) return {n, 0, 0, 0};
  const int at = __builtin_ctzll(in);
  return {b + at, __builtin_amdgcn_readlane(first, at), __builtin_amdgcn_readlane(last, at),
          __builtin_amdgcn_readlane(length, at)};
}

}  // namespace w8a8
