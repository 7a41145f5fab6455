// A wave of 64 lanes on the CPU, for device code that searches: 64 threads, which
// meet where lanes exchange values, and integers with nothing readable around them.
#pragma once

#include <pthread.h>
#include <stdint.h>
#include <sys/mman.h>
#include <unistd.h>

#include <algorithm>
#include <cstdio>
#include <cstdlib>
#include <thread>
#include <vector>

#define __device__
#define __forceinline__ inline
using std::max;
using std::min;

static thread_local struct { unsigned x; } threadIdx;
static pthread_barrier_t meet;
static bool voted[64];
static int held[64];

static uint64_t __builtin_amdgcn_ballot_w64(bool x) {
  voted[threadIdx.x] = x;
  pthread_barrier_wait(&meet);
  uint64_t m = 0;
  for (int i = 0; i < 64; ++i) m |= (uint64_t)voted[i] << i;
  pthread_barrier_wait(&meet);
  return m;
}
static int __builtin_amdgcn_readlane(int v, int lane) {
  held[threadIdx.x] = v;
  pthread_barrier_wait(&meet);
  const int r = held[lane];
  pthread_barrier_wait(&meet);
  return r;
}
static int scalar_int(const int32_t* p, int64_t i) { return p[i]; }

// n integers at the beginning (side 0) or the end (side 1) of memory of their own.
static int32_t* guarded(int n, int side) {
  const size_t page = (size_t)sysconf(_SC_PAGESIZE), bytes = 4 * (size_t)n, whole = (bytes + page - 1) / page * page;
  char* at = static_cast<char*>(mmap(nullptr, whole + 2 * page, PROT_NONE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0));
  if (at == MAP_FAILED || mprotect(at + page, whole, PROT_READ | PROT_WRITE)) std::abort();
  return reinterpret_cast<int32_t*>(at + page + (side ? whole - bytes : 0));
}

// f(lane) on every lane at once.
template <typename F>
static void wave(F f) {
  pthread_barrier_init(&meet, nullptr, 64);
  std::vector<std::thread> lanes;
  for (unsigned lane = 0; lane < 64; ++lane)
    lanes.emplace_back([&f, lane] {
      threadIdx.x = lane;
      f((int)lane);
    });
  for (std::thread& t : lanes) t.join();
  pthread_barrier_destroy(&meet);
}
