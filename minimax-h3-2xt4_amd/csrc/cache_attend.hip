// Attention of one new token of every sequence over a paged cache.
//
//   o = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m),  t_j = log2(e) scale q . k_j
//
// in one pass, every key read once, with a reference m that follows the running
// maximum. A query head does 4 flops per element read, so even sixteen heads on
// one kv head are far from the MFMA's rate (3 to 5 % of it): HBM bounds this, and
// the work is cut by keys. All keys of all (sequence, kv head) pairs, in blocks of
// 128, are one line that is cut into equal ranges, one for each workgroup,
// whatever the sequences' lengths; a pair inside one range is finished there, one
// that several ranges share leaves partial sums, which a second kernel joins in
// order. Loads run a block ahead, over the pairs' ends too.
//
// 131072 keys of 8 heads of 128 in bf16, 64 query heads (537 MB): 82 us and 5 for
// the join, 6.2 TB/s in all; 64 contexts of 261850 keys as codes (555 MB): 95 us
// and 5; 354 keys: 7 us, the launch and one pass of latencies. Four waves a
// workgroup and two of them a CU keep 8 KB and more a wave under way.
//
// A wave takes 32 keys of a block (two groups of 16, each within a page), and
// up to 16 query heads of the pair, straight from memory into the operands:
//   S[key][head] = K Q^T  on the 16 x 16 x 32 MFMA, keys as rows: lane l reads
//     key l % 16, channels 8 (l / 16) + 32 s, which is how rows lie in memory.
//   O[channel][head] += V^T P^T: S leaves lane l with the keys 4 (l / 16) + r of
//     both groups for head l % 16, and the same lane reads those eight keys'
//     channels VL (l % 16) + j. Its eight keys are then the eight k of an
//     operand (any order of k is as good, if both operands have it), and P
//     needs no exchange between lanes; pairs of keys of one channel are picked
//     by v_perm_b32. Row i of product j is channel VL i + j.
// Nothing passes through LDS before the waves' sums meet at the pair's end.
//
// Keys behind the end and pages that are not there are cut off by the buffer
// descriptor of their group: their loads return zeros, whatever memory holds.
#include "paged.h"

#include <algorithm>

namespace w8a8 {

constexpr int kAttendWaves = 4;
constexpr int kHeadTile = 16;
constexpr int kWaveKeys = 32;   // keys of a wave at a time: two groups
constexpr int kBlockKeys = kAttendWaves * kWaveKeys;
// dim rounded up to the channels that a kernel works on.
constexpr int attend_dp(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }
// Workgroups that a CU's ranges are cut for: with one of eight waves, the ends of
// pairs leave it idle (64 contexts of codes 115 -> 124 us), with three there are more
// ends (94.5 -> 104). Registers are for three, which calls of a workgroup for each
// pair fill (1024 contexts of 200 keys as codes 131 -> 110 us). 256 channels are one
// workgroup's, all registers: with two that spill, 64 contexts of 4096 keys took
// 394 us instead of 349.
constexpr int attend_per_cu(int dim) { return dim > 128 ? 1 : 2; }
constexpr int attend_fit(int dim) { return dim > 128 ? 1 : 3; }
// Codes: P is p times the value's scale, and relative to a reference of its own, of
// what keys contribute, so that no key's scale takes precision from keys of more
// weight (relative to the largest scale, a row 2^18 times the others' with a weight
// of 2^-46 left the output 4 % off). That reference is a power of 2, the largest
// product so far at most kPartSlack times it, and P relative to 1 / kPartLift of it:
// at most 2^15, of fp16's 2^16, and what is lost lies below 2^-32 of the largest. p
// is at most 1, so that its product with the largest scale of bf16 rows, 2^121, is finite.
constexpr float kPartSlack = 256.0f, kPartLift = 128.0f, kLeastPart = 0x1p-119f;
// kPartLift / x of a power of 2 from kLeastPart on (of 0 some finite value).
__device__ __forceinline__ float part_inv(float x) { return __uint_as_float((261u << 23) - __float_as_uint(x)); }
__device__ __forceinline__ float power_of_2(float x) { return __uint_as_float(__float_as_uint(x) & 0x7f800000u); }

struct AttendParams {
  CacheView cache;
  const char* q;
  char* out;
  int64_t q_row, q_head, o_row, o_head;   // bytes
  int sequences, heads, group, tiles;     // tiles: of 16 query heads of a kv head
  int width;
  int whole;    // a workgroup for each pair
  int stream;   // more keys and values than the last cache holds
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  float c;   // log2(e) * scale
  float* part;       // [workgroups][2][kHeadTile][dim padded]
  float* part_ml;    // [workgroups][2][2][kHeadTile]: reference, sum
  int4* shared;      // [workgroups]: sequence, pair and last range of a pair that begins in a range and goes on, or -1
};

__device__ __forceinline__ int attend_length(const AttendParams& p, int len) {
  return min(max(len, 0), p.width * p.cache.page_size);
}
// Blocks of a pair of this length; an empty sequence has a block of no keys.
__device__ __forceinline__ int attend_blocks(const AttendParams& p, int len) {
  return max((attend_length(p, len) + kBlockKeys - 1) / kBlockKeys, 1);
}

__device__ __forceinline__ int wave_sum(int v) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) v += __shfl_xor(v, off, 64);
  return __builtin_amdgcn_readfirstlane(v);
}

// The line of all pairs' blocks, cut into ranges that differ by one block at
// most: the first `extra` have per + 1.
struct Ranges {
  int per, extra, used;
  __device__ __forceinline__ Ranges(int total, int workgroups) {
    used = min(total, workgroups);
    per = total / used;
    extra = total - per * used;
  }
  __device__ __forceinline__ int begin(int g) const { return per * g + min(g, extra); }
  static __device__ __forceinline__ int of(int n, int per, int extra) {   // the range that block n lies in
    const int big = extra * (per + 1);
    return n < big ? n / (per + 1) : extra + (n - big) / per;
  }
};

// Blocks of all pairs, and of those of the sequences before one.
__device__ __forceinline__ int attend_total(const AttendParams& p) {
  int n = 0;
  for (int b = threadIdx.x & 63; b < p.sequences; b += 64) n += attend_blocks(p, p.lengths[b]);
  return wave_sum(n) * (p.cache.heads * p.tiles);
}
__device__ __forceinline__ int attend_total(const AttendParams& p, int sequence, int& before) {
  int n = 0, first = 0;
  for (int b = threadIdx.x & 63; b < p.sequences; b += 64) {
    const int mine = attend_blocks(p, p.lengths[b]);
    n += mine;
    if (b < sequence) first += mine;
  }
  before = wave_sum(first) * (p.cache.heads * p.tiles);
  return wave_sum(n) * (p.cache.heads * p.tiles);
}

// The sequence that block n of the line belongs to, and the blocks before it.
__device__ __forceinline__ int attend_find(const AttendParams& p, int n, int& before) {
  const int lane = threadIdx.x & 63, pairs = p.cache.heads * p.tiles;
  int sum = 0;
  for (int b0 = 0; b0 < p.sequences; b0 += 64) {
    const int mine = b0 + lane < p.sequences ? attend_blocks(p, p.lengths[b0 + lane]) * pairs : 0;
    int upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int t = __shfl_up(upto, off, 64);
      if (lane >= off) upto += t;
    }
    upto += sum;
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > n);
    if (past) {
      const int at = __builtin_ctzll(past);
      before = __builtin_amdgcn_readlane(upto - mine, at);
      return b0 + at;
    }
    sum = __builtin_amdgcn_readlane(upto, 63);
  }
  before = sum;
  return p.sequences;
}

template <int DT>
__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// Four codes of a word as two words of fp16 values: 0x6400 | (code + 128) is 1152 + code.
__device__ __forceinline__ v2u codes4(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;
  const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
  const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
  return v2u{__builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, lo) - off),
             __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, hi) - off)};
}

// A lane's loads of a group of 16 tokens: W words from byte offset off of its
// descriptor. AUX 2: non-temporal.
template <int W, int AUX>
__device__ __forceinline__ void group_load(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t (&w)[W]) {
  if constexpr (W == 1) {
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, AUX);
  } else if constexpr (W == 2) {
    const v2u t = __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, AUX);
    w[0] = t.x; w[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const v4u t = __builtin_amdgcn_raw_buffer_load_b128(r, (int)off + 16 * i, 0, AUX);
      w[4 * i] = t.x; w[4 * i + 1] = t.y; w[4 * i + 2] = t.z; w[4 * i + 3] = t.w;
    }
  }
}

constexpr uint32_t kNowhere = 0x7fffff00u;   // an offset behind every descriptor's end

// DT: type of q and out; CODES: the cache holds I8; DP: dim rounded up to 64, 128
// or 256; STREAM: the keys and values pass through the caches without staying.
template <int DT, bool CODES, int DP, bool STREAM>
__global__ __launch_bounds__(64 * kAttendWaves, attend_fit(DP)) void cache_attend_kernel(AttendParams p) {
  constexpr int ES = CODES ? 1 : 2, AUX = STREAM ? 2 : 0;
  // Codes are multiplied as fp16, whatever q's type: cheaper to make than bf16,
  // and P keeps eleven bits. q of bf16 is scaled by a power of 2 for it, so that a
  // head's largest is from 1 to 2: exact but for what lies 2^-14 below that.
  constexpr int MT = CODES ? kF16 : DT;
  constexpr int G = kWaveKeys / kGroupTokens;
  constexpr int NS = DP / 32;          // products of a key tile
  constexpr int VL = DP / 16;          // channels a lane reads of a value row
  // Channel of lane quad in step s of K Q^T, any order being as good as another:
  // loads are 16 bytes a lane, eight channels of a step, or with codes of two.
  constexpr int KS = CODES ? 2 : 1;
  auto channel = [](int quad, int s) { return CODES ? 64 * (s / 2) + 16 * quad + 8 * (s % 2) : 32 * s + 8 * quad; };
  constexpr int VW = VL * ES / 4;      // words of VL channels
  constexpr int kRow = DP + 4;         // a head's sums in LDS, padded
  __shared__ __attribute__((aligned(16))) float sums[kAttendWaves][kHeadTile][kRow];
  __shared__ float stat[kAttendWaves][3][kHeadTile];
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int dim = p.cache.dim;

  int b, pair, blk = 0, nblk, at = 0, end, ranges_per = 0, ranges_extra = 0;
  if (p.whole) {
    const int pairs = p.cache.heads * p.tiles;
    b = blockIdx.x / pairs;
    pair = blockIdx.x - b * pairs;
    end = nblk = attend_blocks(p, scalar_int(p.lengths, b));
  } else {
    const Ranges r(attend_total(p), gridDim.x);
    if (threadIdx.x == 0) p.shared[blockIdx.x] = make_int4(-1, 0, 0, 0);
    if ((int)blockIdx.x >= r.used) return;
    ranges_per = r.per;
    ranges_extra = r.extra;
    at = r.begin(blockIdx.x);
    end = r.begin(blockIdx.x + 1);
    int before;
    b = attend_find(p, at, before);
    nblk = attend_blocks(p, scalar_int(p.lengths, b));
    pair = (at - before) / nblk;
    blk = at - before - pair * nblk;
  }

  // Byte offsets within a group of 16 tokens.
  uint32_t koff[NS / KS], voff[4];
#pragma unroll
  for (int s = 0; s < NS / KS; ++s) {
    const int d = channel(quad, KS * s);
    koff[s] = d < dim ? col * p.cache.token_b + d * ES : kNowhere;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    voff[i] = VL * col < dim ? (4 * quad + i) * p.cache.token_b + VL * col * ES : kNowhere;

  // What is loaded runs ahead of what is computed, over the pairs' ends too: the
  // place of this wave's two groups of 16 keys in the next block, and how many
  // keys of each count.
  struct Keys {
    int page[G], token[G], n[G], kvh;
  };
  struct {
    int b, pair, blk, nblk, len, left;
  } ahead = {b, pair, blk, nblk, attend_length(p, scalar_int(p.lengths, b)), end - at};
  const int pairs = p.cache.heads * p.tiles;
  auto next_keys = [&]() {
    Keys k;
    const int k0 = (ahead.blk * kAttendWaves + wave) * kWaveKeys;
    k.kvh = ahead.pair / p.tiles;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int first = k0 + i * kGroupTokens;
      int n = ahead.left > 0 ? min(max(ahead.len - first, 0), kGroupTokens) : 0, entry, page = 0;
      group_place(p.cache, (uint32_t)first / kGroupTokens, entry, k.token[i]);
      if (n > 0) page = scalar_int(p.table, (int64_t)ahead.b * p.ld_table + entry);
      if (page < 0 || page >= p.cache.pages) page = n = 0;
      k.page[i] = page;
      k.n[i] = n;
    }
    if (--ahead.left > 0 && ++ahead.blk == ahead.nblk) {
      ahead.blk = 0;
      if (++ahead.pair == pairs) {
        ahead.pair = 0;
        const int len = scalar_int(p.lengths, ++ahead.b);
        ahead.len = attend_length(p, len);
        ahead.nblk = attend_blocks(p, len);
      }
    }
    return k;
  };
  auto group_rsrc = [&](const char* base, const Keys& k, int i) {
    const char* t = base + (int64_t)k.page[i] * p.cache.page_b + k.kvh * p.cache.head_b +
                    (int64_t)k.token[i] * p.cache.token_b;
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(t), 0,
                                             k.n[i] ? (int)((k.n[i] - 1) * p.cache.token_b) + dim * ES : 0, 0x00027000);
  };
  uint32_t kr[G][NS / KS][4], vr[4 * G][VW];
  auto load_k = [&](const Keys& k) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const auto r = group_rsrc(p.cache.k, k, i);
#pragma unroll
      for (int s = 0; s < NS / KS; ++s) group_load<4, AUX>(r, koff[s], kr[i][s]);
    }
  };
  auto load_v = [&](const Keys& k) {
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const auto r = group_rsrc(p.cache.v, k, i);
#pragma unroll
      for (int t = 0; t < 4; ++t) group_load<VW, AUX>(r, voff[t], vr[4 * i + t]);
    }
  };
  struct Scales {
    v4f k[G], v[G];
  };
  auto load_scales = [&](const Keys& k) {
    Scales sc{};
    if constexpr (!CODES) return sc;
#pragma unroll
    for (int i = 0; i < G; ++i) {
      const int64_t s = (int64_t)k.page[i] * p.cache.s_page + k.kvh * p.cache.s_head + k.token[i] + 4 * quad;
      sc.k[i] = *reinterpret_cast<const v4f*>(p.cache.ks + s);
      sc.v[i] = *reinterpret_cast<const v4f*>(p.cache.vs + s);
    }
    return sc;
  };
  Keys now = next_keys();
  load_k(now);
  load_v(now);
  Scales sc = load_scales(now);
  Keys next = next_keys();

  v4u qf[NS];
  auto load_q = [&](int seq, int pr) {
    const int kvh = pr / p.tiles, first = kHeadTile * (pr - kvh * p.tiles) + col;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int d = channel(quad, s);
      qf[s] = v4u{0, 0, 0, 0};
      if (first < p.group && d < dim)
        qf[s] = *reinterpret_cast<const v4u*>(p.q + (int64_t)seq * p.q_row + (kvh * p.group + first) * p.q_head + 2 * d);
    }
  };
  // bf16 queries as fp16 ones, and the scores' factor for them.
  float factor = p.c;
  auto convert_q = [&]() {
    if constexpr (CODES && DT == kBF16) {
      uint32_t top = 0;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) top = max(top, max(qf[s][i] & 0x7fffu, (qf[s][i] >> 16) & 0x7fffu));
      top = max(top, (uint32_t)__shfl_xor((int)top, 16, 64));
      top = max(top, (uint32_t)__shfl_xor((int)top, 32, 64));
      const int e = (int)(top >> 7) - 127;
#pragma unroll
      for (int s = 0; s < NS; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t w = qf[s][i];
          qf[s][i] = pack2<kF16>(ldexpf(__uint_as_float(w << 16), -e), ldexpf(__uint_as_float(w & 0xffff0000u), -e));
        }
      factor = ldexpf(p.c, e);
    }
  };
  load_q(b, pair);

  while (true) {
    const int kvh = pair / p.tiles, tile = pair - kvh * p.tiles;
    const int take = min(nblk - blk, end - at);
    const int nh = min(p.group - kHeadTile * tile, kHeadTile);
    const int head0 = kvh * p.group + kHeadTile * tile;
    convert_q();
    v4f o[VL];
#pragma unroll
    for (int j = 0; j < VL; ++j) o[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float ref = -INFINITY, l = 0.0f, top = 0.0f;   // top: codes' reference of P

    auto spread_max = [&](float x) {   // over the four quads: the keys of a column
      x = fmaxf(x, __shfl_xor(x, 16, 64));
      return fmaxf(x, __shfl_xor(x, 32, 64));
    };
    for (int block = 0; block < take; ++block) {
      float t[4 * G];
#pragma unroll
      for (int i = 0; i < G; ++i) {
        v4f s = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int x = 0; x < NS; ++x) {
          v4u a;
          if constexpr (CODES) {
            const v2u lo = codes4(kr[i][x / 2][2 * (x % 2)]), hi = codes4(kr[i][x / 2][2 * (x % 2) + 1]);
            a = v4u{lo.x, lo.y, hi.x, hi.y};
          } else {
            a = v4u{kr[i][x][0], kr[i][x][1], kr[i][x][2], kr[i][x][3]};
          }
          s = mfma16<MT>(a, qf[x], s);
        }
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          t[4 * i + x] = s[x] * factor;
          if constexpr (CODES) t[4 * i + x] = t[4 * i + x] * sc.k[i][x];
        }
      }
      load_k(next);
      const Scales sn = load_scales(next);
      int fewest = now.n[0];
#pragma unroll
      for (int i = 1; i < G; ++i) fewest = min(fewest, now.n[i]);
      if (fewest < kGroupTokens) {
#pragma unroll
        for (int i = 0; i < 4 * G; ++i)
          if (4 * quad + i % 4 >= now.n[i / 4]) {
            t[i] = -INFINITY;
            if constexpr (CODES) sc.v[i / 4][i % 4] = 0.0f;
          }
      }
      // The references follow the maxima only once those lie far enough above.
      auto fade_sums = [&](float fade) {
#pragma unroll
        for (int j = 0; j < VL; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][i] = o[j][i] * fade;
      };
      float mx = t[0];
#pragma unroll
      for (int i = 1; i < 4 * G; ++i) mx = fmaxf(mx, t[i]);
      if (__builtin_amdgcn_ballot_w64(mx > ref + kSlack)) {
        float to = spread_max(mx);
        if constexpr (CODES) to = floorf(to);   // (the other reference fades by powers of 2)
        to = fmaxf(ref, to);
        const float fade = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - to);
        l = l * fade;
        if constexpr (CODES) {   // O stays as it is, but for what the least reference does not hold
          const float faded = ldexpf(top, (int)fmaxf(ref - to, -300.0f));
          if (to != -INFINITY) top = fmaxf(faded, kLeastPart);
          if (__builtin_amdgcn_ballot_w64(faded != top)) fade_sums(top > 0.0f ? faded / top : 0.0f);
        } else {
          fade_sums(fade);
        }
        ref = to;
      }
      const float base = ref == -INFINITY ? 0.0f : CODES ? ref + kSlack : ref - kLift<DT>;
      float w[4 * G];
#pragma unroll
      for (int i = 0; i < 4 * G; ++i) w[i] = __builtin_amdgcn_exp2f(t[i] - base);
      if constexpr (CODES) {
        float u = 0.0f;
#pragma unroll
        for (int i = 0; i < 4 * G; ++i) {
          l += w[i];
          w[i] = w[i] * sc.v[i / 4][i % 4];
          u = fmaxf(u, fabsf(w[i]));
        }
        if (__builtin_amdgcn_ballot_w64(u > top * kPartSlack)) {
          const float to = power_of_2(fmaxf(top, spread_max(u)));
          fade_sums(to > 0.0f ? top / to : 0.0f);
          top = to;
        }
        const float inv = part_inv(top);
#pragma unroll
        for (int i = 0; i < 4 * G; ++i) w[i] = w[i] * inv;
      }
#pragma unroll
      for (int g = 0; g < G; g += 2) {
        const v4u pf = {pack2<MT>(w[4 * g], w[4 * g + 1]), pack2<MT>(w[4 * g + 2], w[4 * g + 3]),
                        pack2<MT>(w[4 * g + 4], w[4 * g + 5]), pack2<MT>(w[4 * g + 6], w[4 * g + 7])};
        if constexpr (!CODES) {   // the sum of what the values are weighted with
#pragma unroll
          for (int x = 0; x < 4; ++x) l = add2<DT>(pf[x], l);
        }
        uint32_t x[8][VL / 2];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
          for (int j = 0; j < VL / 2; j += 2) {
            if constexpr (CODES) {
              const v2u c = codes4(vr[4 * g + i][j / 2]);
              x[i][j] = c.x;
              x[i][j + 1] = c.y;
            } else {
              x[i][j] = vr[4 * g + i][j];
              x[i][j + 1] = vr[4 * g + i][j + 1];
            }
          }
#pragma unroll
        for (int j = 0; j < VL; ++j) {
          const uint32_t pick = j % 2 ? 0x07060302u : 0x05040100u;
          v4u a;
#pragma unroll
          for (int i = 0; i < 4; ++i) a[i] = __builtin_amdgcn_perm(x[2 * i + 1][j / 2], x[2 * i][j / 2], pick);
          o[j] = mfma16<MT>(a, pf, o[j]);
        }
      }
      load_v(next);
      now = next;
      sc = sn;
      next = next_keys();
    }

    if (at + take < end) load_q(pair + 1 == pairs ? b + 1 : b, pair + 1 == pairs ? 0 : pair + 1);
    // The waves' sums meet: O's lane (col, quad) holds head col, channels
    // VL (4 quad + r) + j.
    l = l + __shfl_xor(l, 16, 64);
    l = l + __shfl_xor(l, 32, 64);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < VL; j += 4)
        *reinterpret_cast<v4f*>(&sums[wave][col][VL * (4 * quad + r) + j]) = v4f{o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]};
    // Whether a wave without a score has keys is looked up here: kept up in the loop
    // it took 64 contexts of codes from 98.7 to 107.5 us.
    if (__builtin_amdgcn_ballot_w64(ref == -INFINITY && l == 0.0f)) {
      const int len = attend_length(p, scalar_int(p.lengths, b));
      bool any = false;
      for (int i = 0; i < take * G && !any; ++i) {
        const int first = ((blk + i / G) * kAttendWaves + wave) * kWaveKeys + i % G * kGroupTokens;
        if (first >= len) break;
        int entry, token;
        group_place(p.cache, (uint32_t)first / kGroupTokens, entry, token);
        const int page = scalar_int(p.table, (int64_t)b * p.ld_table + entry);
        any = page >= 0 && page < p.cache.pages;
      }
      ref = with_keys(ref, any);
    }
    if (quad == 0) {
      stat[wave][0][col] = ref;
      stat[wave][1][col] = l;
      stat[wave][2][col] = top;
    }
    __syncthreads();
    const bool whole = blk == 0 && take == nblk;
    const int slot = blockIdx.x * 2 + (blk == 0 ? 1 : 0);   // the pair begins in this range, or before it
    for (int i = threadIdx.x; i < nh * (DP / 4); i += 64 * kAttendWaves) {
      const int h = i / (DP / 4), d = 4 * (i - h * (DP / 4));
      float mx = stat[0][0][h], sum = 0.0f;
#pragma unroll
      for (int w = 1; w < kAttendWaves; ++w) mx = fmaxf(mx, stat[w][0][h]);
      const float ref = mx == -INFINITY ? 0.0f : mx;
      v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int w = 0; w < kAttendWaves; ++w) {
        const float f = __builtin_amdgcn_exp2f(stat[w][0][h] - ref);
        const v4f part = *reinterpret_cast<const v4f*>(&sums[w][h][d]);
        const float g = CODES ? f * (stat[w][2][h] * (1.0f / kPartLift)) : f;
        sum = __builtin_fmaf(stat[w][1][h], f, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(part[e], g, y[e]);
      }
      if (whole) {
        if (d < dim) {
          const float rcp = mx == -INFINITY ? 0.0f : 1.0f / sum;
          *reinterpret_cast<uint2*>(p.out + (int64_t)b * p.o_row + (head0 + h) * p.o_head + 2 * d) =
              make_uint2(pack2<DT>(y[0] * rcp, y[1] * rcp), pack2<DT>(y[2] * rcp, y[3] * rcp));
        }
      } else {
        *reinterpret_cast<v4f*>(p.part + ((int64_t)slot * kHeadTile + h) * DP + d) = y;
        if (d == 0) {
          p.part_ml[(slot * 2) * kHeadTile + h] = mx;
          p.part_ml[(slot * 2 + 1) * kHeadTile + h] = sum;
        }
      }
    }
    if (blk == 0 && take < nblk && threadIdx.x == 0)
      p.shared[blockIdx.x] = make_int4(b, pair, Ranges::of(at + nblk - 1, ranges_per, ranges_extra), 0);
    at += take;
    if (at >= end) return;
    __syncthreads();   // the sums have been read
    blk = 0;
    if (++pair == p.cache.heads * p.tiles) {
      pair = 0;
      nblk = attend_blocks(p, scalar_int(p.lengths, ++b));
    }
  }
}

// The partial sums of a pair that several ranges share: a workgroup for some of its
// heads, of the pair that begins in range blockIdx.x and goes on behind it, or with
// `ranges` given of pair blockIdx.x, whose ranges it finds from the lengths. A wave
// takes 256 / DP heads (four channels a lane), `parts` waves share their ranges,
// eight at a time, and meet in LDS. The order is the ranges', whatever ends when.
constexpr int kJoinWaves = 8, kJoinBatch = 8;
constexpr int join_heads(int dp) { return 256 / dp; }
template <int DT, int DP>
__global__ __launch_bounds__(64 * kJoinWaves) void cache_attend_join_kernel(AttendParams p, int parts, int ranges) {
  constexpr int LANES = DP / 4;
  __shared__ v4f sums[kJoinWaves][64];
  __shared__ float refs[kJoinWaves][64], totals[kJoinWaves][64];
  int b, pair, g0, g1;
  if (ranges > 0) {   // a workgroup for each pair
    const int pairs = p.cache.heads * p.tiles;
    b = blockIdx.x / pairs;
    pair = blockIdx.x - b * pairs;
    int before;
    const Ranges r(attend_total(p, b, before), ranges);
    const int n = attend_blocks(p, scalar_int(p.lengths, b)), at = before + pair * n;
    g0 = Ranges::of(at, r.per, r.extra);
    g1 = Ranges::of(at + n - 1, r.per, r.extra);
    if (g0 == g1) return;
  } else {
    const int4 info = p.shared[blockIdx.x];
    if (info.x < 0) return;
    b = info.x;
    pair = info.y;
    g0 = blockIdx.x;
    g1 = info.z;
  }
  const int kvh = pair / p.tiles, tile = pair - kvh * p.tiles;
  const int heads = min(p.group - kHeadTile * tile, kHeadTile);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, part = wave % parts;
  const int h = (blockIdx.y * kJoinWaves + wave) / parts * join_heads(DP) + lane / LANES, d = 4 * (lane % LANES);
  const bool mine = h < heads;
  auto slot = [&](int g) { return 2 * g + (g == g0); };
  v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
  float sum = 0.0f, ref = -INFINITY;
  if (mine) {
    for (int g = g0 + part; g <= g1; g += kJoinBatch * parts) {
      float m[kJoinBatch], l[kJoinBatch];
      v4f x[kJoinBatch];
#pragma unroll
      for (int i = 0; i < kJoinBatch; ++i) {
        const int at = slot(min(g + i * parts, g1));
        m[i] = p.part_ml[(2 * at) * kHeadTile + h];
        l[i] = p.part_ml[(2 * at + 1) * kHeadTile + h];
        x[i] = *reinterpret_cast<const v4f*>(p.part + ((int64_t)at * kHeadTile + h) * DP + d);
      }
      float to = ref;
#pragma unroll
      for (int i = 0; i < kJoinBatch; ++i) to = fmaxf(to, m[i]);
      const float base = to == -INFINITY ? 0.0f : to, fade = __builtin_amdgcn_exp2f(ref - base);
      ref = to;
      sum = sum * fade;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = y[e] * fade;
#pragma unroll
      for (int i = 0; i < kJoinBatch; ++i) {
        if (g + i * parts > g1) continue;
        const float f = __builtin_amdgcn_exp2f(m[i] - base);
        sum = __builtin_fmaf(l[i], f, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(x[i][e], f, y[e]);
      }
    }
  }
  sums[wave][lane] = y;
  refs[wave][lane] = ref;
  totals[wave][lane] = sum;
  __syncthreads();
  if (part > 0 || !mine || d >= p.cache.dim) return;
  for (int i = 1; i < parts; ++i) ref = fmaxf(ref, refs[wave + i][lane]);
  const float base = ref == -INFINITY ? 0.0f : ref;
  sum = 0.0f;
  y = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (int i = 0; i < parts; ++i) {
    const float f = __builtin_amdgcn_exp2f(refs[wave + i][lane] - base);
    sum = __builtin_fmaf(totals[wave + i][lane], f, sum);
    const v4f x = sums[wave + i][lane];
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(x[e], f, y[e]);
  }
  const float rcp = ref == -INFINITY ? 0.0f : 1.0f / sum;
  *reinterpret_cast<uint2*>(p.out + (int64_t)b * p.o_row + (kvh * p.group + kHeadTile * tile + h) * p.o_head + 2 * d) =
      make_uint2(pack2<DT>(y[0] * rcp, y[1] * rcp), pack2<DT>(y[2] * rcp, y[3] * rcp));
}

// Workgroups of a call: what the GPU holds, each with a range of the blocks of
// all pairs; or one for each pair (then nothing has to be joined), if none can
// have more than four blocks, or eight where the pairs are half as many as the
// CUs: 256 pairs of up to six blocks 17.7 -> 12.9 us, 16 of seven 10.8 -> 13.0.
struct AttendPlan {
  int64_t workgroups;
  bool whole;
};
static AttendPlan attend_plan(int64_t pairs, int64_t max_keys, int dim) {
  const int64_t blocks = std::max<int64_t>((max_keys + kBlockKeys - 1) / kBlockKeys, 1), cus = current_device_cus();
  if (blocks <= 4 || (blocks <= 8 && 2 * pairs >= cus)) return {pairs, true};
  return {std::min<int64_t>(pairs * blocks, attend_per_cu(dim) * cus), false};
}

static int64_t attend_tiles(int64_t heads, int64_t kv_heads) {
  return kv_heads * ((heads / kv_heads + kHeadTile - 1) / kHeadTile);
}

template <int DT, bool CODES, int DP>
static int launch_attend(const AttendParams& p, int64_t workgroups, hipStream_t s) {
  const dim3 g((unsigned)workgroups), t(64 * kAttendWaves);
  if (p.stream) hipLaunchKernelGGL((cache_attend_kernel<DT, CODES, DP, true>), g, t, 0, s, p);
  else hipLaunchKernelGGL((cache_attend_kernel<DT, CODES, DP, false>), g, t, 0, s, p);
  if (!p.whole) {
    // Waves for the ranges of a pair, where it can have many of them, or for its
    // heads (64 pairs of 64 sequences, two or three ranges each: 5.0 us that way,
    // 7.0 this way; one sequence's 8 pairs of 64 ranges 9.8 and 6.8). With many, a
    // workgroup for each pair and not each range: 131072 keys of 8 heads 88.6 -> 86.6
    // us in all, but 196 pairs of two or three ranges 22.6 -> 23.2.
    const int64_t pairs = (int64_t)p.sequences * p.cache.heads * p.tiles, each = workgroups / pairs;
    const int parts = each >= 32 ? 8 : each >= 8 ? 4 : 1, per = kJoinWaves / parts * join_heads(DP);
    hipLaunchKernelGGL((cache_attend_join_kernel<DT, DP>),
                       dim3((unsigned)(each >= 8 ? pairs : workgroups), (std::min(p.group, kHeadTile) + per - 1) / per),
                       dim3(64 * kJoinWaves), 0, s, p, parts, each >= 8 ? (int)workgroups : 0);
  }
  return launch_status("w8a8_cache_attend");
}

template <int DT, bool CODES>
static int launch_attend_dim(const AttendParams& p, int64_t workgroups, hipStream_t s) {
  switch (attend_dp(p.cache.dim)) {
    case 64: return launch_attend<DT, CODES, 64>(p, workgroups, s);
    case 128: return launch_attend<DT, CODES, 128>(p, workgroups, s);
    default: return launch_attend<DT, CODES, 256>(p, workgroups, s);
  }
}

}  // namespace w8a8

extern "C" int64_t w8a8_cache_attend_workspace_size(int64_t sequences, int64_t heads, int64_t kv_heads, int32_t dim,
                                                    int64_t max_keys) {
  using namespace w8a8;
  if (sequences <= 0 || sequences >= (1 << 20) || heads <= 0 || heads > 65536 || kv_heads <= 0 || heads % kv_heads ||
      dim <= 0 || dim > 256 || max_keys < 0 || max_keys >= (1 << 27))
    return 0;
  const AttendPlan plan = attend_plan(sequences * attend_tiles(heads, kv_heads), max_keys, dim);
  return plan.whole ? 0 : plan.workgroups * (2 * kHeadTile * (attend_dp(dim) + 2) * (int64_t)sizeof(float) + (int64_t)sizeof(int4));
}

extern "C" int w8a8_cache_attend(const W8A8CacheAttendArgs* a) {
  using namespace w8a8;
  const char* who = "w8a8_cache_attend";
  W8A8_REQUIRE(a != nullptr, "%s: null args", who);
  W8A8_REQUIRE(a->struct_size == sizeof(W8A8CacheAttendArgs), "%s: struct_size %u != %zu", who, a->struct_size,
               sizeof(W8A8CacheAttendArgs));
  W8A8_REQUIRE(a->dtype == W8A8_F16 || a->dtype == W8A8_BF16, "%s: dtype %d not F16/BF16", who, a->dtype);
  if (a->sequences == 0) return W8A8_OK;
  AttendParams p;
  W8A8_PASS(cache_view(who, a->cache, p.cache));
  W8A8_REQUIRE(a->cache.dtype == W8A8_I8 || a->cache.dtype == a->dtype, "%s: a 16-bit cache takes queries of its own dtype",
               who);
  W8A8_REQUIRE(a->sequences > 0 && a->sequences < (1 << 20) && a->heads > 0 && a->heads <= 65536 &&
                   a->heads % a->cache.heads == 0,
               "%s: sequences or heads out of range, or heads not a multiple of the cache's", who);
  W8A8_PASS(rows_check(who, "q", a->q, a->q_strides));
  W8A8_PASS(rows_check(who, "out", a->out, a->out_strides));
  W8A8_REQUIRE(rows_apart(a->sequences, a->heads, a->cache.dim, a->out_strides), "%s: output rows overlap", who);
  const RowsOf om = rows_memory(a->out, a->sequences, a->heads, a->cache.dim, a->out_strides);
  W8A8_REQUIRE(apart(om, rows_memory(a->q, a->sequences, a->heads, a->cache.dim, a->q_strides)), "%s: out overlaps q", who);
  W8A8_REQUIRE(apart_from_cache(om, a->cache), "%s: out overlaps the cache", who);
  W8A8_REQUIRE(a->table_width >= 0 && a->table_width * a->cache.page_size < (1ll << 27) &&
                   (a->table_width == 0 || a->page_table) && (a->sequences == 1 || a->ld_table >= a->table_width) && a->lengths,
               "%s: page table or lengths null, table rows overlap, or 2^27 keys and more", who);
  W8A8_REQUIRE(a->sm_scale > 0.0f && std::isfinite(a->sm_scale * kLog2eF), "%s: sm_scale must be positive and finite", who);
  const int64_t keys = a->table_width * a->cache.page_size;
  const int64_t need = w8a8_cache_attend_workspace_size(a->sequences, a->heads, a->cache.heads, a->cache.dim, keys);
  W8A8_REQUIRE(need == 0 || (a->workspace && aligned16(a->workspace) && a->workspace_bytes >= need),
               "%s: workspace of %lld bytes needed", who, (long long)need);
  W8A8_REQUIRE(apart_from(om, a->page_table, table_bytes(a->sequences, a->ld_table, a->table_width)) &&
                   apart_from(om, a->lengths, 4 * a->sequences) && apart_from(om, a->workspace, need),
               "%s: page table, lengths or workspace lie in the output", who);
  p.q = reinterpret_cast<const char*>(a->q);
  p.out = reinterpret_cast<char*>(a->out);
  p.q_row = 2 * a->q_strides[0]; p.q_head = 2 * a->q_strides[1];
  p.o_row = 2 * a->out_strides[0]; p.o_head = 2 * a->out_strides[1];
  p.sequences = (int)a->sequences;
  p.heads = (int)a->heads;
  p.group = p.heads / p.cache.heads;
  p.tiles = (p.group + kHeadTile - 1) / kHeadTile;
  p.width = (int)a->table_width;
  p.table = a->page_table;
  p.ld_table = a->ld_table;
  p.lengths = a->lengths;
  p.c = a->sm_scale * kLog2eF;
  const int64_t pairs = a->sequences * p.cache.heads * p.tiles;
  const bool codes = a->cache.dtype == W8A8_I8;
  const AttendPlan plan = attend_plan(pairs, keys, p.cache.dim);
  W8A8_REQUIRE(pairs * (keys / kBlockKeys + 1) < (1ll << 31) && plan.workgroups < (1 << 23),
               "%s: too many sequences, heads and keys for one launch", who);   // (2^32 work-items)
  p.whole = plan.whole;
  // What the table can name, against the last cache's 256 MB: read once and never
  // again, so let it pass (512 MB: 102 -> 89 us; 94 MB that the last call left
  // there: 23.3 -> 26.2 that way).
  const int64_t row = codes ? a->cache.dim + 4 : 2 * a->cache.dim;
  p.stream = 2 * row * a->cache.heads * keys * a->sequences > (256ll << 20);
  p.part = reinterpret_cast<float*>(a->workspace);
  p.part_ml = p.part + plan.workgroups * 2 * kHeadTile * attend_dp(p.cache.dim);
  p.shared = reinterpret_cast<int4*>(p.part_ml + plan.workgroups * 4 * kHeadTile);
  hipStream_t s = reinterpret_cast<hipStream_t>(a->stream);
  if (a->dtype == W8A8_F16) return codes ? launch_attend_dim<kF16, true>(p, plan.workgroups, s) : launch_attend_dim<kF16, false>(p, plan.workgroups, s);
  return codes ? launch_attend_dim<kBF16, true>(p, plan.workgroups, s) : launch_attend_dim<kBF16, false>(p, plan.workgroups, s);
}
