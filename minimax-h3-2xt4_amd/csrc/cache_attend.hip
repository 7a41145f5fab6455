// Attention of one new token of every sequence over a paged cache.
//
//   o = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m),  t_j = log2(e) scale q . k_j
//
// in one pass with the running maximum m, every key read once. A query head
// does 4 flops per element read, so even sixteen heads on one kv head are far
// from the MFMA's rate: HBM bounds this, and the work is cut by keys. All keys of
// all (sequence, kv head) pairs, in blocks of 128, are one line that is cut
// into equal ranges, one for each workgroup, whatever the sequences' lengths; a
// pair inside one range is finished there, one that several ranges share
// leaves partial sums, which a second kernel joins in order.
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

namespace w8a8 {

constexpr int kAttendWaves = 4;
constexpr int kWaveKeys = 32;
constexpr int kBlockKeys = kAttendWaves * kWaveKeys;
constexpr int kHeadTile = 16;

struct AttendParams {
  CacheView cache;
  const char* q;
  char* out;
  int64_t q_row, q_head, o_row, o_head;   // bytes
  int sequences, heads, group, tiles;     // tiles: of 16 query heads of a kv head
  int width;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  float c;   // log2(e) * scale
  float* part;       // [workgroups][2][kHeadTile][dim padded]
  float* part_ml;    // [workgroups][2][2][kHeadTile]: maximum, sum
};

__device__ __forceinline__ int attend_length(const AttendParams& p, int len) {
  return min(max(len, 0), p.width * p.cache.page_size);
}
__device__ __forceinline__ int attend_blocks(const AttendParams& p, int len) {
  return max((attend_length(p, len) + kBlockKeys - 1) / kBlockKeys, 1);   // (an empty sequence has a block of no keys)
}

// Blocks of all pairs.
__device__ __forceinline__ int64_t attend_total(const AttendParams& p) {
  int64_t n = 0;
  for (int b = threadIdx.x & 63; b < p.sequences; b += 64) n += attend_blocks(p, p.lengths[b]);
  return wave_sum64(n) * (p.cache.heads * p.tiles);
}

// The sequence that block n of the line belongs to, and the blocks before it.
__device__ __forceinline__ int attend_find(const AttendParams& p, int64_t n, int64_t& before) {
  const int lane = threadIdx.x & 63;
  const int64_t pairs = p.cache.heads * p.tiles;
  int64_t sum = 0;
  for (int b0 = 0; b0 < p.sequences; b0 += 64) {
    const int64_t mine = b0 + lane < p.sequences ? attend_blocks(p, p.lengths[b0 + lane]) * pairs : 0;
    const int64_t upto = sum + wave_prefix64(mine);
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > n);
    if (past) {
      const int at = __builtin_ctzll(past);
      before = __shfl(upto - mine, at, 64);
      return __builtin_amdgcn_readfirstlane(b0 + at);
    }
    sum = __shfl(upto, 63, 64);
  }
  before = sum;
  return p.sequences;
}

__device__ __forceinline__ int64_t uniform64(int64_t v) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = __builtin_amdgcn_readfirstlane((int)(v >> 32));
  return (int64_t)(((uint64_t)hi << 32) | lo);
}

// Ranges that hold a block, of so many workgroups: none in between is empty.
__device__ __forceinline__ int attend_used(int64_t total, int ranges) { return (int)min(total, (int64_t)ranges); }

// Where range g of n blocks begins.
__device__ __forceinline__ int64_t range_at(int64_t n, int g, int ranges) { return n / ranges * g + n % ranges * g / ranges; }

template <int DT>
__device__ __forceinline__ v4f mfma16(v4u a, v4u b, v4f c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// Four codes of a word as two words of DT values (exact in both types).
template <int DT>
__device__ __forceinline__ v2u codes4(uint32_t w) {
  if constexpr (DT == kF16) {
    // 0x6400 | (code + 128) is the fp16 value 1152 + code.
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t lo = __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u), hi = __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u);
    const v2h off = {(_Float16)1152.0f, (_Float16)1152.0f};
    return v2u{__builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, lo) - off),
               __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, hi) - off)};
  } else {
    uint32_t f[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __float_as_uint((float)(int8_t)(w >> (8 * i)));
    return v2u{__builtin_amdgcn_perm(f[1], f[0], 0x07060302u), __builtin_amdgcn_perm(f[3], f[2], 0x07060302u)};
  }
}

// A lane's loads of a group of 16 tokens: W words from byte offset off of its descriptor.
template <int W>
__device__ __forceinline__ void group_load(__amdgpu_buffer_rsrc_t r, uint32_t off, uint32_t (&w)[W]) {
  if constexpr (W == 1) {
    w[0] = __builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0);
  } else if constexpr (W == 2) {
    const v2u t = __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0);
    w[0] = t.x; w[1] = t.y;
  } else {
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
      const v4u t = __builtin_amdgcn_raw_buffer_load_b128(r, (int)off + 16 * i, 0, 0);
      w[4 * i] = t.x; w[4 * i + 1] = t.y; w[4 * i + 2] = t.z; w[4 * i + 3] = t.w;
    }
  }
}

constexpr uint32_t kNowhere = 0x7fffff00u;   // an offset behind every descriptor's end

// DT: type of q and out; CODES: the cache holds I8; DP: dim rounded up to 64, 128 or 256.
template <int DT, bool CODES, int DP>
__global__ __launch_bounds__(64 * kAttendWaves, 2) void cache_attend_kernel(AttendParams p) {
  constexpr int ES = CODES ? 1 : 2;
  constexpr int NS = DP / 32;          // products of a key tile
  constexpr int VL = DP / 16;          // channels a lane reads of a value row
  constexpr int KW = CODES ? 2 : 4;    // words of eight channels
  constexpr int VW = VL * ES / 4;      // words of VL channels
  constexpr int kRow = DP + 4;         // a head's sums in LDS, padded
  __shared__ __attribute__((aligned(16))) float sums[kAttendWaves][kHeadTile][kRow];
  __shared__ float stat[kAttendWaves][3][kHeadTile];
  const int lane = threadIdx.x & 63, col = lane & 15, quad = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int dim = p.cache.dim;

  const int64_t total = uniform64(attend_total(p));
  const int ranges = attend_used(total, gridDim.x);
  if ((int)blockIdx.x >= ranges) return;
  int64_t at = uniform64(range_at(total, blockIdx.x, ranges));
  const int64_t end = uniform64(range_at(total, blockIdx.x + 1, ranges));
  int64_t before;
  int b = attend_find(p, at, before);
  before = uniform64(before);
  int nblk = attend_blocks(p, scalar_int(p.lengths, b));
  int64_t rest = at - before;
  int pair = (int)(rest / nblk), blk = (int)(rest - (int64_t)pair * nblk);

  // Byte offsets within a group of 16 tokens.
  uint32_t koff[NS], voff[4];
#pragma unroll
  for (int s = 0; s < NS; ++s) {
    const int d = 8 * quad + 32 * s;
    koff[s] = d < dim ? col * p.cache.token_b + d * ES : kNowhere;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    voff[i] = VL * col < dim ? (4 * quad + i) * p.cache.token_b + VL * col * ES : kNowhere;

  while (true) {
    const int len = attend_length(p, scalar_int(p.lengths, b));
    const int kvh = pair / p.tiles, tile = pair - kvh * p.tiles;
    const int take = (int)min((int64_t)(nblk - blk), end - at);
    const int nh = min(p.group - kHeadTile * tile, kHeadTile);
    const int head0 = kvh * p.group + kHeadTile * tile;
    const char* kb = p.cache.k + kvh * p.cache.head_b;
    const char* vb = p.cache.v + kvh * p.cache.head_b;
    v4u qf[NS];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int d = 8 * quad + 32 * s;
      qf[s] = v4u{0, 0, 0, 0};
      if (col < nh && d < dim)
        qf[s] = *reinterpret_cast<const v4u*>(p.q + (int64_t)b * p.q_row + (head0 + col) * p.q_head + 2 * d);
    }
    v4f o[VL];
#pragma unroll
    for (int j = 0; j < VL; ++j) o[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    float m = -INFINITY, l = 0.0f, top = 0.0f;   // top: the largest value scale so far (codes)

    // Two groups of 16 keys, their places and how many keys of each count.
    struct Keys {
      int page[2], token[2], n[2];
    };
    auto place = [&](int block) {
      Keys k;
      const int k0 = (block * kAttendWaves + wave) * kWaveKeys;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int first = k0 + i * kGroupTokens;
        int n = min(max(len - first, 0), kGroupTokens), entry, page = 0;
        group_place(p.cache, (uint32_t)first / kGroupTokens, entry, k.token[i]);
        if (n > 0) page = scalar_int(p.table, (int64_t)b * p.ld_table + entry);
        if (page < 0 || page >= p.cache.pages) page = n = 0;
        k.page[i] = page;
        k.n[i] = n;
      }
      return k;
    };
    auto group_rsrc = [&](const char* base, const Keys& k, int i) {
      const char* t = base + (int64_t)k.page[i] * p.cache.page_b + (int64_t)k.token[i] * p.cache.token_b;
      return __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(t), 0, 
                                               k.n[i] ? (int)((k.n[i] - 1) * p.cache.token_b) + dim * ES : 0, 0x00027000);
    };
    uint32_t kr[2][NS][KW], vr[8][VW];
    auto load_k = [&](const Keys& k) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const auto r = group_rsrc(kb, k, i);
#pragma unroll
        for (int s = 0; s < NS; ++s) group_load<KW>(r, koff[s], kr[i][s]);
      }
    };
    auto load_v = [&](const Keys& k) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const auto r = group_rsrc(vb, k, i);
#pragma unroll
        for (int t = 0; t < 4; ++t) group_load<VW>(r, voff[t], vr[4 * i + t]);
      }
    };
    struct Scales {
      v4f k[2], v[2];
    };
    auto load_scales = [&](const Keys& k) {
      Scales sc{};
      if constexpr (!CODES) return sc;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int64_t s = (int64_t)k.page[i] * p.cache.s_page + kvh * p.cache.s_head + k.token[i] + 4 * quad;
        sc.k[i] = *reinterpret_cast<const v4f*>(p.cache.ks + s);
        sc.v[i] = *reinterpret_cast<const v4f*>(p.cache.vs + s);
      }
      return sc;
    };

    auto spread_max = [&](float x) {   // over the four quads: the keys of a column
      x = fmaxf(x, __shfl_xor(x, 16, 64));
      return fmaxf(x, __shfl_xor(x, 32, 64));
    };
    const int last = blk + take;
    Keys now = place(blk);
    load_k(now);
    load_v(now);
    Scales sc = load_scales(now);
    for (int block = blk; block < last; ++block) {
      v4f s[2] = {v4f{0.0f, 0.0f, 0.0f, 0.0f}, v4f{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int t = 0; t < NS; ++t) {
          v4u a;
          if constexpr (CODES) {
            const v2u lo = codes4<DT>(kr[i][t][0]), hi = codes4<DT>(kr[i][t][1]);
            a = v4u{lo.x, lo.y, hi.x, hi.y};
          } else {
            a = v4u{kr[i][t][0], kr[i][t][1], kr[i][t][2], kr[i][t][3]};
          }
          s[i] = mfma16<DT>(a, qf[t], s[i]);
        }
      float t[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        t[i] = s[i / 4][i % 4] * p.c;
        if constexpr (CODES) t[i] = t[i] * sc.k[i / 4][i % 4];
      }
      const Keys next = block + 1 < last ? place(block + 1) : Keys{{0, 0}, {0, 0}, {0, 0}};
      load_k(next);
      const Scales sn = load_scales(next);
      if (now.n[0] < kGroupTokens || now.n[1] < kGroupTokens) {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (4 * quad + i % 4 >= now.n[i / 4]) t[i] = -INFINITY;
      }
      float mx = t[0];
#pragma unroll
      for (int i = 1; i < 8; ++i) mx = fmaxf(mx, t[i]);
      mx = fmaxf(m, spread_max(mx));
      const float ref = mx == -INFINITY ? 0.0f : mx;
      float w[8], fade = __builtin_amdgcn_exp2f(m - ref);
      m = mx;
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = __builtin_amdgcn_exp2f(t[i] - ref);
        sum += w[i];
      }
      l = __builtin_fmaf(l, fade, sum);
      if constexpr (CODES) {
        // P carries the values' scales, relative to the largest so far, so
        // that it keeps the type's precision whatever their size.
        float u = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (4 * quad + i % 4 < now.n[i / 4]) u = fmaxf(u, sc.v[i / 4][i % 4]);
        u = fmaxf(fmaxf(top, spread_max(u)), 0x1p-126f);
        const float inv = 1.0f / u;
        fade = fade * (top * inv);
        top = u;
#pragma unroll
        for (int i = 0; i < 8; ++i)
          w[i] = 4 * quad + i % 4 < now.n[i / 4] ? w[i] * (sc.v[i / 4][i % 4] * inv) : 0.0f;
      }
      if (__builtin_amdgcn_ballot_w64(fade != 1.0f)) {
#pragma unroll
        for (int j = 0; j < VL; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i) o[j][i] = o[j][i] * fade;
      }
      const v4u pf = {pack2<DT>(w[0], w[1]), pack2<DT>(w[2], w[3]), pack2<DT>(w[4], w[5]), pack2<DT>(w[6], w[7])};
      uint32_t x[8][VL / 2];
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < VL / 2; j += 2) {
          if constexpr (CODES) {
            const v2u c = codes4<DT>(vr[i][j / 2]);
            x[i][j] = c.x;
            x[i][j + 1] = c.y;
          } else {
            x[i][j] = vr[i][j];
            x[i][j + 1] = vr[i][j + 1];
          }
        }
#pragma unroll
      for (int j = 0; j < VL; ++j) {
        const uint32_t pick = j % 2 ? 0x07060302u : 0x05040100u;
        v4u a;
#pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = __builtin_amdgcn_perm(x[2 * i + 1][j / 2], x[2 * i][j / 2], pick);
        o[j] = mfma16<DT>(a, pf, o[j]);
      }
      load_v(next);
      now = next;
      sc = sn;
    }

    // The waves' sums meet: O's lane (col, quad) holds head col, channels
    // VL (4 quad + r) + j.
    l = l + __shfl_xor(l, 16, 64);
    l = l + __shfl_xor(l, 32, 64);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int j = 0; j < VL; j += 4)
        *reinterpret_cast<v4f*>(&sums[wave][col][VL * (4 * quad + r) + j]) = v4f{o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]};
    if (quad == 0) {
      stat[wave][0][col] = m;
      stat[wave][1][col] = l;
      stat[wave][2][col] = top;
    }
    __syncthreads();
    const bool whole = blk == 0 && take == nblk;
    const int64_t slot = (int64_t)blockIdx.x * 2 + (blk == 0 ? 1 : 0);   // the pair begins in this range, or before it
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
        const float g = CODES ? f * stat[w][2][h] : f;
        sum = __builtin_fmaf(stat[w][1][h], f, sum);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(part[e], g, y[e]);
      }
      if (whole) {
        if (d < dim) {
          const float rcp = mx == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
          *reinterpret_cast<uint2*>(p.out + (int64_t)b * p.o_row + (head0 + h) * p.o_head + 2 * d) =
              make_uint2(pack2<DT>(y[0] * rcp, y[1] * rcp), pack2<DT>(y[2] * rcp, y[3] * rcp));
        }
      } else {
        *reinterpret_cast<v4f*>(p.part + (slot * kHeadTile + h) * DP + d) = y;
        if (d == 0) {
          p.part_ml[(slot * 2) * kHeadTile + h] = mx;
          p.part_ml[(slot * 2 + 1) * kHeadTile + h] = sum;
        }
      }
    }
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

// The partial sums of a pair that several ranges share, in order: a workgroup
// of one wave takes a query head, four channels a lane (DP 64: 16 lanes work).
template <int DT, int DP>
__global__ __launch_bounds__(64) void cache_attend_join_kernel(AttendParams p, int workgroups) {
  const int head = blockIdx.x, b = blockIdx.y + gridDim.y * blockIdx.z;
  if (b >= p.sequences) return;
  const int kvh = head / p.group, in = head - kvh * p.group, tile = in / kHeadTile, h = in - tile * kHeadTile;
  const int64_t pairs = p.cache.heads * p.tiles;
  int64_t before = 0, total = 0;
  for (int i = threadIdx.x; i < p.sequences; i += 64) {
    const int64_t n = attend_blocks(p, p.lengths[i]);
    total += n;
    if (i < b) before += n;
  }
  total = uniform64(wave_sum64(total) * pairs);
  const int ranges = attend_used(total, workgroups);
  const int nblk = attend_blocks(p, scalar_int(p.lengths, b));
  const int64_t first = uniform64(wave_sum64(before)) * pairs + (int64_t)(kvh * p.tiles + tile) * nblk;
  // The ranges that hold its first and its last block.
  auto range_of = [&](int64_t n) {
    int g = (int)(n * ranges / total);
    while (g > 0 && range_at(total, g, ranges) > n) --g;
    while (range_at(total, g + 1, ranges) <= n) ++g;
    return g;
  };
  const int g0 = range_of(first), g1 = range_of(first + nblk - 1);
  if (g0 == g1) return;
  const int d = 4 * threadIdx.x;
  float mx = -INFINITY;
  for (int g = g0 + (int)threadIdx.x; g <= g1; g += 64)
    mx = fmaxf(mx, p.part_ml[((int64_t)(2 * g + (g == g0)) * 2) * kHeadTile + h]);
  mx = wave_max(mx);
  const float ref = mx == -INFINITY ? 0.0f : mx;
  v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
  float sum = 0.0f;
#pragma unroll 8
  for (int g = g0; g <= g1; ++g) {
    const int64_t slot = 2 * (int64_t)g + (g == g0);
    const float f = __builtin_amdgcn_exp2f(p.part_ml[(slot * 2) * kHeadTile + h] - ref);
    sum = __builtin_fmaf(p.part_ml[(slot * 2 + 1) * kHeadTile + h], f, sum);
    const v4f part = *reinterpret_cast<const v4f*>(p.part + (slot * kHeadTile + h) * DP + (d < DP ? d : 0));
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(part[e], f, y[e]);
  }
  if (d >= p.cache.dim) return;
  const float rcp = mx == -INFINITY && sum == 0.0f ? 0.0f : 1.0f / sum;
  *reinterpret_cast<uint2*>(p.out + (int64_t)b * p.o_row + head * p.o_head + 2 * d) =
      make_uint2(pack2<DT>(y[0] * rcp, y[1] * rcp), pack2<DT>(y[2] * rcp, y[3] * rcp));
}

static int attend_dp(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Ranges of a call: two workgroups a CU, unless all keys that the table can
// hold are fewer blocks.
static int64_t attend_ranges(int64_t pairs, int64_t max_keys) {
  const int64_t most = pairs * std::max<int64_t>((max_keys + kBlockKeys - 1) / kBlockKeys, 1);
  return std::min<int64_t>(most, 2 * current_device_cus());
}

static int64_t attend_tiles(int64_t heads, int64_t kv_heads) {
  return kv_heads * ((heads / kv_heads + kHeadTile - 1) / kHeadTile);
}

template <int DT, bool CODES, int DP>
static int launch_attend(const AttendParams& p, int64_t ranges, hipStream_t s) {
  hipLaunchKernelGGL((cache_attend_kernel<DT, CODES, DP>), dim3((unsigned)ranges), dim3(64 * kAttendWaves), 0, s, p);
  const unsigned y = (unsigned)std::min(p.sequences, 32768);
  hipLaunchKernelGGL((cache_attend_join_kernel<DT, DP>), dim3((unsigned)p.heads, y, (unsigned)((p.sequences + y - 1) / y)),
                     dim3(64), 0, s, p, (int)ranges);
  return launch_status("w8a8_cache_attend");
}

template <int DT, bool CODES>
static int launch_attend_dim(const AttendParams& p, int64_t ranges, hipStream_t s) {
  switch (attend_dp(p.cache.dim)) {
    case 64: return launch_attend<DT, CODES, 64>(p, ranges, s);
    case 128: return launch_attend<DT, CODES, 128>(p, ranges, s);
    default: return launch_attend<DT, CODES, 256>(p, ranges, s);
  }
}

}  // namespace w8a8

extern "C" int64_t w8a8_cache_attend_workspace_size(int64_t sequences, int64_t heads, int64_t kv_heads, int32_t dim,
                                                    int64_t max_keys) {
  using namespace w8a8;
  if (sequences <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads || dim <= 0 || dim > 256) return 0;
  const int64_t ranges = attend_ranges(sequences * attend_tiles(heads, kv_heads), max_keys);
  return ranges * 2 * kHeadTile * (attend_dp(dim) + 2) * (int64_t)sizeof(float);
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
  W8A8_REQUIRE(!spans_overlap(a->q, rows_span(a->sequences, a->heads, a->cache.dim, a->q_strides), a->out,
                              rows_span(a->sequences, a->heads, a->cache.dim, a->out_strides)),
               "%s: out overlaps q", who);
  W8A8_REQUIRE(a->table_width >= 0 && a->table_width * a->cache.page_size < (1ll << 27) &&
                   (a->table_width == 0 || a->page_table) && (a->sequences == 1 || a->ld_table >= a->table_width) && a->lengths,
               "%s: page table or lengths null, table rows overlap, or 2^27 keys and more", who);
  W8A8_REQUIRE(a->sm_scale > 0.0f && std::isfinite(a->sm_scale), "%s: sm_scale must be positive and finite", who);
  const int64_t keys = a->table_width * a->cache.page_size;
  const int64_t need = w8a8_cache_attend_workspace_size(a->sequences, a->heads, a->cache.heads, a->cache.dim, keys);
  W8A8_REQUIRE(need == 0 || (a->workspace && aligned16(a->workspace) && a->workspace_bytes >= need),
               "%s: workspace of %lld bytes needed", who, (long long)need);
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
  W8A8_REQUIRE(pairs * ((keys + kBlockKeys - 1) / kBlockKeys + 1) < (1ll << 48), "%s: too many keys in all", who);
  const int64_t ranges = attend_ranges(pairs, keys);
  p.part = reinterpret_cast<float*>(a->workspace);
  p.part_ml = p.part + ranges * 2 * kHeadTile * attend_dp(p.cache.dim);
  hipStream_t s = reinterpret_cast<hipStream_t>(a->stream);
  const bool codes = a->cache.dtype == W8A8_I8;
  if (a->dtype == W8A8_F16) return codes ? launch_attend_dim<kF16, true>(p, ranges, s) : launch_attend_dim<kF16, false>(p, ranges, s);
  return codes ? launch_attend_dim<kBF16, true>(p, ranges, s) : launch_attend_dim<kBF16, false>(p, ranges, s);
}
