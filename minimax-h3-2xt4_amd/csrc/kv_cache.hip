// Keys and values into a paged cache and back out.
//
// A wave takes one row of the packed keys and values and a run of its heads,
// LPH lanes to a head, eight channels a lane (16 bytes of 16-bit values, 8 of
// codes). It finds the row's sequence by comparing the starts of 64 sequences
// at once, and the page is then one scalar load. With codes the row's largest
// magnitude is a reduction over a head's lanes; scale and codes are those of
// the activation quantizer (quant1). Bound by HBM: 11690 rows of 28 heads of 128
// written in 60 us (5.6 TB/s), 69277 rows of 8 heads of codes read in 68 (6.2).
#include "paged.h"

namespace w8a8 {

struct CacheMoveParams {
  CacheView cache;
  char* k;
  char* v;
  int64_t k_row, k_head, v_row, v_head;   // bytes
  int64_t rows;
  int sequences, width;
  const int32_t* table;
  int64_t ld_table;
  const int32_t* lengths;
  const int32_t* starts;
  int runs;   // runs of heads of a row,
  int pack;   // or rows of a wave, of fewer heads than it takes
  int fill;
  int stream;
};

constexpr int kMoveHeads = 2;   // heads of a lane

// The largest of a head's lanes. Magnitudes are compared as the integers of
// their bits, among which infinities and then NaNs are the largest.
template <int LPH>
__device__ __forceinline__ uint32_t head_max(uint32_t v) {
#pragma unroll
  for (int off = LPH / 2; off >= 1; off >>= 1) v = max(v, (uint32_t)__shfl_xor((int)v, off, 64));
  return v;
}

// 16 bytes in or out: in they are read once; out they are to stay in the caches,
// unless the whole is more than those hold (stream).
__device__ __forceinline__ uint4 take16(const void* p) {
  const v4u v = __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p));
  return make_uint4(v.x, v.y, v.z, v.w);
}
__device__ __forceinline__ void put16(void* p, uint4 x, int stream) {
  if (stream) __builtin_nontemporal_store(v4u{x.x, x.y, x.z, x.w}, reinterpret_cast<v4u*>(p));
  else *reinterpret_cast<uint4*>(p) = x;
}

template <int DT>
__device__ __forceinline__ void widen8(uint4 u, float (&f)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint16_t lo = (uint16_t)(w[i] & 0xffffu), hi = (uint16_t)(w[i] >> 16);
    f[2 * i] = DT == kF16 ? h2f(lo) : bf2f(lo);
    f[2 * i + 1] = DT == kF16 ? h2f(hi) : bf2f(hi);
  }
}

// Eight codes of values f with scale s: rne(x / s), whose quotient is q = x * rcp
// with one correction, q + (x - q s) rcp. rcp is 1 / s correctly rounded and the
// remainder exact, so that is the correctly rounded quotient (Markstein), without
// a branch for ties, which values of 16 bits often are (353 rows of 8 heads 5.9 ->
// 3.9 us). Tiny rows, whose remainder could lose bits below 2^-149, divide.
__device__ __forceinline__ uint2 codes8(const float (&f)[8], float s, bool tiny) {
  const float rcp = 1.0f / s;
  uint32_t w[2] = {0, 0};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    float q = f[j] * rcp;
    q = __builtin_fmaf(__builtin_fmaf(-q, s, f[j]), rcp, q);
    if (tiny) q = f[j] / s;
    w[j / 4] = __builtin_amdgcn_cvt_pk_u8_f32(rintf(q) + 128.0f, j % 4, w[j / 4]);
  }
  return make_uint2(w[0] ^ 0x80808080u, w[1] ^ 0x80808080u);
}

// The page and token of key pos of sequence b; -1 where it is not there.
template <bool SCALAR>
__device__ __forceinline__ int key_place(const CacheMoveParams& p, int b, int pos, int& token) {
  if (pos < 0) return -1;
  int entry, first;
  group_place(p.cache, (uint32_t)pos / kGroupTokens, entry, first);
  if (entry >= p.width) return -1;
  token = first + pos % kGroupTokens;
  const int64_t i = (int64_t)b * p.ld_table + entry;
  const int page = SCALAR ? scalar_int(p.table, i) : p.table[i];
  return page < p.cache.pages ? page : -1;
}

// What a lane moves: eight channels of kMoveHeads heads, each of a row. A row has
// heads for a wave, or runs of them for several. Where a wave takes three times
// the heads and more, and rows are more than the GPU holds waves for at once,
// it takes p.pack rows (PACK): 50000 rows of one head of 128 written as codes 26.1 -> 12.4
// us and read 17.6 -> 9.7; but 353 rows of two heads 3.9 -> 4.8, and 40000 of four,
// two to a wave, 28.8 -> 30.5.
template <int LPH, bool PACK>
struct Move {
  int chunk;
  int64_t row[kMoveHeads];
  int head[kMoveHeads];   // p.cache.heads where there is nothing to move
  int64_t first;          // the wave's first row
  int off[kMoveHeads];    // rows behind it
  __device__ __forceinline__ explicit Move(const CacheMoveParams& p) {
    const int lane = threadIdx.x & 63;
    const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    chunk = lane % LPH;
    first = PACK ? item * p.pack : item / p.runs;
#pragma unroll
    for (int i = 0; i < kMoveHeads; ++i) {
      const int slot = i * (64 / LPH) + lane / LPH;
      off[i] = PACK ? slot / p.cache.heads : 0;
      row[i] = first + off[i];
      head[i] = PACK ? slot - off[i] * p.cache.heads : (int)(item - first * p.runs) * (kMoveHeads * 64 / LPH) + slot;
      if (PACK && (row[i] >= p.rows || off[i] >= p.pack)) head[i] = p.cache.heads;
    }
  }
};

// The sequences of the rows (p.sequences: none), with starts and, if given, lengths.
template <int LPH, bool PACK>
__device__ __forceinline__ void sequences_of(const CacheMoveParams& p, const Move<LPH, PACK>& m, const int32_t* lengths,
                                             SequenceRow (&s)[kMoveHeads]) {
  if constexpr (!PACK) {
    s[0] = sequence_of(p.starts, p.sequences, m.first, lengths);
#pragma unroll
    for (int i = 1; i < kMoveHeads; ++i) s[i] = s[0];
  } else {
    const int lane = threadIdx.x & 63, rows = (int)min((int64_t)p.pack, p.rows - m.first);
    int b0 = sequence_window(p.starts, p.sequences, m.first);
    int found = 0;
#pragma unroll
    for (int i = 0; i < kMoveHeads; ++i) s[i] = {p.sequences, 0, 0, 0};
    for (; b0 < p.sequences && found < rows; b0 += 64) {
      const int at = min(b0 + lane, p.sequences - 1);
      const int first = p.starts[at], last = p.starts[at + 1], length = lengths ? lengths[at] : 0;
      int mine[kMoveHeads];
#pragma unroll
      for (int i = 0; i < kMoveHeads; ++i) mine[i] = -1;
      for (int r = 0; r < rows; ++r) {
        const int64_t row = m.first + r;
        const uint64_t in = __builtin_amdgcn_ballot_w64(b0 + lane < p.sequences && first <= row && row < last);
        if (in == 0) continue;
        ++found;
#pragma unroll
        for (int i = 0; i < kMoveHeads; ++i) mine[i] = r == m.off[i] ? __builtin_ctzll(in) : mine[i];
      }
#pragma unroll
      for (int i = 0; i < kMoveHeads; ++i) {
        const int from = max(mine[i], 0);
        const SequenceRow t{b0 + from, __shfl(first, from, 64), __shfl(last, from, 64), __shfl(length, from, 64)};
        if (mine[i] >= 0 && s[i].b == p.sequences) s[i] = t;
      }
      if (__builtin_amdgcn_readlane(last, 63) > m.first + rows - 1) break;   // ascending: the rest lies behind the rows
    }
  }
}

// codes: the cache holds I8; DT is the rows' type.
template <int DT, bool CODES, int LPH, bool PACK>
__global__ __launch_bounds__(256) void cache_write_kernel(CacheMoveParams p) {
  const Move<LPH, PACK> m(p);
  if (m.first >= p.rows) return;
  const bool mine = 8 * m.chunk < p.cache.dim;   // (lanes beyond the channels stay for the maximum)
  uint4 x[2][kMoveHeads];
#pragma unroll
  for (int i = 0; i < kMoveHeads; ++i) {
    x[0][i] = x[1][i] = make_uint4(0, 0, 0, 0);
    if (m.head[i] < p.cache.heads && mine) {
      x[0][i] = take16(p.k + m.row[i] * p.k_row + m.head[i] * p.k_head + 16 * m.chunk);
      x[1][i] = take16(p.v + m.row[i] * p.v_row + m.head[i] * p.v_head + 16 * m.chunk);
    }
  }
  SequenceRow s[kMoveHeads];
  if (p.starts) {
    sequences_of(p, m, p.lengths, s);
  } else {
#pragma unroll
    for (int i = 0; i < kMoveHeads; ++i) {
      const int b = (int)min(m.row[i], p.rows - 1);
      s[i] = {b, b, b + 1, PACK ? p.lengths[b] : scalar_int(p.lengths, b)};
    }
  }
  int one_token = 0, one = -1;   // the place of the wave's only row
  if constexpr (!PACK) {
    if (s[0].b < p.sequences) one = key_place<true>(p, s[0].b, s[0].length - (s[0].last - (int)m.first), one_token);
    if (one < 0) return;
  }
#pragma unroll
  for (int i = 0; i < kMoveHeads; ++i) {
    const int h = m.head[i];
    int token = one_token, page = one;
    if (h >= p.cache.heads) continue;   // (a head's lanes together)
    if constexpr (PACK) {
      if (s[i].b < p.sequences) page = key_place<false>(p, s[i].b, s[i].length - (s[i].last - (int)m.row[i]), token);
      if (page < 0) continue;
    }
    const int64_t at = (int64_t)page * p.cache.page_b + (int64_t)token * p.cache.token_b;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      char* to = (t ? p.cache.v : p.cache.k) + at + h * p.cache.head_b;
      if constexpr (!CODES) {
        if (mine) put16(to + 16 * m.chunk, x[t][i], p.stream);
      } else {
        float f[8];
        uint32_t top = 0;
        widen8<DT>(x[t][i], f);
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(f[j]) & 0x7fffffffu);
        top = head_max<LPH>(top);
        // A row that holds an infinity or a NaN has the scale NaN.
        const float scale = top < 0x7f800000u ? row_scale_of(__uint_as_float(top)) : __uint_as_float(0x7fc00000u);
        if (!mine) continue;
        const bool tiny = __builtin_amdgcn_ballot_w64(scale < 0x1p-60f) != 0;
        *reinterpret_cast<uint2*>(to + 8 * m.chunk) = tiny ? codes8(f, scale, true) : codes8(f, scale, false);
        if (m.chunk == 0)
          (t ? p.cache.vs : p.cache.ks)[(int64_t)page * p.cache.s_page + h * p.cache.s_head + token] = scale;
      }
    }
  }
}

template <int DT, bool CODES, int LPH, bool PACK>
__global__ __launch_bounds__(256) void cache_read_kernel(CacheMoveParams p) {
  const Move<LPH, PACK> m(p);
  if (m.first >= p.rows) return;
  SequenceRow s0[kMoveHeads];
  sequences_of(p, m, nullptr, s0);
  int one_token = 0, one = -1;   // the place of the wave's only row
  if (!PACK && s0[0].b < p.sequences) one = key_place<true>(p, s0[0].b, (int)m.first - s0[0].first, one_token);
  if (8 * m.chunk >= p.cache.dim) return;
  uint4 x[2][kMoveHeads];
  uint2 c[2][kMoveHeads];
  float s[2][kMoveHeads];
#pragma unroll
  for (int i = 0; i < kMoveHeads; ++i) {
    const int h = m.head[i];
    int token = one_token, page = one;
    if (PACK && h < p.cache.heads && s0[i].b < p.sequences)
      page = key_place<false>(p, s0[i].b, (int)m.row[i] - s0[i].first, token);
    const int64_t at = (int64_t)page * p.cache.page_b + (int64_t)token * p.cache.token_b;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      x[t][i] = make_uint4(0, 0, 0, 0);
      c[t][i] = make_uint2(0, 0);
      s[t][i] = 0.0f;
      if (h >= p.cache.heads || page < 0) continue;
      const char* from = (t ? p.cache.v : p.cache.k) + at + h * p.cache.head_b;
      if constexpr (!CODES) {
        x[t][i] = take16(from + 16 * m.chunk);
      } else {
        c[t][i] = *reinterpret_cast<const uint2*>(from + 8 * m.chunk);
        s[t][i] = (t ? p.cache.vs : p.cache.ks)[(int64_t)page * p.cache.s_page + h * p.cache.s_head + token];
      }
    }
  }
#pragma unroll
  for (int i = 0; i < kMoveHeads; ++i) {
    const int h = m.head[i];
    if (h >= p.cache.heads || (s0[i].b == p.sequences && !p.fill)) continue;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      if constexpr (CODES) {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t q = j < 2 ? c[t][i].x : c[t][i].y;
          const float lo = (float)(int8_t)(q >> (16 * (j & 1))), hi = (float)(int8_t)(q >> (16 * (j & 1) + 8));
          float a = lo * s[t][i], d = hi * s[t][i];   // (rounded to fp32 first, as the plain product is)
          __asm__("" : "+v"(a), "+v"(d));
          w[j] = pack2<DT>(a, d);
        }
        x[t][i] = make_uint4(w[0], w[1], w[2], w[3]);
      }
      char* to = t ? p.v + m.row[i] * p.v_row + h * p.v_head : p.k + m.row[i] * p.k_row + h * p.k_head;
      put16(to + 16 * m.chunk, x[t][i], p.stream);
    }
  }
}

static int head_lanes(int dim) { return dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }
static int64_t move_waves(const CacheMoveParams& p) { return p.pack > 1 ? (p.rows + p.pack - 1) / p.pack : p.rows * p.runs; }

template <bool WRITE, int DT, bool CODES, bool PACK>
static int launch_move(const char* who, const CacheMoveParams& in, hipStream_t stream) {
  CacheMoveParams p = in;
  const int lph = head_lanes(p.cache.dim);
  p.stream = p.rows * p.cache.heads * p.cache.dim * 4 > (64ll << 20);   // (k and v; 69277 rows of codes read: 80 -> 68 us)
  const dim3 g((unsigned)((move_waves(p) + 3) / 4)), t(256);
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, g, t, 0, stream, p); };
  if constexpr (WRITE) {
    lph == 8 ? go(cache_write_kernel<DT, CODES, 8, PACK>)
             : lph == 16 ? go(cache_write_kernel<DT, CODES, 16, PACK>) : go(cache_write_kernel<DT, CODES, 32, PACK>);
  } else {
    lph == 8 ? go(cache_read_kernel<DT, CODES, 8, PACK>)
             : lph == 16 ? go(cache_read_kernel<DT, CODES, 16, PACK>) : go(cache_read_kernel<DT, CODES, 32, PACK>);
  }
  return launch_status(who);
}

template <bool WRITE, int DT, bool CODES>
static int launch_move(const char* who, const CacheMoveParams& p, hipStream_t stream) {
  return p.pack > 1 ? launch_move<WRITE, DT, CODES, true>(who, p, stream) : launch_move<WRITE, DT, CODES, false>(who, p, stream);
}

template <bool WRITE>
static int launch_move_type(const char* who, int dtype, int held, const CacheMoveParams& p, hipStream_t stream) {
  const bool codes = held == W8A8_I8;
  if (!codes) return launch_move<WRITE, kF16, false>(who, p, stream);   // (16 bits are moved as they are)
  return dtype == W8A8_F16 ? launch_move<WRITE, kF16, true>(who, p, stream) : launch_move<WRITE, kBF16, true>(who, p, stream);
}

// The checks that both share; p's fields.
static int move_params(const char* who, int dtype, const W8A8KvCache& c, const void* k, const void* v,
                       const int64_t (&kst)[2], const int64_t (&vst)[2], int64_t rows, int64_t sequences,
                       const int32_t* table, int64_t ld_table, int64_t width, CacheMoveParams& p) {
  W8A8_REQUIRE(dtype == W8A8_F16 || dtype == W8A8_BF16, "%s: dtype %d not F16/BF16", who, dtype);
  W8A8_REQUIRE(rows >= 0 && rows < (1ll << 31) && sequences >= 0 && sequences < (1 << 20), "%s: rows or sequences out of range",
               who);
  W8A8_PASS(cache_view(who, c, p.cache));
  W8A8_REQUIRE(c.dtype == W8A8_I8 || c.dtype == dtype, "%s: a 16-bit cache takes rows of its own dtype", who);
  W8A8_PASS(rows_check(who, "k", k, kst));
  W8A8_PASS(rows_check(who, "v", v, vst));
  W8A8_REQUIRE(width >= 0 && width * c.page_size < (1ll << 27) && (width == 0 || sequences == 0 || table) &&
                   (sequences <= 1 || ld_table >= width),
               "%s: page table null, its rows overlap, or 2^27 keys and more", who);
  for (const RowsOf& r : {rows_memory(k, rows, c.heads, c.dim, kst), rows_memory(v, rows, c.heads, c.dim, vst)})
    W8A8_REQUIRE(apart_from_cache(r, c), "%s: rows overlap the cache", who);
  p.k = reinterpret_cast<char*>(const_cast<void*>(k));
  p.v = reinterpret_cast<char*>(const_cast<void*>(v));
  p.k_row = 2 * kst[0]; p.k_head = 2 * kst[1]; p.v_row = 2 * vst[0]; p.v_head = 2 * vst[1];
  p.rows = rows;
  const int per = kMoveHeads * 64 / head_lanes(c.dim);
  p.runs = (c.heads + per - 1) / per;
  p.pack = rows > 4096 && per / c.heads > 2 ? per / c.heads : 1;
  W8A8_REQUIRE((move_waves(p) + 3) / 4 < (1ll << 24), "%s: too many rows and heads for one launch", who);   // (2^32 work-items)
  p.sequences = (int)sequences;
  p.width = (int)width;
  p.table = table;
  p.ld_table = ld_table;
  p.lengths = nullptr;
  p.starts = nullptr;
  p.fill = 0;
  return W8A8_OK;
}

}  // namespace w8a8

extern "C" int w8a8_cache_write(const W8A8CacheWriteArgs* a) {
  using namespace w8a8;
  const char* who = "w8a8_cache_write";
  W8A8_REQUIRE(a != nullptr, "%s: null args", who);
  W8A8_REQUIRE(a->struct_size == sizeof(W8A8CacheWriteArgs), "%s: struct_size %u != %zu", who, a->struct_size,
               sizeof(W8A8CacheWriteArgs));
  if (a->rows == 0) return W8A8_OK;
  CacheMoveParams p;
  W8A8_PASS(move_params(who, a->dtype, a->cache, a->k, a->v, a->k_strides, a->v_strides, a->rows, a->sequences,
                        a->page_table, a->ld_table, a->table_width, p));
  W8A8_REQUIRE(a->sequences == 0 || a->lengths, "%s: null lengths", who);
  W8A8_REQUIRE(a->starts || a->rows == a->sequences, "%s: without starts every sequence has one row", who);
  W8A8_REQUIRE(places_apart(a->cache), "%s: keys or values of the cache share memory", who);
  W8A8_REQUIRE(cache_apart_from(a->cache, a->page_table, table_bytes(a->sequences, a->ld_table, a->table_width)) &&
                   cache_apart_from(a->cache, a->lengths, 4 * a->sequences) &&
                   cache_apart_from(a->cache, a->starts, 4 * (a->sequences + 1)),
               "%s: page table, lengths or starts lie in the cache", who);
  if (a->sequences == 0) return W8A8_OK;
  p.lengths = a->lengths;
  p.starts = a->starts;
  return launch_move_type<true>(who, a->dtype, a->cache.dtype, p, reinterpret_cast<hipStream_t>(a->stream));
}

extern "C" int w8a8_cache_read(const W8A8CacheReadArgs* a) {
  using namespace w8a8;
  const char* who = "w8a8_cache_read";
  W8A8_REQUIRE(a != nullptr, "%s: null args", who);
  W8A8_REQUIRE(a->struct_size == sizeof(W8A8CacheReadArgs), "%s: struct_size %u != %zu", who, a->struct_size,
               sizeof(W8A8CacheReadArgs));
  if (a->rows == 0) return W8A8_OK;
  CacheMoveParams p;
  W8A8_PASS(move_params(who, a->dtype, a->cache, a->k, a->v, a->k_strides, a->v_strides, a->rows, a->sequences,
                        a->page_table, a->ld_table, a->table_width, p));
  W8A8_REQUIRE(a->starts, "%s: null starts", who);
  W8A8_REQUIRE(rows_apart(a->rows, a->cache.heads, a->cache.dim, a->k_strides) &&
                   rows_apart(a->rows, a->cache.heads, a->cache.dim, a->v_strides) &&
                   apart(rows_memory(a->k, a->rows, a->cache.heads, a->cache.dim, a->k_strides),
                         rows_memory(a->v, a->rows, a->cache.heads, a->cache.dim, a->v_strides)),
               "%s: output rows overlap", who);
  for (const RowsOf& r : {rows_memory(a->k, a->rows, a->cache.heads, a->cache.dim, a->k_strides),
                          rows_memory(a->v, a->rows, a->cache.heads, a->cache.dim, a->v_strides)})
    W8A8_REQUIRE(apart_from(r, a->page_table, table_bytes(a->sequences, a->ld_table, a->table_width)) &&
                     apart_from(r, a->starts, 4 * (a->sequences + 1)),
                 "%s: page table or starts lie in an output", who);
  p.starts = a->starts;
  p.fill = a->fill;
  return launch_move_type<false>(who, a->dtype, a->cache.dtype, p, reinterpret_cast<hipStream_t>(a->stream));
}
