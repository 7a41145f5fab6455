// Packed sequences and the paged key-value cache: what the kernels of
// kv_cache.hip, cache_attend.hip and packed_attention.hip share.
#pragma once

#include "w8a8_device.h"
#include "w8a8_host.h"
#include "sequence_search.h"

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <utility>

namespace w8a8 {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef __bf16 v2b __attribute__((ext_vector_type(2)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

constexpr float kLog2eF = 1.44269504088896341f;
constexpr int kGroupTokens = 16;   // a page holds whole groups of so many tokens

// Tables and lengths are read by scalar loads where a wave agrees on the place
// (a vector load would wait behind the wave's own tiles).
typedef const __attribute__((address_space(4))) int32_t* ScalarInts;
__device__ __forceinline__ int scalar_int(const int32_t* p, int64_t i) { return ((ScalarInts)p)[i]; }

// Two fp32 as a word of two DT values, rounded to nearest even, a in the low half.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (DT == kF16) return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2h));
  else return __builtin_bit_cast(uint32_t, __builtin_convertvector(v2f{a, b}, v2b));
}

// The reference of p may lie so much below the maximum of its exponent (as a power
// of 2): rescaling the sums is rare.
constexpr float kSlack = 8.0f;
// P is p times 2^kLift, so that it ends at 2^15 in fp16, of its 2^16, and what is lost
// there lies below 2^-32 of the largest p: relative to the reference itself, 2^-25,
// thousands of keys that share a part of the weight were 0 beside one key. In bf16,
// whose values reach 2^128 as fp32 sums do, it is at most 1: finite values weigh in
// as finite products.
template <int DT>
constexpr float kLift = DT == kF16 ? 7.0f : -kSlack;

// The reference of a row with keys, whose scores are all -inf: 0 / 0 is its output,
// and 0 that of a row without keys, whose reference is -inf.
__device__ __forceinline__ float with_keys(float ref, bool any) { return any ? fmaxf(ref, -FLT_MAX) : ref; }

// l plus the two DT values of a word.
template <int DT>
__device__ __forceinline__ float add2(uint32_t w, float l) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(v2h, w), __builtin_bit_cast(v2h, 0x3c003c00u), l, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(v2b, w), __builtin_bit_cast(v2b, 0x3f803f80u), l, false);
}

// A cache as the kernels take it: strides in bytes (scales': in floats).
struct CacheView {
  char* k;
  char* v;
  float* ks;
  float* vs;
  int64_t page_b, head_b, s_page, s_head;
  uint32_t token_b;
  int pages, page_size, heads, dim;
  uint64_t magic;   // floor(2^36 / groups a page) + 1
};

// Page of the table and token within it of a sequence's group of 16 tokens
// (g < 2^23): with d groups a page (d <= 256) magic = 2^36/d + e, 0 < e <= 1,
// and g * e / 2^36 < 1/d, so the quotient is floor(g / d).
__device__ __forceinline__ void group_place(const CacheView& c, uint32_t g, int& entry, int& token) {
  entry = (int)(((uint64_t)g * c.magic) >> 36);
  token = ((int)g - entry * (c.page_size / kGroupTokens)) * kGroupTokens;
}

inline bool stride8(int64_t s) { return s >= 0 && s % 8 == 0; }

// Checks of a W8A8KvCache and its view.
inline int cache_view(const char* who, const W8A8KvCache& c, CacheView& v) {
  const bool codes = c.dtype == W8A8_I8;
  W8A8_REQUIRE(codes || c.dtype == W8A8_F16 || c.dtype == W8A8_BF16, "%s: cache dtype %d not F16/BF16/I8", who, c.dtype);
  W8A8_REQUIRE(c.k && c.v && aligned16(c.k) && aligned16(c.v), "%s: cache k or v null or misaligned", who);
  W8A8_REQUIRE(c.dim >= 8 && c.dim <= 256 && c.dim % 8 == 0, "%s: dim %d not a multiple of 8 up to 256", who, c.dim);
  W8A8_REQUIRE(c.heads > 0 && c.heads <= 65536 && c.pages > 0 && c.pages < (1ll << 31), "%s: heads or pages out of range",
               who);
  W8A8_REQUIRE(c.page_size > 0 && c.page_size <= 4096 && c.page_size % kGroupTokens == 0,
               "%s: page_size %d not a multiple of 16 up to 4096", who, c.page_size);
  W8A8_REQUIRE(stride8(c.strides[0]) && stride8(c.strides[1]) && stride8(c.strides[2]) && c.strides[2] >= c.dim &&
                   c.strides[2] < (1ll << 26),
               "%s: cache strides must be multiples of 8, the token's from dim to 2^26", who);
  if (codes)
    W8A8_REQUIRE(c.k_scale && c.v_scale && aligned16(c.k_scale) && aligned16(c.v_scale) && c.scale_strides[0] >= 0 &&
                     c.scale_strides[1] >= 0 && c.scale_strides[0] % 4 == 0 && c.scale_strides[1] % 4 == 0,
                 "%s: codes need k_scale and v_scale, 16-byte aligned, strides multiples of 4", who);
  const int es = codes ? 1 : 2;
  v = CacheView{reinterpret_cast<char*>(c.k), reinterpret_cast<char*>(c.v), c.k_scale, c.v_scale,
                c.strides[0] * es, c.strides[1] * es, c.scale_strides[0], c.scale_strides[1],
                (uint32_t)(c.strides[2] * es), (int)c.pages, c.page_size, c.heads, c.dim,
                (1ull << 36) / (uint64_t)(c.page_size / kGroupTokens) + 1};
  return W8A8_OK;
}

// Checks of rows [n, heads, dim] of 16-bit elements with strides {row, head}.
inline int rows_check(const char* who, const char* name, const void* p, const int64_t (&st)[2]) {
  W8A8_REQUIRE(p && aligned16(p), "%s: %s null or misaligned", who, name);
  W8A8_REQUIRE(stride8(st[0]) && stride8(st[1]), "%s: %s strides must be multiples of 8 elements", who, name);
  return W8A8_OK;
}

// Whether rows [n, heads, dim] with these strides are written once each.
inline bool rows_apart(int64_t n, int64_t heads, int64_t dim, const int64_t (&st)[2]) {
  const bool row_in = n <= 1 || heads <= 1 || st[0] >= st[1];   // heads within a row, or rows within a head
  const int64_t in = row_in ? (heads > 1 ? st[1] : dim) : st[0];
  const int64_t span = (row_in ? (heads - 1) * (heads > 1 ? st[1] : 0) : (n - 1) * st[0]) + dim;
  const int64_t out = row_in ? (n > 1 ? st[0] : span) : st[1];
  return in >= dim && out >= dim && (out >= span || in >= ((row_in ? n : heads) - 1) * out + dim);
}

// The memory of such rows of 16-bit elements, and of a cache's keys or values.
inline RowsOf rows_memory(const void* p, int64_t n, int64_t heads, int64_t dim, const int64_t (&st)[2]) {
  return rows_of(p, st[0], n, (heads - 1) * st[1] + dim, 2);
}
inline RowsOf cache_memory(const W8A8KvCache& c, const void* p) {
  const int es = c.dtype == W8A8_I8 ? 1 : 2;
  const int64_t page = (c.heads - 1) * c.strides[1] + (c.page_size - 1) * c.strides[2] + c.dim;
  return rows_of(p, c.strides[0], c.pages, page, es);
}
inline RowsOf scale_memory(const W8A8KvCache& c, const float* p) {
  return rows_of(p, c.scale_strides[0], c.pages, (c.heads - 1) * c.scale_strides[1] + c.page_size, 4);
}
// Whether rows share no byte with a cache's keys, values and scales.
inline bool apart_from_cache(const RowsOf& r, const W8A8KvCache& c) {
  return apart(r, cache_memory(c, c.k)) && apart(r, cache_memory(c, c.v)) &&
         (c.dtype != W8A8_I8 || (apart(r, scale_memory(c, c.k_scale)) && apart(r, scale_memory(c, c.v_scale))));
}

// Whether rows, or a cache, share no byte with a run of them: the integers that a
// kernel reads while it writes there, a workspace.
inline bool apart_from(const RowsOf& r, const void* p, int64_t bytes) {
  return !p || bytes <= 0 || apart(r, RowsOf{p, r.row, bytes, bytes});
}
inline bool cache_apart_from(const W8A8KvCache& c, const void* p, int64_t bytes) {
  return apart_from(cache_memory(c, c.k), p, bytes) && apart_from(cache_memory(c, c.v), p, bytes) &&
         (c.dtype != W8A8_I8 ||
          (apart_from(scale_memory(c, c.k_scale), p, bytes) && apart_from(scale_memory(c, c.v_scale), p, bytes)));
}
inline int64_t table_bytes(int64_t sequences, int64_t ld, int64_t width) {
  return sequences > 0 && width > 0 ? 4 * ((sequences - 1) * ld + width) : 0;
}

// Runs of `extent` bytes, or of another such nest of `other` bytes, one at each
// place of a nest of steps.
struct Places {
  int64_t step[3], count[3], extent, other;   // the larger steps first
};
// Sorted by their steps; false where steps are less than what they step over.
inline bool places_nest(Places& p) {
  for (int i = 0; i < 3; ++i)
    for (int j = i + 1; j < 3; ++j)
      if (p.count[i] <= 1 || (p.count[j] > 1 && p.step[j] > p.step[i])) {
        std::swap(p.step[i], p.step[j]);
        std::swap(p.count[i], p.count[j]);
      }
  int64_t span = std::max(p.extent, p.other);
  for (int i = 2; i >= 0; --i) {
    if (p.count[i] <= 1) continue;
    if (p.step[i] < span) return false;
    span += (p.count[i] - 1) * p.step[i];
  }
  return true;
}
// Whether two such nests, the other `off` bytes behind the one, share a byte. Places differ by sums
// c_i step_i, |c_i| < count_i, and what the inner steps reach is less than a step,
// so that c_i is one of two.
inline bool places_meet(const Places& p, int64_t off, int i = 0) {
  if (i == 3) return -p.other < off && off < p.extent;
  if (p.count[i] <= 1) return places_meet(p, off, i + 1);
  const int64_t c = off / p.step[i] - (off % p.step[i] < 0);
  for (int64_t at : {c, c + 1})
    if (-p.count[i] < at && at < p.count[i] && places_meet(p, off - at * p.step[i], i + 1)) return true;
  return false;
}
// Whether every key, value and scale of a cache has memory of its own. Codes and
// scales have it where all of a page's lie apart, or all of a head's in steps that
// both take.
inline bool places_apart(const W8A8KvCache& c) {
  const bool codes = c.dtype == W8A8_I8;
  const int64_t es = codes ? 1 : 2, row = c.dim * es, scales = 4ll * c.page_size;
  const int64_t page = c.strides[0] * es, head = c.strides[1] * es, token = c.strides[2] * es;
  const int64_t s_page = c.scale_strides[0] * 4, s_head = c.scale_strides[1] * 4;
  auto own = [](Places p, const void* a, const void* b) {
    return places_nest(p) && !places_meet(p, (int64_t)((uintptr_t)b - (uintptr_t)a));
  };
  auto beside = [&](const void* x, const float* s) {
    return apart(cache_memory(c, x), scale_memory(c, s)) ||
           ((c.pages == 1 || page == s_page) && (c.heads == 1 || head == s_head) &&
            own({{page, head, 0}, {c.pages, c.heads, 1}, (c.page_size - 1) * token + row, scales}, x, s));
  };
  return own({{page, head, token}, {c.pages, c.heads, c.page_size}, row, row}, c.k, c.v) &&
         (!codes || (own({{s_page, s_head, 0}, {c.pages, c.heads, 1}, scales, scales}, c.k_scale, c.v_scale) &&
                     beside(c.k, c.k_scale) && beside(c.k, c.v_scale) && beside(c.v, c.k_scale) && beside(c.v, c.v_scale)));
}

}  // namespace w8a8

#define W8A8_PASS(expr)                  \
  do {                                   \
    const int rc_ = (expr);              \
    if (rc_ != W8A8_OK) return rc_;      \
  } while (0)
