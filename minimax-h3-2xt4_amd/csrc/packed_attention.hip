// Attention of packed sequences of different lengths, causal or not, grouped
// heads, 16-bit operands.
//
//   o_i = sum_j 2^(c s_ij - m_i) v_j / sum_j 2^(c s_ij - m_i),
//   s_ij = q_i . k_j, c = log2(e) sm_scale, m_i the running maximum of c s_ij
//
// A workgroup takes 128 queries of one head, a wave 32 of them, and walks the
// keys in blocks that all four waves read from LDS. Scores are computed
// transposed, S^T = K Q^T on the 32 x 32 x 16 MFMA, so that a lane holds one
// query (l % 32) and sixteen of 32 keys, 8 a + 4 (l / 32) + b (a, b < 4): the
// softmax's maximum and sum are then a lane's own but for one exchange with
// lane l ^ 32, and P^T is the B operand of O^T += V^T P^T as it stands, the
// eight k of step s being keys 16 s + 4 (l / 32) + {0..3, 8..11}. V^T's operand
// is read from rows of V by ds_read_b64_tr_b16, which hands each lane four keys
// of one channel.
//
// Tiles are copied to LDS by the DMA form of buffer loads. A tile's descriptor
// ends with its sequence, so rows behind the end arrive as zeros (a masked key
// must not bring an infinity into a product with 0). 16-byte chunk c of row r
// lies at chunk c ^ k_swizzle(r) of K's tile and c ^ v_swizzle(r) of V's, so
// that the rows of one read fall on different banks.
#include "paged.h"

#include <type_traits>

namespace w8a8 {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

constexpr int kPackWaves = 4;
constexpr int kPackQ = 32 * kPackWaves;

struct PackedParams {
  const char* q;
  const char* k;
  const char* v;
  char* out;
  int64_t q_row, q_head, k_head, v_head, o_row, o_head;   // bytes
  uint32_t k_row, v_row;
  int rows, keys, sequences;
  int group, kv_heads, dim;
  const int32_t* starts;
  const int32_t* k_starts;
  float c;
  int fill;
};

template <int DT>
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// Chunks of 16 bytes: a key row of 2 DP bytes spans all banks (DP 128, 256), half
// or three quarters of them.
template <int DP>
__device__ __forceinline__ int k_swizzle(int r) {
  return DP == 64 ? (r >> 1) & 7 : DP == 96 ? (r >> 2) & 3 : r & 15;
}
template <int DP>
__device__ __forceinline__ int v_swizzle(int r) {
  return DP == 64 ? ((r >> 1) & 1) << 2 : DP == 96 ? 0 : (r & 3) << 2;
}

__device__ __forceinline__ int clamp_to(int v, int lo, int hi) { return min(max(v, lo), hi); }

// The wave's sequence and tile of queries of tile t, the tiles of a sequence
// taken from the last (of causal ones the longest) to the first. Behind the
// sequences come the tiles of the rows behind them, as a sequence of its own.
struct PackedTile {
  int b, first, n;   // first row of the tile in its sequence, the sequence's rows
  int row0;          // the sequence's first row
};

__device__ __forceinline__ PackedTile packed_find(const PackedParams& p, int t) {
  const int lane = threadIdx.x & 63;
  int sum = 0;
  for (int b0 = 0; b0 <= p.sequences; b0 += 64) {
    const int b = b0 + lane;
    int lo = 0, n = 0;
    if (b <= p.sequences) {
      lo = clamp_to(p.starts[b], 0, p.rows);
      n = clamp_to(b < p.sequences ? p.starts[b + 1] : p.rows, lo, p.rows) - lo;
    }
    const int tiles = (n + kPackQ - 1) / kPackQ;
    int upto = tiles;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int u = __shfl_up(upto, off, 64);
      if (lane >= off) upto += u;
    }
    upto += sum;
    const uint64_t past = __builtin_amdgcn_ballot_w64(upto > t);
    if (past) {
      const int at = __builtin_ctzll(past);
      PackedTile r;
      r.b = b0 + at;
      r.row0 = __builtin_amdgcn_readlane(lo, at);
      r.n = __builtin_amdgcn_readlane(n, at);
      r.first = (__builtin_amdgcn_readlane(upto, at) - 1 - t) * kPackQ;
      return r;
    }
    sum = __builtin_amdgcn_readlane(upto, 63);
  }
  return {-1, 0, 0, 0};
}

// DT: F16 or BF16; DP: dim rounded up to 64, 96, 128 or 256.
template <int DT, int DP, bool CAUSAL>
__global__ __launch_bounds__(64 * kPackWaves, 2) void packed_attention_kernel(PackedParams p) {
  constexpr int BK = DP > 128 ? 32 : 64;      // keys of a block
  constexpr int CH = DP / 8;                  // chunks of a row
  constexpr int NS = DP / 16, DF = DP / 32;   // steps of Q K^T, channel tiles of O^T
  constexpr int TF = BK / 32;                 // score tiles
  constexpr int kTile = BK * DP * 2;
  constexpr int kDma = kTile / (1024 * kPackWaves);   // DMA instructions of a wave for a tile
  __shared__ __attribute__((aligned(1024))) char kt[2][kTile], vt[2][kTile];
  __shared__ int again;
  const int lane = threadIdx.x & 63, col = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int item = blockIdx.x / p.kv_heads, kvh = blockIdx.x - item * p.kv_heads;
  const int head = kvh * p.group + item % p.group;
  const PackedTile tile = packed_find(p, item / p.group);
  if (tile.b < 0) return;
  const int q0 = tile.first + 32 * wave;      // the wave's first query of its sequence
  const int mine = q0 + col;
  const bool stored = mine < tile.n;
  char* to = p.out + (int64_t)(tile.row0 + min(mine, tile.n - 1)) * p.o_row + head * p.o_head;
  if (tile.b == p.sequences) {
    if (p.fill && stored)
      for (int d = 4 * half; d < p.dim; d += 8) *reinterpret_cast<uint2*>(to + 2 * d) = make_uint2(0, 0);
    return;
  }
  const int key0 = clamp_to(scalar_int(p.k_starts, tile.b), 0, p.keys);
  const int nk = clamp_to(scalar_int(p.k_starts, tile.b + 1), key0, p.keys) - key0;
  const int shift = nk - tile.n;              // causal: query i sees keys up to i + shift
  const int seen = CAUSAL ? clamp_to(tile.first + kPackQ + shift, 0, nk) : nk;   // of the workgroup
  const int blocks = (seen + BK - 1) / BK;
  const int limit = CAUSAL ? clamp_to(mine + shift + 1, 0, nk) : nk;             // of this query
  const int wave_clean = CAUSAL ? clamp_to(q0 + shift + 1, 0, nk) : nk;          // keys that all of the wave see
  const int wave_seen = CAUSAL ? clamp_to(q0 + 32 + shift, 0, nk) : nk;          // keys that some of it see

  v4u qf[NS];
  {
    const char* from = p.q + (int64_t)(tile.row0 + min(mine, tile.n - 1)) * p.q_row + head * p.q_head;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int d = 16 * s + 8 * half;
      qf[s] = v4u{0, 0, 0, 0};
      if (d < p.dim) qf[s] = *reinterpret_cast<const v4u*>(from + 2 * d);
    }
  }

  // Copies of a tile: lane l of instruction u of wave w brings what lies at
  // chunk (4 u + w) * 64 + l of the tile.
  uint32_t ksrc[kDma], vsrc[kDma];
#pragma unroll
  for (int u = 0; u < kDma; ++u) {
    const int at = (u * kPackWaves + wave) * 64 + lane, r = at / CH, c = at - r * CH;
    const int ck = c ^ k_swizzle<DP>(r), cv = c ^ v_swizzle<DP>(r);
    ksrc[u] = 8 * ck < p.dim ? r * p.k_row + 16 * ck : 0x7fffff00u;
    vsrc[u] = 8 * cv < p.dim ? r * p.v_row + 16 * cv : 0x7fffff00u;
  }
  const char* kbase = p.k + (int64_t)key0 * p.k_row + kvh * p.k_head;
  const char* vbase = p.v + (int64_t)key0 * p.v_row + kvh * p.v_head;
  auto copy = [&](const char* base, uint32_t row_b, const uint32_t (&src)[kDma], int block, char* dst) {
    const int rows = min(nk - block * BK, BK);
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + (int64_t)block * BK * row_b), 0,
                                                     (int)((rows - 1) * row_b) + 2 * p.dim, 0x00027000);
#pragma unroll
    for (int u = 0; u < kDma; ++u)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (__attribute__((address_space(3))) void*)(dst + (u * kPackWaves + wave) * 1024), 16, (int)src[u], 0, 0, 0);
  };
  auto copy_block = [&](int block, int buf) {
    copy(kbase, p.k_row, ksrc, block, kt[buf]);
    copy(vbase, p.v_row, vsrc, block, vt[buf]);
  };
  // Operands: key row col of score tile t, channels 16 s + 8 half; channel tile
  // f's column col of keys 16 s + 4 half + {0..3, 8..11}.
  auto k_frag = [&](const char* tile_at, int t, int s) {
    const int r = 32 * t + col;
    return *reinterpret_cast<const v4u*>(tile_at + r * (2 * DP) + (((2 * s + half) ^ k_swizzle<DP>(r)) << 4));
  };
  auto v_frag = [&](const char* tile_at, int f, int s) {
    v4u a;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 16 * s + 8 * e + 4 * half + ((lane & 15) >> 2);
      const int d = 32 * f + (lane & 16) + 4 * (lane & 3);
      const char* at = tile_at + r * (2 * DP) + (((d >> 3) ^ v_swizzle<DP>(r)) << 4) + 2 * (d & 7);
      const v2u w = __builtin_bit_cast(
          v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(at)));
      a[2 * e] = w.x;
      a[2 * e + 1] = w.y;
    }
    return a;
  };
  auto other_half = [](float x) {   // the larger or the sum over lanes l and l ^ 32 needs the other's value
    return __shfl_xor(x, 32, 64);
  };

  v16f o[DF];
  float m = -INFINITY, l = 0.0f;

  // One walk over the keys. CAREFUL: a masked key's value may be infinite or
  // NaN, and its product with P = 0 would not be 0. Such values are set to 0
  // for the product, and a count of the visible ones brings them back.
  auto walk = [&](auto careful_tag) {
    constexpr bool CAREFUL = decltype(careful_tag)::value;
#pragma unroll
    for (int f = 0; f < DF; ++f) o[f] = v16f{};
    m = -INFINITY;
    l = 0.0f;
    if (blocks > 0) copy_block(0, 0);
    for (int j = 0; j < blocks; ++j) {
      const int buf = j & 1;
      __builtin_amdgcn_s_waitcnt(0x0F70);   // this wave's copies of block j have landed,
      __syncthreads();                      // and everyone's; block j - 1 has been read
      if (j + 1 < blocks) copy_block(j + 1, buf ^ 1);
      const int first = j * BK;
      if (first >= wave_seen) continue;
      v16f s[TF];
#pragma unroll
      for (int t = 0; t < TF; ++t) {
        s[t] = v16f{};
#pragma unroll
        for (int i = 0; i < NS; ++i) s[t] = mfma32<DT>(k_frag(kt[buf], t, i), qf[i], s[t]);
      }
      const bool masked = first + BK > wave_clean;
      if (masked) {
#pragma unroll
        for (int t = 0; t < TF; ++t)
#pragma unroll
          for (int x = 0; x < 16; ++x)
            if (first + 32 * t + 8 * (x / 4) + 4 * half + x % 4 >= limit) s[t][x] = -INFINITY;
      }
      float mx = s[0][0];
#pragma unroll
      for (int t = 0; t < TF; ++t)
#pragma unroll
        for (int x = 0; x < 16; ++x) mx = fmaxf(mx, s[t][x]);
      mx = fmaxf(mx, other_half(mx));
      mx = fmaxf(m, mx);
      const float ref = mx == -INFINITY ? 0.0f : mx * p.c;
      const float fade = __builtin_amdgcn_exp2f(__builtin_fmaf(m, p.c, -ref));
      m = mx;
      float sum = 0.0f;
#pragma unroll
      for (int t = 0; t < TF; ++t)
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          s[t][x] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[t][x], p.c, -ref));
          sum += s[t][x];
        }
      l = __builtin_fmaf(l, fade, sum);
      if (__builtin_amdgcn_ballot_w64(fade != 1.0f)) {
#pragma unroll
        for (int f = 0; f < DF; ++f)
#pragma unroll
          for (int x = 0; x < 16; ++x) o[f][x] = o[f][x] * fade;
      }
      v4u pf[BK / 16];
#pragma unroll
      for (int i = 0; i < BK / 16; ++i)
#pragma unroll
        for (int x = 0; x < 4; ++x)
          pf[i][x] = pack2<DT>(s[i / 2][8 * (i % 2) + 2 * x], s[i / 2][8 * (i % 2) + 2 * x + 1]);
      if (!CAREFUL || !masked) {
#pragma unroll
        for (int i = 0; i < BK / 16; ++i)
#pragma unroll
          for (int f = 0; f < DF; ++f) o[f] = mfma32<DT>(v_frag(vt[buf], f, i), pf[i], o[f]);
      } else {
        constexpr uint32_t kInf = DT == kF16 ? 0x7c00u : 0x7f80u, kOne = DT == kF16 ? 0x3c00u : 0x3f80u;
#pragma unroll 1
        for (int f = 0; f < DF; ++f) {
          v16f up{}, down{}, add{};
#pragma unroll
          for (int i = 0; i < BK / 16; ++i) {
            const v4u a = v_frag(vt[buf], f, i);
            v4u fin, pos, neg, vis;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              uint32_t wf = 0, wp = 0, wn = 0, wv = 0;
#pragma unroll
              for (int y = 0; y < 2; ++y) {
                const uint32_t u = (a[x] >> (16 * y)) & 0xffffu, mag = u & 0x7fffu;
                const int key = first + 16 * i + 8 * (x / 2) + 4 * half + 2 * (x % 2) + y;
                wf |= (mag < kInf ? u : 0u) << (16 * y);
                wp |= (mag > kInf || u == kInf ? kOne : 0u) << (16 * y);
                wn |= (mag > kInf || u == (kInf | 0x8000u) ? kOne : 0u) << (16 * y);
                wv |= (key < limit ? kOne : 0u) << (16 * y);
              }
              fin[x] = wf; pos[x] = wp; neg[x] = wn; vis[x] = wv;
            }
            add = mfma32<DT>(fin, pf[i], add);
            up = mfma32<DT>(pos, vis, up);
            down = mfma32<DT>(neg, vis, down);
          }
#pragma unroll
          for (int x = 0; x < 16; ++x) {
            float y = add[x];
            if (up[x] > 0.0f) y += INFINITY;
            if (down[x] > 0.0f) y -= INFINITY;
            add[x] = y;
          }
#pragma unroll
          for (int g = 0; g < DF; ++g)
            if (g == f) {
#pragma unroll
              for (int x = 0; x < 16; ++x) o[g][x] = o[g][x] + add[x];
            }
        }
      }
    }
  };
  walk(std::false_type{});
  if constexpr (CAUSAL) {
    // Finite sums times 0 are 0: only where they are not can a masked value have come in.
    float z = 0.0f;
#pragma unroll
    for (int f = 0; f < DF; ++f)
#pragma unroll
      for (int x = 0; x < 16; ++x) z = __builtin_fmaf(o[f][x], 0.0f, z);
    if (threadIdx.x == 0) again = 0;
    __syncthreads();
    if (z != 0.0f) again = 1;
    __syncthreads();
    if (again) walk(std::true_type{});
  }

  l = l + other_half(l);
  const float rcp = l == 0.0f ? 0.0f : 1.0f / l;
  if (!stored) return;
#pragma unroll
  for (int f = 0; f < DF; ++f)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * f + 8 * g + 4 * half;
      if (d >= p.dim) continue;
      *reinterpret_cast<uint2*>(to + 2 * d) = make_uint2(pack2<DT>(o[f][4 * g] * rcp, o[f][4 * g + 1] * rcp),
                                                          pack2<DT>(o[f][4 * g + 2] * rcp, o[f][4 * g + 3] * rcp));
    }
}

template <int DT, int DP>
static int launch_packed(const PackedParams& p, bool causal, int64_t grid, hipStream_t s) {
  const dim3 g((unsigned)grid), t(64 * kPackWaves);
  if (causal) hipLaunchKernelGGL((packed_attention_kernel<DT, DP, true>), g, t, 0, s, p);
  else hipLaunchKernelGGL((packed_attention_kernel<DT, DP, false>), g, t, 0, s, p);
  return launch_status("w8a8_packed_attention");
}

template <int DT>
static int launch_packed_dim(const PackedParams& p, bool causal, int64_t grid, hipStream_t s) {
  if (p.dim <= 64) return launch_packed<DT, 64>(p, causal, grid, s);
  if (p.dim <= 96) return launch_packed<DT, 96>(p, causal, grid, s);
  if (p.dim <= 128) return launch_packed<DT, 128>(p, causal, grid, s);
  return launch_packed<DT, 256>(p, causal, grid, s);
}

}  // namespace w8a8

extern "C" int64_t w8a8_packed_attention_workspace_size(int64_t, int64_t, int64_t, int64_t, int32_t) { return 0; }

extern "C" int w8a8_packed_attention(const W8A8PackedAttentionArgs* a) {
  using namespace w8a8;
  const char* who = "w8a8_packed_attention";
  W8A8_REQUIRE(a != nullptr, "%s: null args", who);
  W8A8_REQUIRE(a->struct_size == sizeof(W8A8PackedAttentionArgs), "%s: struct_size %u != %zu", who, a->struct_size,
               sizeof(W8A8PackedAttentionArgs));
  W8A8_REQUIRE(a->dtype == W8A8_F16 || a->dtype == W8A8_BF16, "%s: dtype %d not F16/BF16", who, a->dtype);
  W8A8_REQUIRE(a->dim >= 8 && a->dim <= 256 && a->dim % 8 == 0, "%s: dim %d not a multiple of 8 up to 256", who, a->dim);
  W8A8_REQUIRE(a->kv_heads > 0 && a->heads > 0 && a->heads <= 65536 && a->heads % a->kv_heads == 0,
               "%s: heads out of range, or not a multiple of kv_heads", who);
  W8A8_REQUIRE(a->rows >= 0 && a->rows < (1 << 27) && a->keys >= 0 && a->keys < (1 << 27) && a->sequences >= 0 &&
                   a->sequences < (1 << 20),
               "%s: rows, keys or sequences out of range", who);
  W8A8_REQUIRE(a->sm_scale > 0.0f && std::isfinite(a->sm_scale), "%s: sm_scale must be positive and finite", who);
  W8A8_REQUIRE(a->causal == 0 || a->causal == 1, "%s: causal must be 0 or 1", who);
  if (a->rows == 0) return W8A8_OK;
  W8A8_PASS(rows_check(who, "q", a->q, a->q_strides));
  W8A8_PASS(rows_check(who, "out", a->out, a->out_strides));
  if (a->keys > 0) {
    W8A8_PASS(rows_check(who, "k", a->k, a->k_strides));
    W8A8_PASS(rows_check(who, "v", a->v, a->v_strides));
    W8A8_REQUIRE(a->k_strides[0] >= a->dim && a->v_strides[0] >= a->dim && a->k_strides[0] < (1 << 23) &&
                     a->v_strides[0] < (1 << 23),
                 "%s: row strides of k and v must be from dim to 2^23", who);
  }
  W8A8_REQUIRE(a->starts && a->k_starts, "%s: null starts", who);
  W8A8_REQUIRE(rows_apart(a->rows, a->heads, a->dim, a->out_strides), "%s: output rows overlap", who);
  const int64_t osize = rows_span(a->rows, a->heads, a->dim, a->out_strides);
  W8A8_REQUIRE(!spans_overlap(a->q, rows_span(a->rows, a->heads, a->dim, a->q_strides), a->out, osize) &&
                   (a->keys == 0 ||
                    (!spans_overlap(a->k, rows_span(a->keys, a->kv_heads, a->dim, a->k_strides), a->out, osize) &&
                     !spans_overlap(a->v, rows_span(a->keys, a->kv_heads, a->dim, a->v_strides), a->out, osize))),
               "%s: out overlaps an input", who);
  const int64_t grid = (a->rows / kPackQ + a->sequences + 1) * a->heads;
  W8A8_REQUIRE(grid < (1 << 24), "%s: too many rows, sequences and heads for one launch", who);   // (2^32 work-items)
  const PackedParams p{reinterpret_cast<const char*>(a->q), reinterpret_cast<const char*>(a->k),
                       reinterpret_cast<const char*>(a->v), reinterpret_cast<char*>(a->out),
                       2 * a->q_strides[0], 2 * a->q_strides[1], 2 * a->k_strides[1], 2 * a->v_strides[1],
                       2 * a->out_strides[0], 2 * a->out_strides[1],
                       (uint32_t)(2 * a->k_strides[0]), (uint32_t)(2 * a->v_strides[0]),
                       (int)a->rows, (int)a->keys, (int)a->sequences, a->heads / a->kv_heads, a->kv_heads, a->dim,
                       a->starts, a->k_starts, a->sm_scale * kLog2eF, a->fill};
  hipStream_t s = reinterpret_cast<hipStream_t>(a->stream);
  return a->dtype == W8A8_F16 ? launch_packed_dim<kF16>(p, a->causal != 0, grid, s)
                              : launch_packed_dim<kBF16>(p, a->causal != 0, grid, s);
}
