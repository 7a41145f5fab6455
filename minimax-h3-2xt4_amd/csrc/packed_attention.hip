// Attention of packed sequences of different lengths, causal or not, grouped
// heads, 16-bit operands.
//
//   o_i = sum_j 2^(c s_ij - m_i) v_j / sum_j 2^(c s_ij - m_i),
//   s_ij = q_i . k_j, c = log2(e) sm_scale, m_i a reference near the running maximum
//   of c s_ij
//
// A workgroup takes 128 rows of a key head (a query with one of the group's query
// heads each), a wave 32 of them, and walks the keys in blocks that all four
// waves read from LDS. Scores are computed transposed, S^T = K Q^T on the 32 x 32
// x 16 MFMA, so that a lane holds one row (l % 32) and sixteen of 32 keys,
// 8 a + 4 (l / 32) + b (a, b < 4): the softmax's maximum and sum are then a lane's
// own but for one exchange with lane l ^ 32, and P^T is the B operand of
// O^T += V^T P^T as it stands, the eight k of step s being keys 16 s + 4 (l / 32) +
// {0..3, 8..11}. V^T's operand is read from rows of V by ds_read_b64_tr_b16, which
// hands each lane four keys of one channel.
//
// Bound by the board's power where it is long: 16384 causal rows of 64 heads of
// 128 in bf16 take 3.75 to 4.05 ms by the board, 1086 to 1174 TFLOP/s, with the MFMAs
// busy 62 % of the cycles at 1.79 GHz. A loop of nothing but MFMAs and these LDS reads
// reaches 1540 to 1640 TFLOP/s on random operands, and 1170 to 1220 with the softmax's
// instructions between them (1180 to 1206 on 16 x 16 x 32 MFMAs); the library's 8192^3
// product 1185 to 1440. Moving work between
// the MFMAs, reading further ahead or raising waves' priorities changes it by less
// than 1 %. Fewer instructions do: a lazy reference, a row sum by dot products of
// the packed words. Two workgroups a CU, so that the two waves of a SIMD wait at
// different barriers. A prompt of 353 rows (13 us) is its chain: 1.5 us to find the
// tile, 1.3 for the first tiles, six steps of about 1, 1.2 to store.
//
// Tiles are copied to LDS by the DMA form of buffer loads. A tile's descriptor
// ends with its sequence, so rows behind the end arrive as zeros (a masked key
// must not bring an infinity into a product with 0). 16-byte chunk c of row r
// lies at chunk c ^ k_swizzle(r) of K's tile and c ^ v_swizzle(r) of V's, so
// that the rows of one read fall on different banks.
#include "paged.h"
#include "packed_tiles.h"

#include <algorithm>
#include <type_traits>
#include <utility>

namespace w8a8 {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef short v4s __attribute__((ext_vector_type(4)));

struct PackedParams {
  const char* q;
  const char* k;
  const char* v;
  char* out;
  int64_t q_row, q_head, k_head, v_head, o_row, o_head;   // bytes
  uint32_t k_row, v_row;
  int rows, keys, sequences;
  int group, kv_heads, dim;
  uint64_t group_magic;   // floor((2^64 - 1) / group) + 1
  const int32_t* starts;
  const int32_t* k_starts;
  float c;
  int fill;
  int splits;       // ranges of a tile's keys, each a workgroup's
  float* part;      // [splits][rows][heads][channels, whole tiles of 32]
  float* part_ml;   // [splits][rows][heads][2]: reference, sum
};

template <int DT>
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// Both halves' values of a pair of lanes l, l ^ 32.
__device__ __forceinline__ std::pair<float, float> lane_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return {__uint_as_float(r[0]), __uint_as_float(r[1])};
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

// r / group (r >= 0): the high half of r * (2^64 / group + e), 0 < e <= 1, where
// r e < 2^32 leaves the quotient's floor.
__device__ __forceinline__ int by_group(const PackedParams& p, int r) {
  return p.group == 1 ? r : (int)__umul64hi((uint64_t)(uint32_t)r, p.group_magic);
}

// What a workgroup and its waves work on, DP channels wide, BK keys a block.
// TID is the thread's index (a copy of it that the compiler takes for another
// value keeps nothing alive from the one's use to the other's). Tiles are PITCH
// channels wide, whole MFMA tiles of O: 80 channels are five steps of Q K^T, but
// three tiles. The 16 channels to spare then are ones in V's tile, and those of O
// the sums of P, without instructions of their own (21591 rows of 72 channels
// 645 -> 608 us).
template <int DT, int DP, bool CAUSAL, bool SPLIT>
struct Packed {
  static constexpr int BK = DP > 128 ? 32 : 64;      // keys of a block
  static constexpr int NS = DP / 16, DF = (DP + 31) / 32;   // steps of Q K^T, channel tiles of O^T
  static constexpr int PITCH = 32 * DF, CH = PITCH / 8;     // channels and chunks of a row
  static constexpr int TF = BK / 32;                        // score tiles
  static constexpr bool kOnes = PITCH > DP;
  static constexpr int kTile = BK * PITCH * 2;
  static constexpr uint32_t kOnesHere = 0xffffffffu;   // (not copied)
  static constexpr int kDma = kTile / (1024 * kPackWaves);   // DMA instructions of a wave for a tile

  const PackedParams& p;
  char* tiles;
  int lane, wave, col, half;
  PackedTile tile;
  int query, head, nk, split;   // of this lane's row
  bool stored;
  int blocks, limit, wave_clean, wave_blocks;
  const char* kbase;
  const char* vbase;
  uint32_t ksrc[kDma], vsrc[kDma];

  __device__ __forceinline__ Packed(const PackedParams& p_, char* tiles_, int tid) : p(p_), tiles(tiles_) {
    lane = tid & 63;
    wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    col = lane & 31;
    half = lane >> 5;
    // Neighbours are the key heads: workgroups go round the XCDs in turn, so with
    // a multiple of eight of them a key head's stay with one XCD's cache.
    int item = blockIdx.x / p.kv_heads;
    const int kvh = blockIdx.x - item * p.kv_heads;
    split = 0;
    if constexpr (SPLIT) {
      split = item % p.splits;
      item /= p.splits;
    }
    tile = packed_find(p, item);
    if (tile.b < 0) return;
    const int r0 = tile.first + 32 * wave, row = min(r0 + col, tile.n - 1);   // the wave's first row, and this lane's
    stored = r0 + col < tile.n;
    query = by_group(p, row);
    head = kvh * p.group + row - query * p.group;
    if (tile.b == p.sequences) return;
    nk = tile.nk;
    const int shift = nk - by_group(p, tile.n);    // causal: query i sees keys up to i + shift
    auto sees = [&](int r) { return CAUSAL ? clamp_to(by_group(p, min(r, tile.n - 1)) + shift + 1, 0, nk) : nk; };
    const int seen = sees(tile.first + kPackQ - 1);                 // keys that the workgroup sees,
    limit = CAUSAL ? clamp_to(query + shift + 1, 0, nk) : nk;       // this query,
    wave_clean = sees(r0);                                          // all of the wave's,
    wave_blocks = ((r0 < tile.n ? sees(r0 + 31) : 0) + BK - 1) / BK;   // and some of them (in blocks)
    blocks = (seen + BK - 1) / BK;
    int64_t from = tile.key0;
    if constexpr (SPLIT) {   // the keys before this range's first are another's: count from there
      const int begin = blocks * split / p.splits, end = blocks * (split + 1) / p.splits, off = begin * BK;
      blocks = end - begin;
      wave_blocks = clamp_to(wave_blocks - begin, 0, blocks);
      nk -= off;
      limit -= off;
      wave_clean -= off;
      from += off;
    }
    kbase = p.k + from * p.k_row + kvh * p.k_head;
    vbase = p.v + from * p.v_row + kvh * p.v_head;
    // Copies of a tile: lane l of instruction u of wave w brings what lies at
    // chunk (4 u + w) * 64 + l of the tile.
#pragma unroll
    for (int u = 0; u < kDma; ++u) {
      const int at = (u * kPackWaves + wave) * 64 + lane, r = at / CH, c = at - r * CH;
      const int ck = c ^ k_swizzle<PITCH>(r), cv = c ^ v_swizzle<PITCH>(r);
      ksrc[u] = 8 * ck < p.dim ? r * p.k_row + 16 * ck : 0x7fffff00u;
      vsrc[u] = 8 * cv < p.dim ? r * p.v_row + 16 * cv : kOnes && 8 * cv >= DP ? kOnesHere : 0x7fffff00u;
    }
  }

  __device__ __forceinline__ char* to() const {
    return p.out + (int64_t)(tile.row0 + query) * p.o_row + head * p.o_head;
  }

  __device__ __forceinline__ void queries(v4u (&qf)[NS]) const {
    const char* from = p.q + (int64_t)(tile.row0 + query) * p.q_row + head * p.q_head;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const int d = 16 * s + 8 * half;
      qf[s] = v4u{0, 0, 0, 0};
      if (d < p.dim) qf[s] = *reinterpret_cast<const v4u*>(from + 2 * d);
    }
  }

  __device__ __forceinline__ char* kt(int i) const { return tiles + i * kTile; }
  __device__ __forceinline__ char* vt(int i) const { return tiles + (2 + i) * kTile; }
  template <bool ONES>
  __device__ __forceinline__ void copy(const char* base, uint32_t row_b, const uint32_t (&src)[kDma], int block,
                                       char* dst) const {
    const int rows = min(nk - block * BK, BK);
    const auto r = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(base + (int64_t)block * BK * row_b), 0,
                                                     (int)((rows - 1) * row_b) + 2 * p.dim, 0x00027000);
#pragma unroll
    for (int u = 0; u < kDma; ++u)
      if (!ONES || src[u] != kOnesHere) __builtin_amdgcn_raw_ptr_buffer_load_lds(
          r, (__attribute__((address_space(3))) void*)(dst + (u * kPackWaves + wave) * 1024), 16, (int)src[u], 0, 0, 0);
  }
  __device__ __forceinline__ void copy_k(int block, char* dst) const { copy<false>(kbase, p.k_row, ksrc, block, dst); }
  __device__ __forceinline__ void copy_v(int block, char* dst) const { copy<kOnes>(vbase, p.v_row, vsrc, block, dst); }
  // The ones, before the first copies are waited for.
  __device__ __forceinline__ void put_ones(int tid) const {
    if constexpr (kOnes) {
      static_assert(64 * kPackWaves == 4 * BK && CH - DP / 8 == 2, "a thread for each chunk of two tiles");
      const int r = tid % BK, c = DP / 8 + tid / BK % 2;
      constexpr uint32_t kOne = DT == kF16 ? 0x3c003c00u : 0x3f803f80u;
      *reinterpret_cast<v4u*>(vt(tid / BK / 2) + r * (2 * PITCH) + ((c ^ v_swizzle<PITCH>(r)) << 4)) = v4u{kOne, kOne, kOne, kOne};
    }
  }
  // This half's sum of P.
  __device__ __forceinline__ float sum_of(const v16f (&o)[DF], float l) const {
    if constexpr (!kOnes) return l;
    else return half == 0 ? o[DP / 32][DP % 32 / 2] : 0.0f;   // channel DP
  }

  // Operands: key row col of score tile t, channels 16 s + 8 half; channel tile
  // f's column col of keys 16 s + 4 half + {0..3, 8..11}.
  __device__ __forceinline__ v4u k_frag(const char* from, int t, int s) const {
    const int r = 32 * t + col;
    return *reinterpret_cast<const v4u*>(from + r * (2 * PITCH) + (((2 * s + half) ^ k_swizzle<PITCH>(r)) << 4));
  }
  __device__ __forceinline__ v4u v_frag(const char* from, int f, int s) const {
    v4u a;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int r = 16 * s + 8 * e + 4 * half + ((lane & 15) >> 2);
      const int d = 32 * f + (lane & 16) + 4 * (lane & 3);
      const char* at = from + r * (2 * PITCH) + (((d >> 3) ^ v_swizzle<PITCH>(r)) << 4) + 2 * (d & 7);
      const v2u w = __builtin_bit_cast(
          v2u, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) v4s*)(at)));
      a[2 * e] = w.x;
      a[2 * e + 1] = w.y;
    }
    return a;
  }
  // Product n of a block's scores is step n / TF of score tile n % TF, product n
  // of its values step n / DF of channel tile n % DF: neighbours are independent.
  __device__ __forceinline__ v4u k_of(const char* from, int n) const { return k_frag(from, n % TF, n / TF); }
  __device__ __forceinline__ v4u v_of(const char* from, int n) const { return v_frag(from, n % DF, n / DF); }

  // The largest of a block's scores; those behind a query's last key set to -inf.
  static __device__ __forceinline__ float largest(const v16f (&x)[TF]) {
    float mx = x[0][0];
#pragma unroll
    for (int t = 0; t < TF; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e) mx = fmaxf(mx, x[t][e]);
    return mx;
  }
  __device__ __forceinline__ void mask(int j, v16f (&x)[TF]) const {
    __asm__ volatile("");   // (not to be done without the branch)
#pragma unroll
    for (int t = 0; t < TF; ++t)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (j * BK + 32 * t + 8 * (e / 4) + 4 * half + e % 4 >= limit) x[t][e] = -INFINITY;
  }

  __device__ __forceinline__ void store(const v16f (&o)[DF], float ref, float l) const {
    const auto both = lane_halves(l);
    l = both.first + both.second;
    ref = with_keys(ref, limit > 0);   // (of a range: whether the row sees keys from its first on)
    if constexpr (SPLIT) {
      if (!stored) return;
      const int64_t at = ((int64_t)split * p.rows + tile.row0 + query) * (p.group * p.kv_heads) + head;
#pragma unroll
      for (int f = 0; f < DF; ++f)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<v4f*>(p.part + at * PITCH + 32 * f + 8 * g + 4 * half) =
              v4f{o[f][4 * g], o[f][4 * g + 1], o[f][4 * g + 2], o[f][4 * g + 3]};
      if (half == 0) *reinterpret_cast<float2*>(p.part_ml + 2 * at) = make_float2(ref, l);
      return;
    }
    const float rcp = ref == -INFINITY ? 0.0f : 1.0f / l;
    if (!stored) return;
    char* at = to();
#pragma unroll
    for (int f = 0; f < DF; ++f)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d = 32 * f + 8 * g + 4 * half;
        if (d >= p.dim) continue;
        *reinterpret_cast<uint2*>(at + 2 * d) = make_uint2(pack2<DT>(o[f][4 * g] * rcp, o[f][4 * g + 1] * rcp),
                                                            pack2<DT>(o[f][4 * g + 2] * rcp, o[f][4 * g + 3] * rcp));
      }
  }
};

// The sums, the exponent that p is relative to and this half's sum of p. The
// reference follows the maximum only once that lies more than kSlack above it.
template <int DT, int DF>
struct PackedState {
  v16f o[DF];
  float ref, l;
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int f = 0; f < DF; ++f) o[f] = v16f{};
    ref = -INFINITY;
    l = 0.0f;
  }
  __device__ __forceinline__ void follow(float mx) {
    if (__builtin_amdgcn_ballot_w64(mx > ref + kSlack) == 0) return;
    const auto both = lane_halves(mx);
    const float to = fmaxf(ref, fmaxf(both.first, both.second));
    const float fade = to == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(ref - to);
    ref = to;
    l = l * fade;
#pragma unroll
    for (int f = 0; f < DF; ++f)
#pragma unroll
      for (int x = 0; x < 16; ++x) o[f][x] = o[f][x] * fade;
  }
  __device__ __forceinline__ float at() const { return ref == -INFINITY ? 0.0f : ref - kLift<DT>; }
};

// The walk again for a workgroup with sums that are not finite, causal only: a
// masked key's value may be infinite or NaN, and its product with P = 0 is not 0.
// In blocks with masked keys such values are set to 0 for the product, and a
// count of those that a query sees brings them back. One block at a time.
template <int DT, int DP, bool SPLIT>
__device__ __forceinline__ void packed_careful(const PackedParams& p, char* tiles) {
  int tid = threadIdx.x;
  __asm__ volatile("" : "+v"(tid));
  using W = Packed<DT, DP, true, SPLIT>;
  const W w(p, tiles, tid);
  v4u qf[W::NS];
  w.queries(qf);
  PackedState<DT, W::DF> st;
  st.clear();
#pragma unroll 1
  for (int j = 0; j < w.blocks; ++j) {
    __syncthreads();   // the last block has been read
    w.copy_k(j, w.kt(0));
    w.copy_v(j, w.vt(0));
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
    if (j >= w.wave_blocks) continue;
    v16f s[W::TF];
#pragma unroll
    for (int t = 0; t < W::TF; ++t) s[t] = v16f{};
#pragma unroll
    for (int n = 0; n < W::TF * W::NS; ++n) s[n % W::TF] = mfma32<DT>(w.k_of(w.kt(0), n), qf[n / W::TF], s[n % W::TF]);
    w.mask(j, s);
    st.follow(W::largest(s) * p.c);
    v4u pf[W::BK / 16];
    const float at = st.at();
#pragma unroll
    for (int i = 0; i < 8 * W::TF; ++i) {
      const float a = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 8][2 * (i % 8)], p.c, -at));
      const float b = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i / 8][2 * (i % 8) + 1], p.c, -at));
      pf[i / 4][i % 4] = pack2<DT>(a, b);
      st.l = add2<DT>(pf[i / 4][i % 4], st.l);
    }
    const int sees = (j + 1) * W::BK > w.wave_clean ? w.limit : INT32_MAX;
    constexpr uint32_t kInf = DT == kF16 ? 0x7c00u : 0x7f80u, kOne = DT == kF16 ? 0x3c00u : 0x3f80u;
#pragma unroll
    for (int f = 0; f < W::DF; ++f) {
      v16f up{}, down{};
#pragma unroll
      for (int i = 0; i < W::BK / 16; ++i) {
        const v4u a = w.v_frag(w.vt(0), f, i);
        v4u fin, pos, neg, vis;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          uint32_t wf = 0, wp = 0, wn = 0, wv = 0;
#pragma unroll
          for (int y = 0; y < 2; ++y) {
            const uint32_t u = (a[x] >> (16 * y)) & 0xffffu, mag = u & 0x7fffu;
            const int key = j * W::BK + 16 * i + 8 * (x / 2) + 4 * w.half + 2 * (x % 2) + y;
            wf |= (mag < kInf ? u : 0u) << (16 * y);
            wp |= (mag > kInf || u == kInf ? kOne : 0u) << (16 * y);
            wn |= (mag > kInf || u == (kInf | 0x8000u) ? kOne : 0u) << (16 * y);
            wv |= (key < sees ? kOne : 0u) << (16 * y);
          }
          fin[x] = wf; pos[x] = wp; neg[x] = wn; vis[x] = wv;
        }
        st.o[f] = mfma32<DT>(fin, pf[i], st.o[f]);
        up = mfma32<DT>(pos, vis, up);
        down = mfma32<DT>(neg, vis, down);
      }
#pragma unroll
      for (int x = 0; x < 16; ++x) {
        float y = st.o[f][x];
        if (up[x] > 0.0f) y += INFINITY;
        if (down[x] > 0.0f) y -= INFINITY;
        st.o[f][x] = y;
      }
    }
  }
  w.store(st.o, st.ref, st.l);
}

// DT: F16 or BF16; DP: dim rounded up to 64, 80, 96, 128 or 256.
//
// Step j forms block j's probabilities between the MFMAs that score block j + 1
// and, the last of them, between the first that add block j's values; between
// the others it takes block j + 1's maximum. K of block j + 1 and V of block j are
// read in a step, so K's copies run a step ahead of V's. The order is laid out
// product by product (left to the compiler, all fragments are read at once, whose
// registers spill, and the VALU's work follows the MFMAs'). As laid out the 128-wide
// kernels still spill 6 to 10 registers, the others none.
template <int DT, int DP, bool CAUSAL, bool SPLIT>
__global__ __launch_bounds__(64 * kPackWaves, DP > 128 ? 1 : 2) void packed_attention_kernel(PackedParams p) {
  using W = Packed<DT, DP, CAUSAL, SPLIT>;
  constexpr int BK = W::BK, NS = W::NS, DF = W::DF, TF = W::TF;
  constexpr int QK = TF * NS, PV = BK / 16 * DF, AHEAD = 3;
  __shared__ __attribute__((aligned(1024))) char tiles[4 * W::kTile];   // two of K, two of V
  const W w(p, tiles, threadIdx.x);
  if (w.tile.b < 0) return;
  if (w.tile.b == p.sequences) {
    if (p.fill && w.stored && w.split == 0)
      for (int d = 4 * w.half; d < p.dim; d += 8) *reinterpret_cast<uint2*>(w.to() + 2 * d) = make_uint2(0, 0);
    return;
  }
  v4u qf[NS];
  w.queries(qf);
  PackedState<DT, DF> st;
  st.clear();

  // Step j with block j's scores in s and K of block j + 1 and V of block j in
  // the tiles of these numbers; block j + 1's scores go to next.
  auto step = [&](int j, const v16f (&s)[TF], v16f (&next)[TF], auto ktile_tag, auto last_tag) {
    constexpr bool LAST = decltype(last_tag)::value;   // the wave's last block
    const char* kn = w.kt(decltype(ktile_tag)::value);
    const char* vc = w.vt(1 - decltype(ktile_tag)::value);
    v4u pf[BK / 16], vf[AHEAD + 1];
    const float at = st.at();
    float ea = 0.0f, eb = 0.0f;   // a pair of probabilities on its way
    auto form = [&](int pair) {
      ea = __builtin_amdgcn_exp2f(__builtin_fmaf(s[pair / 8][2 * (pair % 8)], p.c, -at));
      eb = __builtin_amdgcn_exp2f(__builtin_fmaf(s[pair / 8][2 * (pair % 8) + 1], p.c, -at));
    };
    auto keep = [&](int pair) {
      const uint32_t x = pack2<DT>(ea, eb);
      pf[pair / 4][pair % 4] = x;
      if constexpr (!W::kOnes) {
        st.l = add2<DT>(x, st.l);
        __asm__ volatile("" : "+v"(st.l));   // (not to be put off behind the products)
      }
    };
    // A quarter of the pairs while the first fragments are on their way, a
    // quarter with the first half of the values (which need them last).
    constexpr int PAIRS = 8 * TF, EARLY = PAIRS / 4, LATE = PAIRS / 4;
    if constexpr (LAST) {
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) vf[n] = w.v_of(vc, n);
#pragma unroll
      for (int i = 0; i < PAIRS; ++i) {
        form(i);
        keep(i);
      }
    } else {
      v4u kf[AHEAD + 1];
#pragma unroll
      for (int t = 0; t < TF; ++t) next[t] = v16f{};
#pragma unroll
      for (int n = 0; n < AHEAD; ++n) kf[n] = w.k_of(kn, n);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < EARLY; ++i) {
        if (i > 0) keep(i - 1);
        form(i);
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < QK; ++n) {
        if (n + AHEAD < QK) kf[(n + AHEAD) % (AHEAD + 1)] = w.k_of(kn, n + AHEAD);
        else vf[n + AHEAD - QK] = w.v_of(vc, n + AHEAD - QK);
        next[n % TF] = mfma32<DT>(kf[n % (AHEAD + 1)], qf[n / TF], next[n % TF]);
#pragma unroll
        for (int i = EARLY + (PAIRS - EARLY - LATE) * n / QK; i < EARLY + (PAIRS - EARLY - LATE) * (n + 1) / QK; ++i) {
          keep(i - 1);
          form(i);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    float mx = LAST ? 0.0f : next[0][0];
#pragma unroll
    for (int n = 0; n < PV; ++n) {
      if (n + AHEAD < PV) vf[(n + AHEAD) % (AHEAD + 1)] = w.v_of(vc, n + AHEAD);
      st.o[n % DF] = mfma32<DT>(vf[n % (AHEAD + 1)], pf[n / DF], st.o[n % DF]);
      if constexpr (!LAST) {
#pragma unroll
        for (int i = PAIRS - LATE + 2 * LATE * n / PV; i < PAIRS - LATE + 2 * LATE * (n + 1) / PV && i < PAIRS; ++i) {
          keep(i - 1);
          form(i);
          if (i == PAIRS - 1) keep(i);
        }
#pragma unroll
        for (int e = max(16 * TF * (2 * n - PV) / PV, 0); e < 16 * TF * (2 * n + 2 - PV) / PV; ++e)
          mx = fmaxf(mx, next[e / 16][e % 16]);
        __asm__ volatile("" : "+v"(mx));
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    if constexpr (!LAST) {
      if ((j + 2) * BK > w.wave_clean) {
        w.mask(j + 1, next);
        mx = W::largest(next);
      }
      st.follow(mx * p.c);
    }
  };
  auto sync = [&](int j) {
    __builtin_amdgcn_s_waitcnt(0x0F70);   // this wave's copies of K j + 1 and V j have landed,
    __syncthreads();                      // and everyone's; K j and V j - 1 have been read
    if (j + 2 < w.blocks) w.copy_k(j + 2, w.kt(j & 1));
    if (j + 1 < w.blocks) w.copy_v(j + 1, w.vt((j + 1) & 1));
  };
  using Tile0 = std::integral_constant<int, 0>;
  using Tile1 = std::integral_constant<int, 1>;
  if (w.blocks > 0) {
    w.copy_k(0, w.kt(0));
    if (w.blocks > 1) w.copy_k(1, w.kt(1));
    w.copy_v(0, w.vt(0));
    w.put_ones(threadIdx.x);
    __builtin_amdgcn_s_waitcnt(0x0F70);
    __syncthreads();
  }
  int j = 0;
  if (w.wave_blocks > 0) {
    v16f sa[TF], sb[TF];
#pragma unroll
    for (int t = 0; t < TF; ++t) sa[t] = v16f{};
#pragma unroll
    for (int n = 0; n < QK; ++n) sa[n % TF] = mfma32<DT>(w.k_of(w.kt(0), n), qf[n / TF], sa[n % TF]);
    if (BK > w.wave_clean) w.mask(0, sa);
    st.follow(W::largest(sa) * p.c);
    for (; j + 2 < w.wave_blocks; j += 2) {
      sync(j);
      step(j, sa, sb, Tile1{}, std::false_type{});
      sync(j + 1);
      step(j + 1, sb, sa, Tile0{}, std::false_type{});
    }
    if (j + 2 == w.wave_blocks) {
      sync(j);
      step(j, sa, sb, Tile1{}, std::false_type{});
      sync(++j);
      step(j, sb, sa, Tile0{}, std::true_type{});
    } else {
      sync(j);
      step(j, sa, sb, Tile1{}, std::true_type{});
    }
    ++j;
  }
  for (; j < w.blocks; ++j) sync(j);   // the rest is the other waves'

  if constexpr (CAUSAL) {
    // Finite sums times 0 are 0: only where they are not can a masked value have come in.
    float zs[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int f = 0; f < DF; ++f)
#pragma unroll
      for (int x = 0; x < 16; ++x) zs[x % 4] = __builtin_fmaf(st.o[f][x], 0.0f, zs[x % 4]);
    const float z = (zs[0] + zs[1]) + (zs[2] + zs[3]);
    w.store(st.o, st.ref, w.sum_of(st.o, st.l));
    const bool odd = __builtin_amdgcn_ballot_w64(z != 0.0f) != 0;
    __syncthreads();   // the tiles have been read
    int* again = reinterpret_cast<int*>(tiles);
    if (w.lane == 0) again[w.wave] = odd;
    __syncthreads();
    if (again[0] | again[1] | again[2] | again[3]) packed_careful<DT, DP, SPLIT>(p, tiles);
  } else {
    w.store(st.o, st.ref, w.sum_of(st.o, st.l));
  }
}

// The ranges' sums of a row and head, joined in order, four channels a lane.
template <int DT, int DP>
__global__ __launch_bounds__(256) void packed_join_kernel(PackedParams p) {
  constexpr int PITCH = (DP + 31) / 32 * 32, LANES = PITCH == 96 ? 32 : PITCH / 4;
  const int heads = p.group * p.kv_heads;
  const int64_t item = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LANES;
  const int d = 4 * (threadIdx.x % LANES);
  const int64_t row = item / heads;
  const int head = (int)(item - row * heads);
  if (row >= p.rows || row >= scalar_int(p.starts, p.sequences) || d >= p.dim) return;
  float ref = -INFINITY, sum = 0.0f;
  v4f y = {0.0f, 0.0f, 0.0f, 0.0f};
  constexpr int BATCH = 8;
  for (int s = 0; s < p.splits; s += BATCH) {
    float2 ml[BATCH];
    v4f x[BATCH];
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      const int64_t at = ((int64_t)min(s + i, p.splits - 1) * p.rows + row) * heads + head;
      ml[i] = *reinterpret_cast<const float2*>(p.part_ml + 2 * at);
      x[i] = *reinterpret_cast<const v4f*>(p.part + at * PITCH + d);
    }
    float to = ref;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) to = fmaxf(to, ml[i].x);
    const float base = to == -INFINITY ? 0.0f : to, fade = __builtin_amdgcn_exp2f(ref - base);
    ref = to;
    sum = sum * fade;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = y[e] * fade;
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
      if (s + i >= p.splits) continue;
      const float f = __builtin_amdgcn_exp2f(ml[i].x - base);
      sum = __builtin_fmaf(ml[i].y, f, sum);
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = __builtin_fmaf(x[i][e], f, y[e]);
    }
  }
  const float rcp = ref == -INFINITY ? 0.0f : 1.0f / sum;
  *reinterpret_cast<uint2*>(p.out + row * p.o_row + head * p.o_head + 2 * d) =
      make_uint2(pack2<DT>(y[0] * rcp, y[1] * rcp), pack2<DT>(y[2] * rcp, y[3] * rcp));
}

static int packed_dp(int dim) { return dim <= 64 ? 64 : dim <= 80 ? 80 : dim <= 96 ? 96 : dim <= 128 ? 128 : 256; }
static int packed_pitch(int dim) { return (packed_dp(dim) + 31) / 32 * 32; }

// Ranges of a tile's keys. A step along the keys takes a wave about 1 us however
// few workgroups there are. Where the tiles of all heads are fewer than half of
// what the GPU holds, several workgroups take a tile's keys: four blocks each or
// more (one row behind 8000 keys 130 us alone, 16.7 so, 19.5 by two blocks), or two
// for up to eight workgroups, which the second kernel joins in one go (one behind
// 1000 keys 11.4 -> 9.5, 23 of 28 heads behind 587 16.1 -> 12.5). That is, if the steps
// saved are more than the second kernel (5 steps; 23 rows behind 300 keys save four
// and lose, 11.5 -> 12.2) and the sums' way through memory (3.6 MB a step): 512
// rows of a prompt 17 -> 29. (The halves of a workgroup of eight waves sharing the
// keys and meeting in LDS: 353 rows 13.0 -> 14.7.)
static int packed_splits(int64_t rows, int64_t keys, int64_t sequences, int64_t heads, int64_t kv_heads, int dim) {
  if (rows <= 0 || rows >= (1 << 27) || keys <= 0 || keys >= (1 << 27) || sequences <= 0 || sequences >= (1 << 20)) return 1;
  if (heads <= 0 || heads > 65536 || kv_heads <= 0 || heads % kv_heads || dim < 8 || dim > 256 || dim % 8) return 1;
  const int64_t filled = std::min(rows, sequences), tiles = (rows * (heads / kv_heads) + (kPackQ - 1) * filled) / kPackQ * kv_heads;
  const int64_t slots = (dim > 128 ? 1 : 2) * current_device_cus(), block = dim > 128 ? 32 : 64;
  const int64_t steps = (keys / sequences + block - 1) / block, splits = std::min(slots / tiles, std::max(steps / 4, std::min<int64_t>(steps / 2, 8)));
  return splits >= 2 && steps - steps / splits >= 5 + rows * heads * splits * packed_pitch(dim) * 8 / 3600000 ? (int)splits : 1;
}

template <int DT, int DP, bool CAUSAL>
static int launch_packed(const PackedParams& p, int64_t grid, hipStream_t s) {
  const dim3 g((unsigned)(grid * p.splits)), t(64 * kPackWaves);
  if (p.splits == 1) {
    hipLaunchKernelGGL((packed_attention_kernel<DT, DP, CAUSAL, false>), g, t, 0, s, p);
  } else {
    hipLaunchKernelGGL((packed_attention_kernel<DT, DP, CAUSAL, true>), g, t, 0, s, p);
    const int64_t per = DP <= 64 ? 16 : DP <= 128 ? 8 : 4, items = (int64_t)p.rows * p.group * p.kv_heads;
    hipLaunchKernelGGL((packed_join_kernel<DT, DP>), dim3((unsigned)((items + per - 1) / per)), dim3(256), 0, s, p);
  }
  return launch_status("w8a8_packed_attention");
}

template <int DT, int DP>
static int launch_packed(const PackedParams& p, bool causal, int64_t grid, hipStream_t s) {
  return causal ? launch_packed<DT, DP, true>(p, grid, s) : launch_packed<DT, DP, false>(p, grid, s);
}

template <int DT>
static int launch_packed_dim(const PackedParams& p, bool causal, int64_t grid, hipStream_t s) {
  switch (packed_dp(p.dim)) {
    case 64: return launch_packed<DT, 64>(p, causal, grid, s);
    case 80: return launch_packed<DT, 80>(p, causal, grid, s);
    case 96: return launch_packed<DT, 96>(p, causal, grid, s);
    case 128: return launch_packed<DT, 128>(p, causal, grid, s);
    default: return launch_packed<DT, 256>(p, causal, grid, s);
  }
}

}  // namespace w8a8

extern "C" int64_t w8a8_packed_attention_workspace_size(int64_t rows, int64_t keys, int64_t sequences, int64_t heads,
                                                        int64_t kv_heads, int32_t dim) {
  using namespace w8a8;
  const int splits = packed_splits(rows, keys, sequences, heads, kv_heads, dim);
  return splits == 1 ? 0 : splits * rows * heads * (packed_pitch(dim) + 2) * (int64_t)sizeof(float);
}

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
  W8A8_REQUIRE(a->sm_scale > 0.0f && std::isfinite(a->sm_scale * kLog2eF), "%s: sm_scale must be positive and finite", who);
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
  const RowsOf om = rows_memory(a->out, a->rows, a->heads, a->dim, a->out_strides);
  W8A8_REQUIRE(apart(om, rows_memory(a->q, a->rows, a->heads, a->dim, a->q_strides)) &&
                   (a->keys == 0 || (apart(om, rows_memory(a->k, a->keys, a->kv_heads, a->dim, a->k_strides)) &&
                                     apart(om, rows_memory(a->v, a->keys, a->kv_heads, a->dim, a->v_strides)))),
               "%s: out overlaps an input", who);
  const int splits = packed_splits(a->rows, a->keys, a->sequences, a->heads, a->kv_heads, a->dim);
  const int64_t need = w8a8_packed_attention_workspace_size(a->rows, a->keys, a->sequences, a->heads, a->kv_heads, a->dim);
  W8A8_REQUIRE(need == 0 || (a->workspace && aligned16(a->workspace) && a->workspace_bytes >= need),
               "%s: workspace of %lld bytes needed", who, (long long)need);
  W8A8_REQUIRE(apart_from(om, a->starts, 4 * (a->sequences + 1)) && apart_from(om, a->k_starts, 4 * (a->sequences + 1)) &&
                   apart_from(om, a->workspace, need),
               "%s: starts or workspace lie in the output", who);
  const int64_t packed = a->rows * (a->heads / a->kv_heads), grid = (packed / kPackQ + a->sequences + 1) * a->kv_heads;
  W8A8_REQUIRE(packed < (1ll << 31) - kPackQ && grid * splits < (1 << 24), "%s: too many rows, sequences and heads for one launch", who);   // (2^32 work-items)
  const PackedParams p{reinterpret_cast<const char*>(a->q), reinterpret_cast<const char*>(a->k),
                       reinterpret_cast<const char*>(a->v), reinterpret_cast<char*>(a->out),
                       2 * a->q_strides[0], 2 * a->q_strides[1], 2 * a->k_strides[1], 2 * a->v_strides[1],
                       2 * a->out_strides[0], 2 * a->out_strides[1],
                       (uint32_t)(2 * a->k_strides[0]), (uint32_t)(2 * a->v_strides[0]),
                       (int)a->rows, (int)a->keys, (int)a->sequences, a->heads / a->kv_heads, a->kv_heads, a->dim,
                       ~0ull / (uint64_t)(a->heads / a->kv_heads) + 1,
                       a->starts, a->k_starts, a->sm_scale * kLog2eF, a->fill, splits,
                       reinterpret_cast<float*>(a->workspace),
                       reinterpret_cast<float*>(a->workspace) + splits * a->rows * a->heads * packed_pitch(a->dim)};
  hipStream_t s = reinterpret_cast<hipStream_t>(a->stream);
  return a->dtype == W8A8_F16 ? launch_packed_dim<kF16>(p, a->causal != 0, grid, s)
                              : launch_packed_dim<kBF16>(p, a->causal != 0, grid, s);
}
