// Projections with 4-bit weights and group scales on 16-bit activations.
//
//   y[m][n] = sum_g s[g][n] * sum_{k in g} (c[n][k] - z[g][n]) x[m][k]
//
// A code goes into the top bits of the mantissa of 16 in the activations' type
// (16 + c, exact in both types): one shift and one and-or make two weights, and
// the type's own MFMA takes them. Their group sum is the codes' plus 16 times
// the group's sum of x, which an MFMA with a row of ones gives, so that
//   sum (c - z) x = sum (16 + c) x - (16 + z) sum x
// in fp32. The error is fp32's relative to (16 + z) sum |x|, whatever the difference
// leaves of it: the two sums are some five times the result at the median of normal
// inputs and random codes (32 times at the ninth decile), 45 and 233 times with inputs
// of one sign. Times the scale that stays below half a 16-bit step of results of
// ordinary size, not of those that cancel out. (fp16 tiles take z off the
// weights and have no such sums.) Scales apply to a group's sum, in fp32.
//
// A 16-bit operand fragment of the 16 x 16 x 32 MFMA is eight inputs a lane,
// one word of codes; a lane's inputs of a block of GB (a group, or 128 inputs of
// a longer one) are a quarter of it in a row, so codes and activations are
// loaded as they lie, GB / 32 words and as many 16-byte runs a lane.
#include "w8a8_device.h"
#include "w8a8_host.h"

#include <algorithm>
#include <type_traits>

namespace w8a8 {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));

struct W4Params {
  const void* x;
  int64_t ldx;
  const uint32_t* codes;
  int64_t ldw;
  const uint16_t* scales;
  const uint8_t* zeros;
  int64_t m, n, k;
  int group;
  const uint16_t* bias;
  const uint16_t* residual;
  int64_t ldr;
  uint16_t* out;
  int64_t ldo;
  bool quads;   // scales, zeros and outputs of four neighbouring rows are read and written as one
};

// The eight weights of a word as 16 + c, in the order of their inputs: a shift
// and a v_and_or_b32 for two, which takes one constant from a vector register
// and one from a scalar one (both out of the compiler's sight, which would make
// it two instructions with literals).
template <int DT>
struct Unpack {
  uint32_t mask, one;
  __device__ __forceinline__ Unpack() {
    mask = DT == kF16 ? 0x03c003c0u : 0x00780078u;
    one = DT == kF16 ? 0x4c004c00u : 0x41804180u;
    __asm__("" : "+v"(mask));
    __asm__("" : "+s"(one));
  }
  __device__ __forceinline__ uint32_t pick(uint32_t w) const {
    uint32_t r;
    __asm__("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(w), "v"(mask), "s"(one));
    return r;
  }
  __device__ __forceinline__ v4u operator()(uint32_t w) const {
    if constexpr (DT == kF16) return v4u{pick(w << 6), pick(w << 2), pick(w >> 2), pick(w >> 6)};
    else return v4u{pick(w << 3), pick(w >> 1), pick(w >> 5), pick(w >> 9)};
  }
};

// Eight fp16 less one (in both halves of z), exact here.
__device__ __forceinline__ v4u less(v4u a, uint32_t z) {
  const v2h y = __builtin_bit_cast(v2h, z);
  v4u r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t e = a[i];
    r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(v2h, e) - y);
  }
  return r;
}

template <int DT>
__device__ __forceinline__ v4f mfma(v4u a, v4u b, v4f c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ float wide(uint16_t u) { return DT == kF16 ? h2f(u) : bf2f(u); }
template <int DT>
__device__ __forceinline__ uint16_t slim(float f) { return DT == kF16 ? f2h(f) : f2bf(f); }

// The epilogue of four neighbouring outputs of row m: y (and up, where gated)
// before the bias.
template <int DT, bool GATED>
__device__ __forceinline__ void finish4(const W4Params& p, int64_t m, int64_t n, int64_t width, v4f y, v4f up) {
  uint16_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t c = min(n + i, width - 1);
    float v = y[i];
    if (p.bias) v = v + wide<DT>(p.bias[c]);
    if constexpr (GATED) {
      const float u = p.bias ? up[i] + wide<DT>(p.bias[width + c]) : up[i];
      v = swiglu(v, u);
    }
    if (p.residual) v = v + wide<DT>(p.residual[m * p.ldr + c]);
    o[i] = slim<DT>(v);
  }
  uint16_t* dst = p.out + m * p.ldo + n;
  if (p.quads) {
    if (n < width)
      *reinterpret_cast<uint2*>(dst) = make_uint2(o[0] | ((uint32_t)o[1] << 16), o[2] | ((uint32_t)o[3] << 16));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (n + i < width) dst[i] = o[i];
  }
}

// Up to eight rows of x: a workgroup of W waves takes 16 NT weight rows (gated: half
// of them gate, half the same rows of up); its waves share out the blocks of k and
// add their sums in LDS, in the order of the waves. A wave's next `AHEAD` blocks
// are under way while one is multiplied: the weights' bytes are the call's time.
// The MFMA's first operand is the weights here, so that a lane's four results are
// neighbouring outputs of one row.
template <int DT, int GB, int NT, int W, bool GATED, int AHEAD>
__global__ __launch_bounds__(64 * W)
void linear_w4_kernel(W4Params p) {
  constexpr int S = GB / 32;   // MFMA steps of a block, and a lane's words of it
  constexpr int TILES = GATED ? NT / 2 : NT;   // tiles of outputs
  __shared__ v4f part[W][NT][64];
  const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t width = GATED ? p.n / 2 : p.n;
  const int64_t n0 = (int64_t)blockIdx.x * (16 * TILES);
  const uint32_t* wrow[NT];
  int64_t nd[NT];      // the lane's first row of the tile's result
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t base = n0 + 16 * (t % TILES), shift = t >= TILES ? width : 0;
    wrow[t] = p.codes + (shift + min(base + r, width - 1)) * p.ldw + g * S;
    nd[t] = shift + base + 4 * g;
  }
  const uint16_t* const xrow =
      reinterpret_cast<const uint16_t*>(p.x) + min((int64_t)r, p.m - 1) * p.ldx + g * (GB / 4);
  const v4u ones = DT == kF16 ? v4u{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u}
                              : v4u{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  const Unpack<DT> unpack;
  const int blocks = (int)(p.k / GB), per_group = p.group / GB;
  struct Block {
    uint32_t w[NT][S];
    v4u x[S];
    uint32_t s[NT][2], z[NT];   // four scales, four zeros
  };
  // The blocks go to the waves in pairs, neighbours to one wave in turn, so that it
  // reads whole 128-byte lines of codes (14336 x 4096, one row: 12.9 -> 10.7 us).
  auto at_of = [](int i) {
    const int turn = i / W, w = i - turn * W;
    return (turn >> 1) * (2 * W) + 2 * w + (turn & 1);
  };
  auto load = [&](int b, Block& o) {
    b = min(at_of(b), blocks - 1);   // (past the last one: loaded and left)
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      const uint32_t* at = wrow[t] + (int64_t)b * (GB / 8);
      if constexpr (S == 4) *reinterpret_cast<v4u*>(&o.w[t][0]) = *reinterpret_cast<const v4u*>(at);
      else if constexpr (S == 2) *reinterpret_cast<uint2*>(&o.w[t][0]) = *reinterpret_cast<const uint2*>(at);
      else o.w[t][0] = *at;
    }
#pragma unroll
    for (int j = 0; j < S; ++j) o.x[j] = *reinterpret_cast<const v4u*>(xrow + (int64_t)b * GB + 8 * j);
    const int64_t grow = (int64_t)(b / per_group) * p.n;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      // (Past the last row its values again.)
      if (p.quads) {
        const int64_t at = grow + min(nd[t], p.n - 4);
        *reinterpret_cast<uint2*>(&o.s[t][0]) = *reinterpret_cast<const uint2*>(p.scales + at);
        o.z[t] = p.zeros ? *reinterpret_cast<const uint32_t*>(p.zeros + at) : 0x08080808u;
      } else {
        uint32_t z = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t at = grow + min(nd[t] + i, p.n - 1);
          o.s[t][i >> 1] = i & 1 ? o.s[t][i >> 1] | ((uint32_t)p.scales[at] << 16) : p.scales[at];
          z |= (uint32_t)(p.zeros ? p.zeros[at] : 8) << (8 * i);
        }
        o.z[t] = z;
      }
    }
  };
  v4f tot[NT] = {};
  Block q[AHEAD + 1];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) load(wave + i * W, q[i]);
  const int turns = (blocks + 2 * W - 1) / (2 * W) * 2;
  for (int turn = 0; turn < turns; turn += AHEAD + 1) {
#pragma unroll
    for (int i = 0; i <= AHEAD; ++i) {
      const Block& f = q[i];
      load(wave + (turn + i + AHEAD) * W, q[(i + AHEAD) % (AHEAD + 1)]);
      if (turn + i >= turns || at_of(wave + (turn + i) * W) >= blocks) continue;
      v4f sum = {}, acc[NT] = {};
#pragma unroll
      for (int j = 0; j < S; ++j) {
        sum = mfma<DT>(ones, f.x[j], sum);
#pragma unroll
        for (int t = 0; t < NT; ++t) acc[t] = mfma<DT>(unpack(f.w[t][j]), f.x[j], acc[t]);
      }
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float s = wide<DT>((uint16_t)(f.s[t][e >> 1] >> (16 * (e & 1))));
          const float z = (float)((f.z[t] >> (8 * e)) & 0xffu) + 16.0f;
          tot[t][e] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[e], acc[t][e]), tot[t][e]);
        }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t) part[wave][t][lane] = tot[t];
  __syncthreads();
  for (int t = wave; t < TILES; t += W) {
    v4f y = part[0][t][lane], up = {};
    for (int v = 1; v < W; ++v) y = y + part[v][t][lane];
    if constexpr (GATED) {
      up = part[0][TILES + t][lane];
      for (int v = 1; v < W; ++v) up = up + part[v][TILES + t][lane];
    }
    if (r < p.m) finish4<DT, GATED>(p, r, n0 + 16 * t + 4 * g, width, y, up);
  }
}

// Sum of a value over the aligned N lanes (4, 8 or 16) of a row of 16, in all of them.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  return v + __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(v), CTRL, 0xf, 0xf, true));
}
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  v = add_dpp<0xb1>(v);                       // xor 1 within a quad
  v = add_dpp<0x4e>(v);                       // xor 2
  if constexpr (N >= 8) v = add_dpp<0x141>(v);   // the other quad of eight
  if constexpr (N >= 16) v = add_dpp<0x140>(v);  // the other eight of sixteen
  return v;
}

// The sums of x over blocks of GB inputs, as three bf16 that add up to the fp32
// sum: sums[block][m] = (hi, mid, lo, 0), rows padded to a multiple of 128. A
// thread takes a 16-byte run of x, and another a grid on.
constexpr int64_t kSumsBlocks = 1 << 20;
template <int DT, int GB>
__global__ __launch_bounds__(256)
void w4_sums_kernel(W4Params p, uint2* sums) {
  const int runs = (int)(p.k / 8);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < p.m * runs; i += (int64_t)gridDim.x * 256) {
    const int64_t m = i / runs;   // (whole groups of lanes: a row is whole blocks)
    const int run = (int)(i - m * runs);
    const v4u x = *reinterpret_cast<const v4u*>(reinterpret_cast<const uint16_t*>(p.x) + m * p.ldx + 8 * run);
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) s = s + (wide<DT>((uint16_t)x[j]) + wide<DT>((uint16_t)(x[j] >> 16)));
    s = lanes_sum<GB / 8>(s);
    if (run % (GB / 8)) continue;
    const uint16_t hi = f2bf(s);
    const float s1 = s - bf2f(hi);
    const uint16_t mid = f2bf(s1);
    const uint16_t lo = f2bf(s1 - bf2f(mid));
    sums[(int64_t)(run / (GB / 8)) * ((p.m + 127) & ~(int64_t)127) + m] = make_uint2(hi | ((uint32_t)mid << 16), lo);
  }
}

typedef float v16f __attribute__((ext_vector_type(16)));

template <int DT>
__device__ __forceinline__ v16f mfma32(v4u a, v4u b, v16f c) {
  if constexpr (DT == kF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(v8h, a), __builtin_bit_cast(v8h, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(v8b, a), __builtin_bit_cast(v8b, b), c, 0, 0, 0);
}

// -(16 + z) sum x into fresh accumulators: the three bf16 of a row's sum (from
// lanes 0-31, inputs 0-2) times the zero's column (lanes 32-63 hold zeros there).
__device__ __forceinline__ v16f mfma_zero(uint2 sum, uint2 z) {
  typedef short v4s __attribute__((ext_vector_type(4)));
  return __builtin_amdgcn_mfma_f32_32x32x8bf16_1k(__builtin_bit_cast(v4s, sum), __builtin_bit_cast(v4s, z), v16f{}, 0, 0, 0);
}

// A uniform base for dma(), and SIZE bytes a lane from `off` bytes behind it to LDS:
// lane i's at l + 16 i, or a word each at l + 4 i (shorter values zero-extended).
// (The global form counts as an LDS access with the compiler, which then waits for
// every LDS read in flight before the first one's use.)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t dma_base(const void* p) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0, -1, 0x00027000);
}
template <int SIZE>
__device__ __forceinline__ void dma(__amdgpu_buffer_rsrc_t base, uint32_t off, char* l) {
  auto* to = (__attribute__((address_space(3))) void*)l;
  if constexpr (SIZE == 16) __builtin_amdgcn_raw_ptr_buffer_load_lds(base, to, 16, (int)off, 0, 0, 0);
  else if constexpr (SIZE == 4) __builtin_amdgcn_raw_ptr_buffer_load_lds(base, to, 4, (int)off, 0, 0, 0);
  else if constexpr (SIZE == 2) __builtin_amdgcn_raw_ptr_buffer_load_lds(base, to, 2, (int)off, 0, 0, 0);
  else __builtin_amdgcn_raw_ptr_buffer_load_lds(base, to, 1, (int)off, 0, 0, 0);
}

// A tile's outputs, or (part: the lane's column of the range's tile, rows `width`
// apart) its sums over a range of k.
template <int DT, int U, bool GATED>
__device__ __forceinline__ void store_tile(const W4Params& p, const v16f (&tot)[U], float* part, int width, int64_t m0,
                                           int64_t n0, int mrows, int nrows, int64_t wr, int ncol, int c, int h) {
  const int64_t n = n0 + ncol;
  if (part) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int m = 32 * u + 8 * (i >> 2) + 4 * h + (i & 3);
        if (m < mrows) part[m * width] = tot[u][i];
      }
    return;
  }
  const float bias = p.bias ? wide<DT>(p.bias[wr]) : 0.0f;
  const int64_t nc = n0 + min(ncol, nrows - 1);
#pragma unroll
  for (int u = 0; u < U; ++u) {
    // (Sixteen loads at once, of the last row and column where the tile ends.)
    uint16_t r[16];
    if (p.residual) {
#pragma unroll
      for (int i = 0; i < 16; ++i)
        r[i] = p.residual[(m0 + min(32 * u + 8 * (i >> 2) + 4 * h + (i & 3), mrows - 1)) * p.ldr + nc];
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int m = 32 * u + 8 * (i >> 2) + 4 * h + (i & 3);
      float v = tot[u][i] + bias;
      if constexpr (GATED) v = swiglu(v, __shfl_xor(v, 16, 64));
      if (p.residual) v = v + wide<DT>(r[i]);
      if (m < mrows && ncol < nrows && (!GATED || c < 16)) p.out[(m0 + m) * p.ldo + n] = slim<DT>(v);
    }
  }
}

// More than eight rows: a workgroup of W waves takes 32 U rows of x and 32 W weight
// rows (gated: 16 W of gate and the same of up); each wave takes all of x's rows
// and 32 of the weight's (gated: 16 of each), so that every code is unpacked once
// a workgroup, and the waves of a SIMD do each other's unpacking and scaling in
// the shadow of their MFMAs. The 32 x 32 x 16 MFMA's first operand is x, its second
// the weights, a word of codes a lane: a lane's column is one weight row, whose
// scale it holds.
//
// Everything comes by DMA: x (16-byte run c of row r at run c ^ (r & 15)), codes,
// scales and zeros (sub-word loads, a word each in LDS), into a ring of stages of
// 128 inputs each, RING - 1 ahead, so that a counted wait leaves the later stages'
// loads in flight (a load into registers behind a DMA waits for all of them). A
// step's work is laid out product by product (below), since the compiler's own
// order reads each operand right before its use and scales and unpacks between the
// chains of MFMAs. 2048 x 14336 x 4096: bf16 in groups of 64 278 to 291 us (381 in
// the compiler's order; 827 to 865 TFLOP/s), fp16 in groups of 128 254 (294). What
// bounds it: VALU and MFMA add up to the time (bf16 265 and 287 of 494 thousand cycles
// a SIMD, the gated fp16 call below 101 and 96 of 196: 7.4 and 8.4 VALU instructions a
// product), so the two waves of a SIMD hardly overlap; LDS has cycles to spare (144
// and 55 thousand a CU).
//
// fp16 takes the zeros off its weights (packed subtraction, exact). bf16 has no
// such instruction. Where the rows are many (U = 4) an MFMA puts -(16 + z) sum x
// into the accumulators before a block's products, with the sum in three bf16
// (exact) as three inputs, loaded one step ahead; where they are few a second MFMA
// beside each product sums x, which costs less than the launch that sums it
// beforehand.
//
// The tiles past the last whole round of the GPU (all of them, where they are few)
// split the steps of k over `splits` workgroups each, whose sums
// linear_w4_join_kernel adds in order.
template <int DT, int GB, int U, int W>
struct W4Stage {
  static constexpr bool kOnes = DT == kBF16 && U < 4, kPre = DT == kBF16 && U == 4;
  static constexpr int NB = 128 / GB, PAIRS = (NB + 1) / 2;
  static constexpr int kRing = U > 1 && GB == 32 ? 2 : 3;        // (what 160 KB hold; two workgroups a CU below U = 4)
  static constexpr int kX = U * 32 * 256, kCodes = W * 2048, kMeta = W * 512 * PAIRS, kBytes = kX + kCodes + kMeta;
  static constexpr int kXDma = 8 * U / W, kDma = kXDma + 2 + 2 * PAIRS;   // instructions of a wave
  static constexpr int kSums = kPre ? NB * 1024 : 0;
  static constexpr int kLds = kRing * kBytes + 2 * kSums;
};

template <int N>
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0f70); }

// Workgroup barrier without a fence, which would wait for the DMA in flight: the
// caller waits for what it needs, and every LDS read before it has been used.
__device__ __forceinline__ void block_barrier() {
  __asm__ volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __asm__ volatile("" ::: "memory");
}

template <int DT, int GB, int U, int W, bool GATED>
__global__ __launch_bounds__(64 * W, 2)
void linear_w4_tiles_kernel(W4Params p, const uint2* sums, float* parts, int mtiles, int whole, int rest, int splits) {
  using Stage = W4Stage<DT, GB, U, W>;
  constexpr int S = GB / 16, NB = Stage::NB, BN = GATED ? 16 * W : 32 * W, RING = Stage::kRing;
  constexpr int DEEP = 4;   // (6 and 8 the same within 1 %)
  __shared__ __attribute__((aligned(16))) char lds[Stage::kLds];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t width = GATED ? p.n / 2 : p.n;
  // Workgroups go to the eight XCDs in turn: each XCD takes a run of the whole tiles
  // (the row tiles of a few weight tiles at a time), then one of the rest's ranges.
  const int head = (whole + 7) & ~7;
  const bool split_up = (int)blockIdx.x >= head;
  const int at_block = split_up ? (int)blockIdx.x - head : (int)blockIdx.x, items = split_up ? rest * splits : whole;
  const int per = (items + 7) / 8, item = (at_block & 7) * per + (at_block >> 3);
  if (item >= items || (at_block >> 3) >= per) return;
  const int left = split_up ? item / splits : 0, split = split_up ? item - left * splits : 0;
  const int tile = split_up ? whole + left : item, ranges = split_up ? splits : 1;
  const int64_t m0 = (int64_t)(tile % mtiles) * (32 * U), n0 = (int64_t)(tile / mtiles) * BN;
  const int mrows = (int)min((int64_t)(32 * U), p.m - m0), nrows = (int)min((int64_t)BN, width - n0);
  // The tile's column of the wave's column col (0..31: gated, 16 of gate and the same of up).
  auto column = [&](int col) { return GATED ? 16 * wave + (col & 15) : 32 * wave + col; };
  const int ncol = column(c), nclamped = min(ncol, nrows - 1);
  const int64_t wr = (GATED && c >= 16 ? width : 0) + n0 + nclamped;
  const auto xbase = dma_base(reinterpret_cast<const uint16_t*>(p.x) + m0 * p.ldx);
  uint32_t xoff[Stage::kXDma];
#pragma unroll
  for (int i = 0; i < Stage::kXDma; ++i)
    xoff[i] = (uint32_t)min(4 * (Stage::kXDma * wave + i) + (lane >> 4), mrows - 1) * (uint32_t)(p.ldx * 2);
  // A wave brings its own codes: instruction i rows 16 i .. 16 i + 15, four 16-byte
  // runs a row, run q at q ^ (row >> 2 & 3).
  __amdgpu_buffer_rsrc_t cbase[2];
  uint32_t coff[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    cbase[i] = dma_base(p.codes + ((GATED && i ? width : 0) + n0) * p.ldw);
    coff[i] = (uint32_t)min(column(16 * i + (lane >> 2)), nrows - 1) * (uint32_t)(p.ldw * 4);
  }
  const int crun = 16 * ((lane & 3) ^ ((lane >> 4) & 3));
  const uint32_t roff = (uint32_t)wr;
  // (Without zeros a byte of the scales is read and left.)
  const uint8_t* const zrow = p.zeros ? p.zeros : reinterpret_cast<const uint8_t*>(p.scales);
  const int all = (int)((p.k + 127) / 128), blocks = (int)(p.k / GB), kbytes = (int)(p.k / 2);
  const int first = (int)((int64_t)all * split / ranges), last = (int)((int64_t)all * (split + 1) / ranges);
  const int per_group = p.group / GB;
  const int64_t mpad = (p.m + 127) & ~(int64_t)127;

  // Piece i of a step's loads. A step past the last is the last again; past the end
  // of k the last runs and codes again, whose blocks' scales are taken as zero.
  auto load = [&](int step, char* to, int i) {
    step = min(step, last - 1);
    constexpr int X = Stage::kXDma;
    if (i < X) {
      const int row = 4 * (X * wave + i), run = (lane & 15) ^ ((row + (lane >> 4)) & 15);
      dma<16>(xbase, xoff[i] + (uint32_t)min(step * 256 + run * 16, (int)p.k * 2 - 16), to + row * 256);
    } else if (i < X + 2) {
      dma<16>(cbase[i - X], coff[i - X] + (uint32_t)min(step * 64 + crun, kbytes - 16),
              to + Stage::kX + 2048 * wave + 1024 * (i - X));
    } else {
      const int j = (i - X - 2) / 2;
      // (Two neighbouring blocks of less than 128 inputs, half the lanes each.)
      const int one = min(step * NB + 2 * j, blocks - 1), two = min(step * NB + 2 * j + 1, blocks - 1);
      const int64_t group = NB > 1 ? one : one / per_group;   // (blocks are groups below 128 inputs)
      const uint32_t at = roff + (NB > 1 && h && two != one ? (uint32_t)p.n : 0);
      char* const meta = to + Stage::kX + Stage::kCodes + 512 * (Stage::PAIRS * wave + j);
      if ((i - X) & 1) dma<1>(dma_base(zrow + group * p.n), at, meta + 256);
      else dma<2>(dma_base(p.scales + group * p.n), 2 * at, meta);
    }
  };
  auto load_sums = [&](int step, char* to) {
    // (4 bytes a lane; the waves that are left load the same again. Rows past the
    // last are never stored.)
    if constexpr (Stage::kPre) {
#pragma unroll
      for (int i = 0; i < (NB + 1) / 2; ++i) {
        const int part = (8 * i + wave) & (4 * NB - 1);
        const int64_t block = min(min(step, last - 1) * NB + part / 4, blocks - 1);
        dma<4>(dma_base(sums + block * mpad + m0), 256 * (part & 3) + 4 * lane, to + 256 * part);
      }
    }
  };

  const uint32_t zero_mask = p.zeros ? 0xffu : 0u, zero_else = p.zeros ? 0u : 8u, half_mask = h ? 0u : ~0u;
  const Unpack<DT> unpack;
  // A block's codes, scale and zero as they lie in LDS, and its weights, scale and
  // zero (fp16: to take off the weights; bf16: the correction's column, or factor)
  // ready for the MFMAs.
  struct Raw {
    uint32_t w[S], scale, zero;
  };
  struct Ready {
    v4u w[S];
    float scale;
    uint32_t zero;
  };
  auto fetch = [&](const char* at, int b, Raw& o) {
    const char* const cw = at + Stage::kX + 2048 * wave + 64 * c;
    if constexpr (S == 8) {
      *reinterpret_cast<v4u*>(&o.w[0]) = *reinterpret_cast<const v4u*>(cw + 16 * ((2 * h) ^ ((c >> 2) & 3)));
      *reinterpret_cast<v4u*>(&o.w[4]) = *reinterpret_cast<const v4u*>(cw + 16 * ((2 * h + 1) ^ ((c >> 2) & 3)));
    } else if constexpr (S == 4) {
      *reinterpret_cast<v4u*>(&o.w[0]) = *reinterpret_cast<const v4u*>(cw + 16 * ((2 * b + h) ^ ((c >> 2) & 3)));
    } else {
      *reinterpret_cast<v2u*>(&o.w[0]) = *reinterpret_cast<const v2u*>(cw + 16 * (b ^ ((c >> 2) & 3)) + 8 * h);
    }
    const char* const meta = at + Stage::kX + Stage::kCodes + 512 * (Stage::PAIRS * wave + b / 2) + 4 * (32 * (b & 1) + c);
    o.scale = *reinterpret_cast<const uint32_t*>(meta);
    o.zero = *reinterpret_cast<const uint32_t*>(meta + 256);
  };
  auto open = [&](int step, int b, const Raw& r, Ready& o) {
    // (Selects by arithmetic: behind a branch the compiler waits for every load.)
    o.scale = wide<DT>((uint16_t)r.scale) * (NB == 1 || step * NB + b < blocks ? 1.0f : 0.0f);
    const float z = 16.0f + (float)((r.zero & zero_mask) | zero_else);
    if constexpr (Stage::kOnes) o.zero = __float_as_uint(-z);
    else o.zero = DT == kF16 ? (uint32_t)f2h(z) * 0x10001u
                             : ((__float_as_uint(-z) >> 16) * 0x10001u) & half_mask;   // (exact: a small integer)
  };
  auto weights = [&](const Raw& r, int j, Ready& o) {
    o.w[j] = unpack(r.w[j]);
    if constexpr (DT == kF16) o.w[j] = less(o.w[j], o.zero);
  };

  constexpr int P = U * S, N = NB * P;        // products of a block and a step
  constexpr bool ODD = NB * U == 1;           // one chain a step: accumulators change places between steps
  v16f tot[U] = {}, acc[2] = {}, ones[2] = {};
  float carry = 0.0f, carry_zero = 0.0f;      // of the last chain, whose sums are still to be scaled
  int at = 0, to = (RING - 1) * Stage::kBytes, sums_of = RING * Stage::kBytes, sums_to = sums_of + Stage::kSums;
  auto next_stage = [&](int q) { return q == (RING - 1) * Stage::kBytes ? 0 : q + Stage::kBytes; };
  auto scaled = [&](float scale, float zero, int a, int e, float t) {
    const float v = Stage::kOnes ? __builtin_fmaf(zero, ones[a][e], acc[a][e]) : acc[a][e];
    return __builtin_fmaf(scale, v, t);
  };
  // A step: products of 32 x 32 x 16, in chains of a block's S for 32 rows of x. Each
  // is followed, in the shadow of its MFMA, by the read of x for the product DEEP on,
  // its share of the loads for the step RING - 1 on, a share of the last chain's
  // scaling, and in the second half of a block a share of unpacking the next.
  auto run = [&](int step, Ready& fa, Ready& fb, auto swap) {
    block_barrier();
    load_sums(step + 1, lds + sums_to);
    const char* const xs = lds + at;
    const int after = next_stage(at);
    auto read = [&](int i) {
      const int b = i / P, u = i / S % U, j = i % S;
      return *reinterpret_cast<const v4u*>(xs + (32 * u + c) * 256 + 16 * ((b * (GB / 8) + h * S + j) ^ (c & 15)));
    };
    auto read_sum = [&](int b, int u) {
      // (Not as a uint2: the compiler would wait for every DMA in flight before it.)
      const v2u q = *reinterpret_cast<const v2u*>(lds + sums_of + 1024 * b + 256 * u + 8 * c);
      return make_uint2(q[0], q[1]);
    };
    v4u x[DEEP];
    uint2 sum[2];
    Raw raw;
    if constexpr (Stage::kPre) sum[0] = read_sum(0, 0);
#pragma unroll
    for (int i = 0; i < DEEP; ++i) x[i] = read(i);
    __builtin_amdgcn_sched_barrier(0);
    // The step's loads go out before the fetch of the next step's first codes, whose
    // wait counts them.
    constexpr int kFetch = P / 4, kEach = (Stage::kDma - 1) / ((NB - 1) * P + kFetch) + 1;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int b = i / P, u = i / S % U, j = i % S, in = i % P, a = (i / S + swap()) & 1;
      Ready& f = b & 1 ? fb : fa;
      Ready& g = b & 1 ? fa : fb;
      if (in == kFetch) {
        // (A wave's codes are its own DMA.)
        if (b + 1 == NB) wait_loads<(RING - 2) * Stage::kDma>();
        fetch(lds + (b + 1 == NB ? after : at), b + 1 == NB ? 0 : b + 1, raw);
      }
      if (j == 0) {
        if constexpr (Stage::kPre) acc[a] = mfma_zero(sum[u & 1], make_uint2(f.zero, f.zero));
        else acc[a] = v16f{};
        ones[a] = v16f{};
      }
      acc[a] = mfma32<DT>(x[i % DEEP], f.w[j], acc[a]);
      if constexpr (Stage::kOnes)
        ones[a] = mfma32<DT>(x[i % DEEP], v4u{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u}, ones[a]);
      if (i + DEEP < N) x[i % DEEP] = read(i + DEEP);
      if (Stage::kPre && j == 0 && i + S < N) sum[(u + 1) & 1] = read_sum((i + S) / P, (u + 1) % U);
#pragma unroll
      for (int d = i * kEach; d < (i + 1) * kEach; ++d)
        if (d < Stage::kDma) load(step + RING - 1, lds + to, d);
      if (j > 0) {
        const float scale = u ? f.scale : carry, zero = u ? __uint_as_float(f.zero) : carry_zero;
        const int last_u = (u + U - 1) % U;
#pragma unroll
        for (int e = 16 * (j - 1) / (S - 1); e < 16 * j / (S - 1); ++e)
          tot[last_u][e] = scaled(scale, zero, a ^ 1, e, tot[last_u][e]);
      }
      if (in == P / 2) open(step + (b + 1 == NB), b + 1 == NB ? 0 : b + 1, raw, g);
      const int past = in - P / 2;
      if (past >= 0 && past * 2 % U == 0) weights(raw, past * 2 / U, g);
      if (past >= 0 && U == 1) weights(raw, past * 2 + 1, g);
      if (in == P - 1) {
        carry = f.scale;
        carry_zero = __uint_as_float(f.zero);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    at = after;
    to = next_stage(to);
    const int q = sums_of;
    sums_of = sums_to;
    sums_to = q;
  };
  load_sums(first, lds + sums_of);
#pragma unroll
  for (int i = 0; i < RING - 1; ++i)
#pragma unroll
    for (int j = 0; j < Stage::kDma; ++j) load(first + i, lds + i * Stage::kBytes, j);
  wait_loads<(RING - 2) * Stage::kDma>();
  Ready f0, f1;
  {
    Raw raw;
    fetch(lds, 0, raw);
    open(first, 0, raw, f0);
#pragma unroll
    for (int j = 0; j < S; ++j) weights(raw, j, f0);
  }
  // (The last chain's accumulators are acc[1], but after an odd number of steps of one chain.)
  auto flush = [&](int a) {
#pragma unroll
    for (int e = 0; e < 16; ++e) tot[U - 1][e] = scaled(carry, carry_zero, a, e, tot[U - 1][e]);
  };
  constexpr std::integral_constant<int, 0> zero;
  if constexpr (NB == 1) {
    int step = first;
    for (; step + 1 < last; step += 2) {
      run(step, f0, f1, zero);
      run(step + 1, f1, f0, std::integral_constant<int, ODD>{});
    }
    if (step < last) {
      run(step, f0, f1, zero);
      flush(ODD ? 0 : 1);
    } else {
      flush(1);
    }
  } else {
    for (int step = first; step < last; ++step) run(step, f0, f1, zero);
    flush(1);
  }
  wait_loads<0>();     // no DMA outlives the workgroup's LDS
  float* const part =
      split_up ? parts + ((int64_t)split * rest + left) * (32 * U * 32 * W) + 32 * wave + c : nullptr;
  store_tile<DT, U, GATED>(p, tot, part, 32 * W, m0, n0, mrows, nrows, wr, ncol, c, h);
}

// The outputs of the split tiles: the ranges' sums in order, then the epilogue. Four
// neighbouring outputs of a row a thread.
template <int DT, int U, int W, bool GATED>
__global__ __launch_bounds__(256)
void linear_w4_join_kernel(W4Params p, const float* parts, int mtiles, int whole, int rest, int splits) {
  constexpr int BN = GATED ? 16 * W : 32 * W, BLOCKS = 32 * U * BN / 1024;
  const int64_t width = GATED ? p.n / 2 : p.n;
  const int left = blockIdx.x / BLOCKS, tile = whole + left;
  const int i = (blockIdx.x - left * BLOCKS) * 256 + threadIdx.x, row = i / (BN / 4), col = 4 * (i - row * (BN / 4));
  const int64_t m = (int64_t)(tile % mtiles) * (32 * U) + row, n = (int64_t)(tile / mtiles) * BN + col;
  if (m >= p.m || n >= width) return;
  const int64_t stride = (int64_t)rest * (32 * U * 32 * W);
  const float* at = parts + ((int64_t)left * (32 * U) + row) * (32 * W) + (GATED ? 32 * (col / 16) + col % 16 : col);
  auto of = [&](int s, int half) { return *reinterpret_cast<const v4f*>(at + s * stride + 16 * half); };
  v4f v = of(0, 0), up = {};
  if constexpr (GATED) up = of(0, 1);
  int s = 1;
  for (; s + 4 <= splits; s += 4) {   // (four loads at once)
    v4f a[4], b[4] = {};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      a[j] = of(s + j, 0);
      if constexpr (GATED) b[j] = of(s + j, 1);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v = v + a[j];
      if constexpr (GATED) up = up + b[j];
    }
  }
  for (; s < splits; ++s) {
    v = v + of(s, 0);
    if constexpr (GATED) up = up + of(s, 1);
  }
  finish4<DT, GATED>(p, m, n, width, v, up);
}

// How a call of more than eight rows is cut: 32 u rows and 32 w weight rows a tile.
// With 128 rows a tile a CU holds one workgroup, and the tiles past the last whole
// round of the GPU take ranges of k, as many as give each CU one and of at least four
// steps (300 tiles of 353 x 25600 x 5120 gated: 111 to 117 us, 152 to 156 with a second
// round of 44 tiles). Smaller tiles do so where they are fewer than the CUs. (Two ranges a CU
// cost more to join than they hide: us, one / two, 64 x 4096 x 14336 21.3 / 24.2, 16 x
// 4096 x 14336 14.6 / 16.9, 64 x 14336 x 4096 20.3 / 21.4; 32 x 14336 x 4096 15.7 /
// 15.8.)
struct W4Plan {
  int u, w, mtiles, splits;
  int64_t whole, rest;   // tiles with all of k, and tiles in `splits` ranges
  int64_t rows() const { return 32 * u; }
  int64_t cols() const { return 32 * w; }
};

static W4Plan w4_plan(int64_t m, int64_t n, int64_t k, int cus) {
  W4Plan q;
  q.u = m > 64 ? 4 : m > 32 ? 2 : 1;
  q.w = q.u == 4 ? 8 : 4;
  q.mtiles = (int)((m + q.rows() - 1) / q.rows());
  const int64_t tiles = (n + q.cols() - 1) / q.cols() * q.mtiles, steps = (k + 127) / 128;
  q.rest = q.u == 4 || tiles < cus ? tiles % cus : 0;
  const int64_t s = q.rest ? std::min(cus / q.rest, steps / 4) : 1;
  q.splits = s < 2 ? 1 : (int)s;
  if (q.splits == 1) q.rest = 0;
  q.whole = tiles - q.rest;
  return q;
}

// Whether a call takes the tiles (offsets inside a tile are 32 bits there).
static bool w4_tiled(int64_t m) { return m > 8; }

// Bytes of the sums of x (bf16 with many rows; asked of fp16 alike) and, behind
// them, of the ranges' sums.
static int64_t w4_sums_bytes(const W4Plan& q, int64_t m, int64_t k, int group) {
  return q.u == 4 ? 8 * ((m + 127) / 128 * 128) * (k / (group < 128 ? group : 128)) : 0;
}

template <int DT, int GB, int U, int W, bool GATED>
static void launch_w4_plan(const W4Params& p, const W4Plan& q, void* workspace, hipStream_t stream) {
  uint2* sums = reinterpret_cast<uint2*>(workspace);
  float* parts = reinterpret_cast<float*>(reinterpret_cast<char*>(workspace) + w4_sums_bytes(q, p.m, p.k, p.group));
  if (DT == kBF16 && U == 4)
    hipLaunchKernelGGL((w4_sums_kernel<DT, GB>), dim3((unsigned)std::min((p.m * (p.k / 8) + 255) / 256, kSumsBlocks)),
                       dim3(256), 0, stream, p, sums);
  const dim3 grid((unsigned)((q.whole + 7) / 8 * 8 + (q.rest * q.splits + 7) / 8 * 8));
  hipLaunchKernelGGL((linear_w4_tiles_kernel<DT, GB, U, W, GATED>), grid, dim3(64 * W), 0, stream, p, sums, parts,
                     q.mtiles, (int)q.whole, (int)q.rest, q.splits);
  if (q.rest)
    hipLaunchKernelGGL((linear_w4_join_kernel<DT, U, W, GATED>),
                       dim3((unsigned)(q.rest * (32 * U * (GATED ? 16 * W : 32 * W) / 1024))), dim3(256), 0, stream, p,
                       parts, q.mtiles, (int)q.whole, (int)q.rest, q.splits);
}

template <int DT, int GB, bool GATED>
static int launch_w4_tiles(const W4Params& p, void* workspace, hipStream_t stream) {
  const W4Plan q = w4_plan(p.m, p.n, p.k, current_device_cus());
  W8A8_REQUIRE(q.whole + q.rest < ((int64_t)1 << 22) && p.n < (1 << 30) && p.ldx < (1 << 22) && p.ldw < (1 << 22),
               "w8a8_linear_w4: too many outputs, or rows too long, for more than eight rows of x");
  switch (q.u) {
    case 4: launch_w4_plan<DT, GB, 4, 8, GATED>(p, q, workspace, stream); break;
    case 2: launch_w4_plan<DT, GB, 2, 4, GATED>(p, q, workspace, stream); break;
    default: launch_w4_plan<DT, GB, 1, 4, GATED>(p, q, workspace, stream); break;
  }
  return launch_status("w8a8_linear_w4");
}

template <int DT, int GB, bool GATED>
static int launch_w4(const W4Params& p, void* workspace, hipStream_t stream) {
  if (w4_tiled(p.m)) return launch_w4_tiles<DT, GB, GATED>(p, workspace, stream);
  W8A8_REQUIRE(p.n < (1 << 29), "w8a8_linear_w4: too many outputs for one launch");   // (eight threads an output)
  // Two tiles of weight rows share a wave's x, and four waves of ten or so blocks
  // each cost less to set up than eight of five; but where that leaves CUs idle on
  // long sums, one tile and eight waves (us, two tiles / one; one row of x: 14336 x
  // 4096 10.7 / 13.9, 5120 x 5120 7.9 / 9.9, 4096 x 14336 18.4 / 11.4).
  const int64_t width = GATED ? p.n / 2 : p.n, pairs = (width + (GATED ? 15 : 31)) / (GATED ? 16 : 32);
  if (!GATED && pairs < current_device_cus() && p.k > 64 * 128) {
    hipLaunchKernelGGL((linear_w4_kernel<DT, GB, 1, 8, false, 1>), dim3((unsigned)((width + 15) / 16)), dim3(512), 0,
                       stream, p);
  } else {
    hipLaunchKernelGGL((linear_w4_kernel<DT, GB, 2, 4, GATED, 1>), dim3((unsigned)pairs), dim3(256), 0, stream, p);
  }
  return launch_status("w8a8_linear_w4");
}

template <int DT>
static int launch_w4_group(const W4Params& p, bool gated, void* ws, hipStream_t s) {
  switch (p.group) {
    case 32: return gated ? launch_w4<DT, 32, true>(p, ws, s) : launch_w4<DT, 32, false>(p, ws, s);
    case 64: return gated ? launch_w4<DT, 64, true>(p, ws, s) : launch_w4<DT, 64, false>(p, ws, s);
    default: return gated ? launch_w4<DT, 128, true>(p, ws, s) : launch_w4<DT, 128, false>(p, ws, s);
  }
}

}  // namespace w8a8

extern "C" int64_t w8a8_linear_w4_workspace_size(int64_t m, int64_t n, int64_t k, int32_t group, int32_t) {
  using namespace w8a8;
  if (!w4_tiled(m) || n <= 0 || k <= 0 || group <= 0) return 0;
  const W4Plan q = w4_plan(m, n, k, current_device_cus());
  return w4_sums_bytes(q, m, k, group) + 4 * q.splits * q.rest * q.rows() * q.cols();
}

extern "C" int w8a8_linear_w4(const W8A8LinearW4Args* a) {
  using namespace w8a8;
  W8A8_REQUIRE(a != nullptr, "w8a8_linear_w4: null args");
  W8A8_REQUIRE(a->struct_size == sizeof(W8A8LinearW4Args), "w8a8_linear_w4: struct_size %u != %zu", a->struct_size,
               sizeof(W8A8LinearW4Args));
  W8A8_REQUIRE(a->dtype == W8A8_F16 || a->dtype == W8A8_BF16, "w8a8_linear_w4: dtype %d not F16/BF16", a->dtype);
  W8A8_REQUIRE(a->gated == 0 || a->gated == 1, "w8a8_linear_w4: gated must be 0 or 1");
  W8A8_REQUIRE(a->group == 32 || a->group == 64 || (a->group > 0 && a->group % 128 == 0),
               "w8a8_linear_w4: group %d not 32, 64 or a multiple of 128", a->group);
  W8A8_REQUIRE(a->m >= 0 && a->n >= 0 && a->k > 0 && a->m < ((int64_t)1 << 22) && a->n < ((int64_t)1 << 31) &&
                   a->k < ((int64_t)1 << 31),
               "w8a8_linear_w4: size out of range");
  W8A8_REQUIRE(a->k % a->group == 0, "w8a8_linear_w4: k %lld not a multiple of the group %d", (long long)a->k,
               a->group);
  W8A8_REQUIRE(!a->gated || (a->n % 2 == 0 && !a->residual), "w8a8_linear_w4: gated needs an even n and no residual");
  if (a->m == 0 || a->n == 0) return W8A8_OK;
  const int64_t width = a->gated ? a->n / 2 : a->n;
  W8A8_REQUIRE(a->x && aligned16(a->x) && a->ldx >= a->k && a->ldx % 8 == 0,
               "w8a8_linear_w4: x must be 16-byte aligned with ldx >= k, a multiple of 8");
  W8A8_REQUIRE(a->codes && aligned16(a->codes) && a->ldw >= a->k / 8 && a->ldw % 4 == 0,
               "w8a8_linear_w4: codes must be 16-byte aligned with ldw >= k / 8, a multiple of 4");
  W8A8_REQUIRE(a->scales && (uintptr_t)a->scales % 2 == 0, "w8a8_linear_w4: null or misaligned scales");
  W8A8_REQUIRE((uintptr_t)a->bias % 2 == 0 && (uintptr_t)a->residual % 2 == 0 && (!a->residual || a->ldr >= width),
               "w8a8_linear_w4: bias or residual misaligned, or ldr below n");
  W8A8_REQUIRE(a->out && (uintptr_t)a->out % 2 == 0 && a->ldo >= width, "w8a8_linear_w4: null out, or ldo below n");
  const RowsOf vo = rows_of(a->out, a->ldo, a->m, width, 2);
  W8A8_REQUIRE(apart(vo, rows_of(a->x, a->ldx, a->m, a->k, 2)), "w8a8_linear_w4: out overlaps x");
  W8A8_REQUIRE(!a->residual || (a->residual == a->out && a->ldr == a->ldo) ||
                   apart(vo, rows_of(a->residual, a->ldr, a->m, width, 2)),
               "w8a8_linear_w4: out overlaps the residual without being it");
  const int64_t need = w8a8_linear_w4_workspace_size(a->m, a->n, a->k, a->group, a->gated);
  W8A8_REQUIRE(need == 0 || (a->workspace && aligned16(a->workspace) && a->workspace_bytes >= need),
               "w8a8_linear_w4: workspace of %lld bytes needed", (long long)need);
  const W4Params p{a->x, a->ldx, reinterpret_cast<const uint32_t*>(a->codes), a->ldw,
                   reinterpret_cast<const uint16_t*>(a->scales), a->zeros, a->m, a->n, a->k, a->group,
                   reinterpret_cast<const uint16_t*>(a->bias), reinterpret_cast<const uint16_t*>(a->residual), a->ldr,
                   reinterpret_cast<uint16_t*>(a->out), a->ldo,
                   width % 4 == 0 && a->ldo % 4 == 0 && (uintptr_t)a->out % 8 == 0 && (uintptr_t)a->scales % 8 == 0 &&
                       (uintptr_t)a->zeros % 4 == 0};
  hipStream_t s = reinterpret_cast<hipStream_t>(a->stream);
  return a->dtype == W8A8_F16 ? launch_w4_group<kF16>(p, a->gated != 0, a->workspace, s)
                              : launch_w4_group<kBF16>(p, a->gated != 0, a->workspace, s);
}
