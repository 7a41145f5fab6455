// Projections with 4-bit weights and group scales on 16-bit activations.
//
//   y[m][n] = sum_g s[g][n] * sum_{k in g} (c[n][k] - z[g][n]) x[m][k]
//
// A code goes into the top bits of the mantissa of 16 in the activations' type
// (16 + c, exact in both types): one shift and one and-or make two weights, and
// the type's own MFMA takes them. Their group sum is the codes' plus 16 times
// the group's sum of x, which an MFMA with a row of ones gives, so that
//   sum (c - z) x = sum (16 + c) x - (16 + z) sum x
// in fp32: the two sums are at most some five times the result's size, so the
// difference keeps all but three of fp32's bits. Scales apply to a group's sum,
// in fp32.
//
// A 16-bit operand fragment of the 16 x 16 x 32 MFMA is eight inputs a lane,
// one word of codes; a lane's inputs of a block of GB (a group, or 128 inputs of
// a longer one) are a quarter of it in a row, so codes and activations are
// loaded as they lie, GB / 32 words and as many 16-byte runs a lane.
#include "w8a8_device.h"
#include "w8a8_host.h"

#include <type_traits>

namespace w8a8 {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef __bf16 v8b __attribute__((ext_vector_type(8)));
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
};

// The eight weights of a word as 16 + c, in the order of their inputs.
template <int DT>
__device__ __forceinline__ v4u weights8(uint32_t w) {
  if constexpr (DT == kF16) {
    constexpr uint32_t mask = 0x03c003c0u, one = 0x4c004c00u;
    return v4u{((w << 6) & mask) | one, ((w << 2) & mask) | one, ((w >> 2) & mask) | one, ((w >> 6) & mask) | one};
  } else {
    constexpr uint32_t mask = 0x00780078u, one = 0x41804180u;
    return v4u{((w << 3) & mask) | one, ((w >> 1) & mask) | one, ((w >> 5) & mask) | one, ((w >> 9) & mask) | one};
  }
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
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (n + i >= width) break;
    float v = y[i];
    if (p.bias) v = v + wide<DT>(p.bias[n + i]);
    if constexpr (GATED) {
      const float u = p.bias ? up[i] + wide<DT>(p.bias[width + n + i]) : up[i];
      v = swiglu(v, u);
    }
    if (p.residual) v = v + wide<DT>(p.residual[m * p.ldr + n + i]);
    p.out[m * p.ldo + n + i] = slim<DT>(v);
  }
}

// A workgroup of W waves takes 16 NT weight rows (gated: half of them gate, half
// the same rows of up) and 16 MT rows of x; its waves share out the blocks of k
// and add their sums in LDS, in the order of the waves.
template <int DT, int GB, int NT, int MT, int W, bool GATED>
__global__ __launch_bounds__(64 * W)
void linear_w4_kernel(W4Params p) {
  constexpr int S = GB / 32;   // MFMA steps of a block, and a lane's words of it
  __shared__ v4f part[W][NT * MT][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  const int64_t width = GATED ? p.n / 2 : p.n;
  constexpr int TILES = GATED ? NT / 2 : NT;   // tiles of outputs
  const int64_t n0 = (int64_t)blockIdx.x * (16 * TILES), m0 = (int64_t)blockIdx.y * (16 * MT);
  const uint32_t* wrow[NT];
  int64_t nd[NT];      // the lane's first row of the tile's result
#pragma unroll
  for (int t = 0; t < NT; ++t) {
    const int64_t base = n0 + 16 * (t % TILES), shift = t >= TILES ? width : 0;
    wrow[t] = p.codes + (shift + min(base + r, width - 1)) * p.ldw + g * S;
    nd[t] = shift + base + 4 * g;
  }
  const uint16_t* xrow[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t)
    xrow[t] = reinterpret_cast<const uint16_t*>(p.x) + min(m0 + 16 * t + r, p.m - 1) * p.ldx + g * (GB / 4);
  const v4u ones = DT == kF16 ? v4u{0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u}
                              : v4u{0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u};
  v4f tot[NT][MT] = {};
  const int blocks = (int)(p.k / GB);
  for (int b = wave; b < blocks; b += W) {
    uint32_t w[NT][S];
    v4u x[MT][S];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int j = 0; j < S; ++j) w[t][j] = wrow[t][(int64_t)b * (GB / 8) + j];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int j = 0; j < S; ++j)
        x[t][j] = *reinterpret_cast<const v4u*>(xrow[t] + (int64_t)b * GB + 8 * j);
    v4f acc[NT][MT] = {}, sum[MT] = {};
#pragma unroll
    for (int j = 0; j < S; ++j) {
#pragma unroll
      for (int t = 0; t < MT; ++t) sum[t] = mfma<DT>(ones, x[t][j], sum[t]);
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const v4u a = weights8<DT>(w[t][j]);
#pragma unroll
        for (int u = 0; u < MT; ++u) acc[t][u] = mfma<DT>(a, x[u][j], acc[t][u]);
      }
    }
    const int64_t grow = (int64_t)(b * GB / p.group) * p.n;
#pragma unroll
    for (int t = 0; t < NT; ++t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int64_t n = min(nd[t] + i, p.n - 1);
        const float s = wide<DT>(p.scales[grow + n]);
        const float z = p.zeros ? (float)p.zeros[grow + n] + 16.0f : 24.0f;
#pragma unroll
        for (int u = 0; u < MT; ++u)
          tot[t][u][i] = __builtin_fmaf(s, __builtin_fmaf(-z, sum[u][i], acc[t][u][i]), tot[t][u][i]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < NT; ++t)
#pragma unroll
    for (int u = 0; u < MT; ++u) part[wave][t * MT + u][lane] = tot[t][u];
  __syncthreads();
  for (int tu = wave; tu < TILES * MT; tu += W) {
    const int t = tu / MT, u = tu - t * MT;
    v4f y = part[0][tu][lane], up = {};
    for (int v = 1; v < W; ++v) y = y + part[v][tu][lane];
    if constexpr (GATED) {
      up = part[0][TILES * MT + tu][lane];
      for (int v = 1; v < W; ++v) up = up + part[v][TILES * MT + tu][lane];
    }
    const int64_t m = m0 + 16 * u + r;
    if (m < p.m) finish4<DT, GATED>(p, m, n0 + 16 * t + 4 * g, width, y, up);
  }
}

template <int DT, int GB, bool GATED>
static int launch_w4(const W4Params& p, hipStream_t stream) {
  constexpr int NT = 2, W = 8;
  const int64_t width = GATED ? p.n / 2 : p.n, per = GATED ? 16 * NT / 2 : 16 * NT;
  const int mt = p.m <= 16 ? 1 : p.m <= 32 ? 2 : 4;
  const dim3 grid((unsigned)((width + per - 1) / per), (unsigned)((p.m + 16 * mt - 1) / (16 * mt)));
  switch (mt) {
    case 1: hipLaunchKernelGGL((linear_w4_kernel<DT, GB, NT, 1, W, GATED>), grid, dim3(64 * W), 0, stream, p); break;
    case 2: hipLaunchKernelGGL((linear_w4_kernel<DT, GB, NT, 2, W, GATED>), grid, dim3(64 * W), 0, stream, p); break;
    default: hipLaunchKernelGGL((linear_w4_kernel<DT, GB, NT, 4, W, GATED>), grid, dim3(64 * W), 0, stream, p); break;
  }
  return launch_status("w8a8_linear_w4");
}

template <int DT>
static int launch_w4_group(const W4Params& p, bool gated, hipStream_t s) {
  switch (p.group) {
    case 32: return gated ? launch_w4<DT, 32, true>(p, s) : launch_w4<DT, 32, false>(p, s);
    case 64: return gated ? launch_w4<DT, 64, true>(p, s) : launch_w4<DT, 64, false>(p, s);
    default: return gated ? launch_w4<DT, 128, true>(p, s) : launch_w4<DT, 128, false>(p, s);
  }
}

}  // namespace w8a8

extern "C" int64_t w8a8_linear_w4_workspace_size(int64_t, int64_t, int64_t, int32_t, int32_t) { return 0; }

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
                   reinterpret_cast<uint16_t*>(a->out), a->ldo};
  hipStream_t s = reinterpret_cast<hipStream_t>(a->stream);
  return a->dtype == W8A8_F16 ? launch_w4_group<kF16>(p, a->gated != 0, s)
                              : launch_w4_group<kBF16>(p, a->gated != 0, s);
}
