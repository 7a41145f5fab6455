// The residual stream between two blocks: x' = r x + gate * s * norm(branch),
// then the next block's modulated RMSNorm of x', stored or rotated and
// quantized, in one pass over x and the branch.
//
// One wavefront per row, lane l owning the 16-element units u = l + 64 j as in
// norm_quant.hip, so that the sum of squares of x' has that kernel's order and
// y, codes and scales are its bits on the stored rows. The sum of the branch's
// squares is taken unit wave by unit wave (each 64 units' partials in a
// butterfly, then the sums in order of j).
//
// Bound by memory: x and the branch are read once, x' and y or the codes
// written once; the row waits in registers between its three steps.
#include "norm_device.h"
#include "w8a8_host.h"

#include <type_traits>

namespace w8a8 {

constexpr int kResWaves = 4;

struct ResNormParams {
  const void* x;
  const void* branch;
  void* out;
  int64_t ldx, ldb, ldo, rows, cols;
  const float* post_weight;
  const float* gate;
  int64_t ld_gate;
  const int32_t* labels;
  int32_t gate_rows, mod_rows;
  float post_eps, branch_scale, residual_scale, eps, inv_cols;
  const float* weight;
  const float* shift;
  const float* mscale;
  int64_t ld_mod;
  void* y;
  int64_t ldy;
  int8_t* q;
  int64_t ldq;
  float* qscale;
  const uint32_t* signs;   // ConvRot sign words (0 or 0x80000000 per column), or null
  bool post, pre;
};

// MODE: 0 update, and the norm where p.pre, 1 quantize, 2 ConvRot256 (fp32) +
// quantize, 3 ConvRot256 rounded to the storage dtype + quantize.
template <int DT, int BT, int MODE, int J>
__global__ __launch_bounds__(64 * kResWaves)
void residual_norm_kernel(ResNormParams p) {
  constexpr bool ROT = MODE >= 2;
  constexpr bool PS = ROT && kPrescaled<DT>;
  extern __shared__ __attribute__((aligned(16))) float dsm[];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kResWaves + wave;
  if (row >= p.rows) return;
  const int units = (int)(p.cols >> 4);
  const uint16_t* xrow = reinterpret_cast<const uint16_t*>(p.x) + row * p.ldx;
  const char* brow = reinterpret_cast<const char*>(p.branch) + row * p.ldb * (BT == kF32 ? 4 : 2);
  uint16_t* orow = reinterpret_cast<uint16_t*>(p.out) + row * p.ldo;
  uint16_t* yrow = p.y ? reinterpret_cast<uint16_t*>(p.y) + row * p.ldy : nullptr;
  const float* gate = nullptr;
  const float* sh = nullptr;
  const float* sc = nullptr;
  if (p.labels) {
    const int l = p.labels[row];
    if (p.gate) gate = p.gate + (int64_t)min(max(l, 0), p.gate_rows - 1) * p.ld_gate;
    if (p.shift) {
      const int64_t m = (int64_t)min(max(l, 0), p.mod_rows - 1) * p.ld_mod;
      sh = p.shift + m;
      sc = p.mscale + m;
    }
  }
  float* buf = ROT ? rot_slot(dsm, wave, lane) : nullptr;
  const int t = lane & 15;

  auto squares16 = [](float ss, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
    return ss;
  };
  auto butterfly = [](float ss) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) ss = ss + __shfl_xor(ss, off, 64);
    return ss;
  };
  auto inv_rms = [&](float ss, float eps) {
    const float mean = ss * p.inv_cols;
    const float d = mean + eps;
    return 1.0f / __builtin_sqrtf(d);
  };
  // x' of one unit: xr its stored x (replaced by x'), v the branch (replaced
  // by x' as fp32).
  auto update = [&](int u, uint4 (&xr)[4], float (&v)[16], float pinv) {
    float x[16], w[16];
    unpack16<DT>(xr, x);
    const int64_t c0 = (int64_t)u * 16;
    if (p.post) {
#pragma unroll
      for (int i = 0; i < 16; ++i) v[i] = v[i] * pinv;
      if (p.post_weight) {
        load16_f32(p.post_weight + c0, w);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = v[i] * w[i];
      }
    }
    if (gate) load16_f32(gate + c0, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const float s = v[i] * p.branch_scale;
      const float r = x[i] * p.residual_scale;
      v[i] = gate ? __builtin_fmaf(s, w[i], r) : r + s;
    }
    uint32_t bits[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (DT == kF16) bits[i] = f2h2_of_f32(v[2 * i], v[2 * i + 1]);
      else bits[i] = (uint32_t)f2bf(v[2 * i]) | ((uint32_t)f2bf(v[2 * i + 1]) << 16);
    }
    xr[0] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
    xr[1] = make_uint4(bits[4], bits[5], bits[6], bits[7]);
    unpack16<DT>(xr, v);
    uint4* dst = reinterpret_cast<uint4*>(orow + c0);
    dst[0] = xr[0];
    dst[1] = xr[1];
  };
  // Normalize one unit (v holds x'), store y, rotate for the quantizer.
  auto finish = [&](int u, float (&v)[16], float inv, bool store_y) {
    uint32_t bits[8];
    modulate16<DT, kAnyTables, PS>(v, bits, inv, p.weight, sh, sc, (int64_t)u * 16);
    if (store_y && yrow) {
      uint4* dst = reinterpret_cast<uint4*>(yrow + (int64_t)u * 16);
      dst[0] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
      dst[1] = make_uint4(bits[4], bits[5], bits[6], bits[7]);
    }
    if constexpr (ROT) {
      if (p.signs) {
        const uint4* m = reinterpret_cast<const uint4*>(p.signs + (int64_t)u * 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint4 w = m[i];
          v[4 * i] = __uint_as_float(__float_as_uint(v[4 * i]) ^ w.x);
          v[4 * i + 1] = __uint_as_float(__float_as_uint(v[4 * i + 1]) ^ w.y);
          v[4 * i + 2] = __uint_as_float(__float_as_uint(v[4 * i + 2]) ^ w.z);
          v[4 * i + 3] = __uint_as_float(__float_as_uint(v[4 * i + 3]) ^ w.w);
        }
      }
      convrot256_lanes<true, false, PS>(v, buf, t);
      if constexpr (MODE == 3) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = round_to<DT>(v[i]);
      }
    }
  };
  auto absmax16 = [](float amax, const float (&v)[16]) {
#pragma unroll
    for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(v[i]));
    return amax;
  };
  auto store_q = [&](int u, const float (&v)[16], float s, float rcp) {
    *reinterpret_cast<uint4*>(p.q + row * p.ldq + (int64_t)u * 16) = quant16_each(v, s, rcp);
  };

  if constexpr (J > 0) {
    uint4 xr[J][4], br[J][4];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int u = lane + 64 * j;
      if (u < units) {
        raw16<BT>(brow + (int64_t)u * (BT == kF32 ? 64 : 32), br[j]);
        raw16<DT>(xrow + (int64_t)u * 16, xr[j]);
      }
    }
    float pinv = 1.0f;
    if (p.post) {
      float total = 0.0f;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        float part = 0.0f;
        if (lane + 64 * j < units) {
          float v[16];
          unpack16<BT>(br[j], v);
          part = squares16(part, v);
        }
        total = total + butterfly(part);
      }
      pinv = inv_rms(total, p.post_eps);
    }
    float ss = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int u = lane + 64 * j;
      if (u < units) {
        float v[16];
        unpack16<BT>(br[j], v);
        update(u, xr[j], v, pinv);
        ss = squares16(ss, v);
      }
    }
    if (MODE == 0 && !p.pre) return;
    const float inv = inv_rms(butterfly(ss), p.eps);
    float keep[MODE != 0 ? J : 1][16];
    float amax = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int u = lane + 64 * j;
      if (u < units) {
        float (&v)[16] = keep[MODE != 0 ? j : 0];
        unpack16<DT>(xr[j], v);
        finish(u, v, inv, true);
        if constexpr (MODE != 0) amax = absmax16(amax, v);
      }
    }
    if constexpr (MODE != 0) {
      amax = wave_max(amax);
      const float s = row_scale_of(amax);
      const float rcp = 1.0f / s;
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const int u = lane + 64 * j;
        if (u < units) store_q(u, keep[j], s, rcp);
      }
      if (lane == 0) p.qscale[row] = s;
    }
  } else {
    // Rows too wide for registers: a pass per step, x' read back from out (a
    // lane reads what it wrote itself).
    const int jcount = (units + 63) >> 6;
    float pinv = 1.0f;
    if (p.post) {
      float total = 0.0f;
      for (int j = 0; j < jcount; ++j) {
        const int u = lane + 64 * j;
        float part = 0.0f;
        if (u < units) {
          float v[16];
          load16<BT>(brow + (int64_t)u * (BT == kF32 ? 64 : 32), v);
          part = squares16(part, v);
        }
        total = total + butterfly(part);
      }
      pinv = inv_rms(total, p.post_eps);
    }
    float ss = 0.0f;
    for (int j = 0; j < jcount; ++j) {
      const int u = lane + 64 * j;
      if (u < units) {
        uint4 xr[4];
        float v[16];
        raw16<DT>(xrow + (int64_t)u * 16, xr);
        load16<BT>(brow + (int64_t)u * (BT == kF32 ? 64 : 32), v);
        update(u, xr, v, pinv);
        ss = squares16(ss, v);
      }
    }
    if (MODE == 0 && !p.pre) return;
    const float inv = inv_rms(butterfly(ss), p.eps);
    float s = 0.0f, rcp = 0.0f;
    if constexpr (MODE != 0) {
      float amax = 0.0f;
      for (int j = 0; j < jcount; ++j) {
        const int u = lane + 64 * j;
        if (u < units) {
          float v[16];
          load16<DT>(orow + (int64_t)u * 16, v);
          finish(u, v, inv, false);
          amax = absmax16(amax, v);
        }
      }
      amax = wave_max(amax);
      s = row_scale_of(amax);
      rcp = 1.0f / s;
      if (lane == 0) p.qscale[row] = s;
    }
    for (int j = 0; j < jcount; ++j) {
      const int u = lane + 64 * j;
      if (u < units) {
        float v[16];
        load16<DT>(orow + (int64_t)u * 16, v);
        finish(u, v, inv, true);
        if constexpr (MODE != 0) store_q(u, v, s, rcp);
      }
    }
  }
}

template <int DT, int BT, int MODE>
static int launch_residual_norm(const ResNormParams& p, hipStream_t stream) {
  const int jneed = (int)(((p.cols >> 4) + 63) / 64);
  const dim3 grid((unsigned)((p.rows + kResWaves - 1) / kResWaves)), block(64 * kResWaves);
  const size_t lds = MODE >= 2 ? sizeof(float) * kResWaves * kRotWave : 0;
  auto go = [&](auto j_tag) {
    hipLaunchKernelGGL((residual_norm_kernel<DT, BT, MODE, decltype(j_tag)::value>), grid, block, lds, stream, p);
  };
  switch (jneed) {
    case 1: go(std::integral_constant<int, 1>{}); break;
    case 2: go(std::integral_constant<int, 2>{}); break;
    case 3: case 4: go(std::integral_constant<int, 4>{}); break;
    case 5: case 6: go(std::integral_constant<int, 6>{}); break;
    default: go(std::integral_constant<int, 0>{}); break;
  }
  return launch_status("w8a8_residual_norm");
}

template <int DT, int BT>
static int launch_residual_norm_mode(int mode, const ResNormParams& p, hipStream_t stream) {
  switch (mode) {
    case 0: return launch_residual_norm<DT, BT, 0>(p, stream);
    case 1: return launch_residual_norm<DT, BT, 1>(p, stream);
    case 2: return launch_residual_norm<DT, BT, 2>(p, stream);
    default: return launch_residual_norm<DT, BT, 3>(p, stream);
  }
}

}  // namespace w8a8

extern "C" int w8a8_residual_norm(const W8A8ResidualNormArgs* a) {
  using namespace w8a8;
  W8A8_REQUIRE(a != nullptr, "w8a8_residual_norm: null args");
  W8A8_REQUIRE(a->struct_size == sizeof(W8A8ResidualNormArgs), "w8a8_residual_norm: struct_size %u != %zu",
               a->struct_size, sizeof(W8A8ResidualNormArgs));
  W8A8_REQUIRE(a->x_dtype == W8A8_F16 || a->x_dtype == W8A8_BF16, "w8a8_residual_norm: x_dtype %d not F16/BF16",
               a->x_dtype);
  W8A8_REQUIRE(a->branch_dtype == a->x_dtype || a->branch_dtype == W8A8_F32,
               "w8a8_residual_norm: branch_dtype %d neither x's nor F32", a->branch_dtype);
  W8A8_REQUIRE((a->post == 0 || a->post == 1) && (a->post || !a->post_weight),
               "w8a8_residual_norm: post must be 0 or 1, and post_weight comes with post");
  W8A8_REQUIRE(a->rows >= 0 && a->cols >= 0 && a->rows < ((int64_t)1 << 31), "w8a8_residual_norm: bad shape");
  const bool pre = a->y != nullptr || a->q != nullptr;
  W8A8_REQUIRE(pre || (!a->weight && !a->mod_shift && !a->mod_scale),
               "w8a8_residual_norm: weight or modulation without an output of the norm");
  W8A8_REQUIRE(a->convrot == 0 || a->convrot == 256, "w8a8_residual_norm: convrot must be 0 or 256");
  W8A8_REQUIRE(a->round_rotated == 0 || a->round_rotated == 1, "w8a8_residual_norm: round_rotated must be 0 or 1");
  const int group = (a->q && a->convrot) ? 256 : 16;
  W8A8_REQUIRE(a->cols % group == 0, "w8a8_residual_norm: cols %lld not a multiple of %d", (long long)a->cols, group);
  W8A8_REQUIRE(a->cols <= ((int64_t)1 << 30), "w8a8_residual_norm: cols too large");
  W8A8_REQUIRE((a->mod_shift == nullptr) == (a->mod_scale == nullptr),
               "w8a8_residual_norm: mod_shift and mod_scale go together");
  if (a->rows == 0) return W8A8_OK;
  W8A8_REQUIRE(a->cols > 0, "w8a8_residual_norm: zero-width rows have no norm");
  const int bs = a->branch_dtype == W8A8_F32 ? 4 : 2;
  W8A8_REQUIRE(a->x && aligned16(a->x) && a->ldx >= a->cols && a->ldx % 8 == 0,
               "w8a8_residual_norm: x must be 16-byte aligned with ldx >= cols and a 16-byte row stride");
  W8A8_REQUIRE(a->branch && aligned16(a->branch) && a->ldb >= a->cols && (a->ldb * bs) % 16 == 0,
               "w8a8_residual_norm: branch must be 16-byte aligned with ldb >= cols and a 16-byte row stride");
  W8A8_REQUIRE(a->out && aligned16(a->out) && a->ldo >= a->cols && a->ldo % 8 == 0,
               "w8a8_residual_norm: out must be 16-byte aligned with ldo >= cols and a 16-byte row stride");
  const RowsOf vx = rows_of(a->x, a->ldx, a->rows, a->cols, 2), vb = rows_of(a->branch, a->ldb, a->rows, a->cols, bs),
               vo = rows_of(a->out, a->ldo, a->rows, a->cols, 2);
  W8A8_REQUIRE((a->out == a->x && a->ldo == a->ldx) || apart(vo, vx),
               "w8a8_residual_norm: out overlaps x without being it");
  W8A8_REQUIRE(apart(vo, vb), "w8a8_residual_norm: out overlaps the branch");
  if (a->y) {
    const RowsOf vy = rows_of(a->y, a->ldy, a->rows, a->cols, 2);
    W8A8_REQUIRE(aligned16(a->y) && a->ldy >= a->cols && a->ldy % 8 == 0,
                 "w8a8_residual_norm: y must be 16-byte aligned with ldy >= cols and a 16-byte row stride");
    W8A8_REQUIRE(apart(vy, vx) && apart(vy, vb) && apart(vy, vo), "w8a8_residual_norm: y overlaps x, the branch or out");
  }
  if (a->q) {
    W8A8_REQUIRE(a->q_scale != nullptr, "w8a8_residual_norm: q requires q_scale");
    W8A8_REQUIRE(aligned16(a->q) && a->ldq >= a->cols && a->ldq % 16 == 0,
                 "w8a8_residual_norm: q must be 16-byte aligned with ldq >= cols, a multiple of 16");
    for (const RowsOf& v : {rows_of(a->q, a->ldq, a->rows, a->cols, 1), rows_of(a->q_scale, 1, a->rows, 1, 4)})
      W8A8_REQUIRE(apart(v, vx) && apart(v, vb) && apart(v, vo),
                   "w8a8_residual_norm: q or q_scale overlaps x, the branch or out");
  }
  W8A8_REQUIRE((!a->weight || aligned16(a->weight)) && (!a->post_weight || aligned16(a->post_weight)),
               "w8a8_residual_norm: weights must be 16-byte aligned");
  W8A8_REQUIRE(!(a->gate || a->mod_shift) || a->labels, "w8a8_residual_norm: gate and modulation need labels");
  if (a->gate)
    W8A8_REQUIRE(a->gate_rows >= 1 && aligned16(a->gate) && a->ld_gate >= a->cols && a->ld_gate % 4 == 0,
                 "w8a8_residual_norm: gate must be 16-byte aligned with ld_gate >= cols, a multiple of 4");
  if (a->mod_shift)
    W8A8_REQUIRE(a->mod_rows >= 1 && aligned16(a->mod_shift) && aligned16(a->mod_scale) && a->ld_mod >= a->cols &&
                     a->ld_mod % 4 == 0,
                 "w8a8_residual_norm: tables must be 16-byte aligned with ld_mod >= cols, a multiple of 4");
  W8A8_REQUIRE(a->convrot_signs == nullptr || (a->q && a->convrot && aligned16(a->convrot_signs)),
               "w8a8_residual_norm: convrot_signs needs q, convrot and a 16-byte aligned array");
  ResNormParams p;
  p.x = a->x;
  p.branch = a->branch;
  p.out = a->out;
  p.ldx = a->ldx;
  p.ldb = a->ldb;
  p.ldo = a->ldo;
  p.rows = a->rows;
  p.cols = a->cols;
  p.post_weight = a->post_weight;
  p.gate = a->gate;
  p.ld_gate = a->ld_gate;
  p.labels = a->gate || a->mod_shift ? a->labels : nullptr;
  p.gate_rows = a->gate_rows;
  p.mod_rows = a->mod_rows;
  p.post_eps = a->post_eps;
  p.branch_scale = a->branch_scale;
  p.residual_scale = a->residual_scale;
  p.eps = a->eps;
  p.inv_cols = (float)(1.0 / (double)a->cols);
  p.weight = a->weight;
  p.shift = a->mod_shift;
  p.mscale = a->mod_scale;
  p.ld_mod = a->ld_mod;
  p.y = a->y;
  p.ldy = a->ldy;
  p.q = a->q;
  p.ldq = a->ldq;
  p.qscale = a->q_scale;
  p.signs = a->convrot_signs;
  p.post = a->post != 0;
  p.pre = pre;
  hipStream_t stream = reinterpret_cast<hipStream_t>(a->stream);
  const int mode = a->q == nullptr ? 0 : a->convrot == 0 ? 1 : a->round_rotated ? 3 : 2;
  const bool wide = a->branch_dtype == W8A8_F32;
  if (a->x_dtype == W8A8_F16)
    return wide ? launch_residual_norm_mode<kF16, kF32>(mode, p, stream)
                : launch_residual_norm_mode<kF16, kF16>(mode, p, stream);
  return wide ? launch_residual_norm_mode<kBF16, kF32>(mode, p, stream)
              : launch_residual_norm_mode<kBF16, kBF16>(mode, p, stream);
}
