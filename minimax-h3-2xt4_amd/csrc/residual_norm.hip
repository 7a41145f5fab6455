// The residual stream between two blocks: x' = r x + gate * s * norm(branch),
// then the next block's modulated RMSNorm of x', stored or rotated and
// quantized, in one pass over x and the branch.
//
// Lane l owns the 16-element units u = l + 64 j as in norm_quant.hip, and the sum
// of squares of x' has that kernel's order, so that y, codes and scales are its
// bits on the stored rows. The sum of the branch's squares is taken unit wave by
// unit wave (each 64 units' partials in a butterfly, then the sums in order of j).
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

// The tables of one row. Null: absent.
struct RowTables {
  const float* gate;
  const float* mul;    // mod_scale
  const float* add;    // mod_shift
};

__device__ __forceinline__ RowTables tables_of(const ResNormParams& p, int label) {
  RowTables t{};
  if (p.gate) t.gate = p.gate + (int64_t)min(max(label, 0), p.gate_rows - 1) * p.ld_gate;
  if (p.shift) {
    const int64_t m = (int64_t)min(max(label, 0), p.mod_rows - 1) * p.ld_mod;
    t.mul = p.mscale + m;
    t.add = p.shift + m;
  }
  return t;
}

// The factor of the (normalized) branch: (post_weight * branch_scale) * gate.
__device__ __forceinline__ void branch_factor(const ResNormParams& p, const RowTables& t, int64_t c0, float (&g)[16]) {
  float w[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) g[i] = p.branch_scale;
  if (p.post_weight) {
    load16_f32(p.post_weight + c0, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) g[i] = w[i] * g[i];
  }
  if (t.gate) {
    load16_f32(t.gate + c0, w);
#pragma unroll
    for (int i = 0; i < 16; ++i) g[i] = g[i] * w[i];
  }
}

// x' of a unit: xr its stored x (replaced by x'), v the branch (replaced by x' as
// fp32), g the branch's factor.
template <int DT>
__device__ __forceinline__ void update16(const ResNormParams& p, const float (&g)[16], uint4 (&xr)[4], float (&v)[16],
                                         float pinv) {
  float x[16];
  unpack16<DT>(xr, x);
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const float r = x[i] * p.residual_scale;
    v[i] = __builtin_fmaf(p.post ? v[i] * pinv : v[i], g[i], r);
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
}

__device__ __forceinline__ float squares16(float ss, const float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) ss = __builtin_fmaf(v[i], v[i], ss);
  return ss;
}

__device__ __forceinline__ float butterfly(float ss) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) ss = ss + __shfl_xor(ss, off, 64);
  return ss;
}

__device__ __forceinline__ float inv_rms(const ResNormParams& p, float ss, float eps) {
  const float mean = ss * p.inv_cols;
  return 1.0f / __builtin_sqrtf(mean + eps);
}

// The quantizer's rotation of a unit's normalized values (times 1/16 already
// where kPrescaled).
template <int DT, int MODE>
__device__ __forceinline__ void rotate16(const ResNormParams& p, int u, float* buf, int lane16, float (&v)[16]) {
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
  convrot256_lanes<true, false, kPrescaled<DT>>(v, buf, lane16);
}

__device__ __forceinline__ void store_y(const ResNormParams& p, int64_t row, int u, const uint32_t (&bits)[8]) {
  uint4* dst = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.y) + row * p.ldy + (uint32_t)(u * 16));
  dst[0] = make_uint4(bits[0], bits[1], bits[2], bits[3]);
  dst[1] = make_uint4(bits[4], bits[5], bits[6], bits[7]);
}

__device__ __forceinline__ float absmax16(float amax, const float (&v)[16]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) amax = fmaxf(amax, fabsf(v[i]));
  return amax;
}

// MODE: 0 the norm (where p.pre), 1 quantize, 2 ConvRot256 (fp32) + quantize, 3
// ConvRot256 rounded to the storage dtype + quantize (the maximum is taken before
// the rounding and rounded once: rounding is monotonic and odd).
template <int DT, int MODE>
__device__ __forceinline__ float scale_of(float amax) {
  return row_scale_of(MODE == 3 ? round_to<DT>(amax) : amax);
}

__device__ __forceinline__ void store_codes(const ResNormParams& p, int64_t row, int u, const float (&v)[16], float s,
                                            float rcp) {
  *reinterpret_cast<uint4*>(p.q + row * p.ldq + (uint32_t)(u * 16)) = quant16_each(v, s, rcp);
}

template <int BT>
__device__ __forceinline__ const char* branch_at(const ResNormParams& p, int64_t row, int u) {
  constexpr int es = BT == kF32 ? 4 : 2;
  return reinterpret_cast<const char*>(p.branch) + row * p.ldb * es + (uint32_t)(u * (16 * es));
}

__device__ __forceinline__ const uint16_t* x_at(const ResNormParams& p, int64_t row, int u) {
  return reinterpret_cast<const uint16_t*>(p.x) + row * p.ldx + (uint32_t)(u * 16);
}

__device__ __forceinline__ uint16_t* out_at(const ResNormParams& p, int64_t row, int u) {
  return reinterpret_cast<uint16_t*>(p.out) + row * p.ldo + (uint32_t)(u * 16);
}

__device__ __forceinline__ void store_x(const ResNormParams& p, int64_t row, int u, const uint4 (&xr)[4]) {
  uint4* dst = reinterpret_cast<uint4*>(out_at(p, row, u));
  dst[0] = xr[0];
  dst[1] = xr[1];
}

// modulate16's steps on an unit's tables in registers (mul: 1 + mod_scale formed
// already); v is left as the rounded values (times 1/16 where the rotation takes
// them so).
template <int DT, bool SCALED>
__device__ __forceinline__ void normalize16(float (&v)[16], float inv, const float (&gain)[16], bool has_gain,
                                            const float (&mul)[16], const float (&add)[16], bool has_mod,
                                            uint32_t (&bits)[8]) {
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = DT == kF16 ? mul_mix(v[i], inv) : v[i] * inv;
  if (has_gain) {
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = v[i] * gain[i];
  }
  if (has_mod) {
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      v[i] = v[i] * mul[i];
      v[i] = v[i] + add[i];
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == kF16) bits[i] = f2h2_of_f32(v[2 * i], v[2 * i + 1]);
    else bits[i] = (uint32_t)f2bf(v[2 * i]) | ((uint32_t)f2bf(v[2 * i + 1]) << 16);
    v[2 * i] = DT == kF16 ? h2f((uint16_t)bits[i]) : bf2f((uint16_t)bits[i]);
    v[2 * i + 1] = DT == kF16 ? h2f((uint16_t)(bits[i] >> 16)) : bf2f((uint16_t)(bits[i] >> 16));
  }
  if constexpr (SCALED) scale16(v);
}

// Few rows: a workgroup of J waves per row, unit wave j to wave j, whose loads of
// the row and of its tables are all under way at once. The branch's squares meet
// as the unit waves' sums; those of x' have norm_quant.hip's order, a chain through
// a lane's units, so each wave reads the whole row of x' from LDS and adds them
// all. (With rows in turn and the tables kept in registers it is slower than the
// staged kernel below wherever that fills the GPU: the redundant sums bind.)
template <int DT, int BT, int MODE, int J>
__global__ __launch_bounds__(64 * J)
void residual_norm_split_kernel(ResNormParams p) {
  constexpr bool PS = MODE >= 2 && kPrescaled<DT>;
  extern __shared__ __attribute__((aligned(16))) float dsm[];
  __shared__ uint4 xs[J][2][64];
  __shared__ float part[J], peak[J];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row = blockIdx.x;
  const int units = (int)(p.cols >> 4), u = lane + 64 * wave;
  const bool on = u < units;
  float* const buf = MODE >= 2 ? rot_slot(dsm, wave, lane) : nullptr;
  const int64_t c0 = (int64_t)(on ? u : 0) * 16;
  uint4 xr[4] = {}, br[4] = {};
  if (on) {
    raw16<BT>(branch_at<BT>(p, row, u), br);
    raw16<DT>(x_at(p, row, u), xr);
  }
  const RowTables t = tables_of(p, p.labels ? p.labels[row] : 0);
  float g[16], gain[16], mul[16], add[16];
  branch_factor(p, t, c0, g);
  if (p.weight) load16_f32(p.weight + c0, gain);
  if (t.add) {
    load16_f32(t.mul + c0, mul);
    load16_f32(t.add + c0, add);
#pragma unroll
    for (int i = 0; i < 16; ++i) mul[i] = 1.0f + mul[i];
  }
  float v[16];
  float pinv = 1.0f;
  if (p.post) {
    float ss = 0.0f;
    if (on) {
      unpack16<BT>(br, v);
      ss = squares16(ss, v);
    }
    ss = butterfly(ss);
    if (lane == 0) part[wave] = ss;
    __syncthreads();
    float total = 0.0f;
#pragma unroll
    for (int j = 0; j < J; ++j) total = total + part[j];
    pinv = inv_rms(p, total, p.post_eps);
  }
  if (on) {
    unpack16<BT>(br, v);
    update16<DT>(p, g, xr, v, pinv);
    store_x(p, row, u, xr);
  }
  if (MODE == 0 && !p.pre) return;
  float ss = 0.0f;
  if constexpr (J == 1) {
    if (on) ss = squares16(ss, v);
  } else {
    xs[wave][0][lane] = xr[0];
    xs[wave][1][lane] = xr[1];
    __syncthreads();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      if (lane + 64 * j < units) {
        const uint4 w[4] = {xs[j][0][lane], xs[j][1][lane]};
        float o[16];
        unpack16<DT>(w, o);
        ss = squares16(ss, o);
      }
    }
  }
  const float inv = inv_rms(p, butterfly(ss), p.eps);
  float amax = 0.0f;
  if (on) {
    uint32_t bits[8];
    normalize16<DT, PS>(v, inv, gain, p.weight != nullptr, mul, add, p.shift != nullptr, bits);
    if (p.y) store_y(p, row, u, bits);
    if constexpr (MODE >= 2) rotate16<DT, MODE>(p, u, buf, lane & 15, v);
    if constexpr (MODE != 0) amax = absmax16(amax, v);
  }
  if constexpr (MODE != 0) {
    amax = wave_max(amax);
    if constexpr (J > 1) {
      if (lane == 0) peak[wave] = amax;
      __syncthreads();
#pragma unroll
      for (int j = 0; j < J; ++j) amax = fmaxf(amax, peak[j]);
    }
    const float s = scale_of<DT, MODE>(amax);
    if (on) {
      if constexpr (MODE == 3) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = round_to<DT>(v[i]);
      }
      store_codes(p, row, u, v, s, 1.0f / s);
    }
    if (threadIdx.x == 0) p.qscale[row] = s;
  }
}

// Many rows: a row per wave, all its units in the wave's registers. A row's tables
// are up to five times its own bytes, and read from L2 for every row they bound the
// kernel (53504 x 5376 fp16 with all tables: 629 us), so a workgroup of twelve waves
// (eight where the branch is fp32: its units take twice the registers) stages those of
// its middle row's label in LDS - the branch's factor, the gain, 1 + mod_scale and
// mod_shift - and takes `per` rows; a row of another label reads its own from memory.
// 53504 x 5376 fp16 to rows 504 us (its bytes 476); 6814 x 5376 with an fp32 branch to
// codes 112 (68): there VALU is 38 % of the time and half of it is waiting for a row.
constexpr int staged_waves(int bt) { return bt == kF32 ? 8 : 12; }

// A unit's raw words out of the compiler's sight: it would otherwise keep what the
// pass before widened them to, twice the registers.
template <int DT>
__device__ __forceinline__ void unseen(uint4 (&r)[4]) {
#pragma unroll
  for (int i = 0; i < (DT == kF32 ? 4 : 2); ++i) __asm__ volatile("" : "+v"(r[i].x), "+v"(r[i].y), "+v"(r[i].z), "+v"(r[i].w));
}

struct Staged {
  const float* g;      // null: branch_scale
  const float* gain;   // null: none
  const float* mul;    // null: none
  const float* add;
};

template <int DT, int BT, int MODE, int J, bool STAGED>
__device__ __forceinline__ void norm_row(const ResNormParams& p, const Staged& st, const RowTables& t, int64_t row,
                                         int lane, float* buf) {
  constexpr bool PS = MODE >= 2 && kPrescaled<DT>;
  constexpr bool K16 = MODE == 3;   // what waits for the scale: 16 bits or 32
  const int units = (int)(p.cols >> 4);
  uint4 xr[J][4], br[J][4];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int u = lane + 64 * j;
    if (u < units) {
      raw16<BT>(branch_at<BT>(p, row, u), br[j]);
      raw16<DT>(x_at(p, row, u), xr[j]);
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
        unseen<BT>(br[j]);
      }
      total = total + butterfly(part);
    }
    pinv = inv_rms(p, total, p.post_eps);
  }
  float ss = 0.0f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int u = lane + 64 * j;
    if (u < units) {
      float v[16], g[16];
      if constexpr (STAGED) {
#pragma unroll
        for (int i = 0; i < 16; ++i) g[i] = p.branch_scale;
        if (st.g) load16_f32(st.g + 16 * u, g);
      } else {
        branch_factor(p, t, 16 * u, g);
      }
      unpack16<BT>(br[j], v);
      update16<DT>(p, g, xr[j], v, pinv);
      store_x(p, row, u, xr[j]);
      ss = squares16(ss, v);
      unseen<DT>(xr[j]);
    }
    // (One unit's tables at a time: the compiler would load them all at once.)
    __asm__ volatile("" : "+v"(ss) : : "memory");
  }
  if (MODE == 0 && !p.pre) return;
  const float inv = inv_rms(p, butterfly(ss), p.eps);
  uint32_t held[MODE != 0 ? J : 1][K16 ? 8 : 16];
  float amax = 0.0f;
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const int u = lane + 64 * j;
    if (u < units) {
      float v[16], gain[16], mul[16], add[16];
      uint32_t bits[8];
      unpack16<DT>(xr[j], v);
      const float* const from = STAGED ? st.gain : p.weight;
      const float* const sc = STAGED ? st.mul : t.mul;
      const float* const sh = STAGED ? st.add : t.add;
      if (from) load16_f32(from + 16 * u, gain);
      if (sh) {
        load16_f32(sc + 16 * u, mul);
        load16_f32(sh + 16 * u, add);
        if constexpr (!STAGED) {
#pragma unroll
          for (int i = 0; i < 16; ++i) mul[i] = 1.0f + mul[i];
        }
      }
      normalize16<DT, PS>(v, inv, gain, from != nullptr, mul, add, sh != nullptr, bits);
      if (p.y) store_y(p, row, u, bits);
      if constexpr (MODE >= 2) rotate16<DT, MODE>(p, u, buf, lane & 15, v);
      if constexpr (MODE != 0) {
        amax = absmax16(amax, v);
        if constexpr (K16) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            if constexpr (DT == kF16) held[j][i] = f2h2_of_f32(v[2 * i], v[2 * i + 1]);
            else held[j][i] = (uint32_t)f2bf(v[2 * i]) | ((uint32_t)f2bf(v[2 * i + 1]) << 16);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) held[j][i] = __float_as_uint(v[i]);
        }
      }
    }
    __asm__ volatile("" : "+v"(amax) : : "memory");
  }
  if constexpr (MODE != 0) {
    const float s = scale_of<DT, MODE>(wave_max(amax));
    const float rcp = 1.0f / s;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int u = lane + 64 * j;
      if (u < units) {
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          if constexpr (K16) {
            const uint16_t b = (uint16_t)(held[j][i >> 1] >> (16 * (i & 1)));
            v[i] = DT == kF16 ? h2f(b) : bf2f(b);
          } else {
            v[i] = __uint_as_float(held[j][i]);
          }
        }
        store_codes(p, row, u, v, s, rcp);
      }
    }
    if (lane == 0) p.qscale[row] = s;
  }
}

template <int DT, int BT, int MODE, int J>
__global__ __launch_bounds__(64 * staged_waves(BT), staged_waves(BT) / 4)
void residual_norm_staged_kernel(ResNormParams p, int per) {
  constexpr int W = staged_waves(BT);
  extern __shared__ __attribute__((aligned(16))) float dsm[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row0 = (int64_t)blockIdx.x * per, row1 = min(row0 + per, p.rows);
  float* const buf = MODE >= 2 ? rot_slot(dsm, wave, lane) : nullptr;
  float* next = dsm + (MODE >= 2 ? W * kRotWave : 0);
  const int label = p.labels ? p.labels[row0 + (row1 - row0) / 2] : 0, cols = (int)p.cols;
  const RowTables mid = tables_of(p, label);
  Staged st{};
  for (int i = 16 * threadIdx.x; i < cols; i += 16 * 64 * W) {
    float* at = next + i;
    auto put = [&](const float (&v)[16]) {
#pragma unroll
      for (int q = 0; q < 4; ++q)
        reinterpret_cast<float4*>(at)[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
      at += cols;
    };
    float v[16];
    if (p.post_weight || mid.gate) {
      branch_factor(p, mid, i, v);
      put(v);
    }
    if (p.weight) {
      load16_f32(p.weight + i, v);
      put(v);
    }
    if (mid.add) {
      load16_f32(mid.mul + i, v);
#pragma unroll
      for (int q = 0; q < 16; ++q) v[q] = 1.0f + v[q];
      put(v);
      load16_f32(mid.add + i, v);
      put(v);
    }
  }
  if (p.post_weight || mid.gate) {
    st.g = next;
    next += cols;
  }
  if (p.weight) {
    st.gain = next;
    next += cols;
  }
  if (mid.add) {
    st.mul = next;
    st.add = next + cols;
  }
  __syncthreads();
  for (int64_t row = row0 + wave; row < row1; row += W) {
    // (Its addresses formed anew for each row: kept, they take some forty registers.)
    int own = lane;
    __asm__ volatile("" : "+v"(own));
    const int l = p.labels ? p.labels[row] : 0;
    if (l == label) norm_row<DT, BT, MODE, J, true>(p, st, mid, row, own, buf);
    else norm_row<DT, BT, MODE, J, false>(p, st, tables_of(p, l), row, own, buf);
  }
}

// Rows too wide for registers: a wave per row, a pass per step, x' read back
// from out (a lane reads what it wrote itself).
template <int DT, int BT, int MODE>
__global__ __launch_bounds__(64 * kResWaves)
void residual_norm_wide_kernel(ResNormParams p) {
  extern __shared__ __attribute__((aligned(16))) float dsm[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * kResWaves + wave;
  if (row >= p.rows) return;
  const int units = (int)(p.cols >> 4), jcount = (units + 63) >> 6;
  const RowTables t = tables_of(p, p.labels ? p.labels[row] : 0);
  float* const buf = MODE >= 2 ? rot_slot(dsm, wave, lane) : nullptr;
  float v[16];
  float pinv = 1.0f;
  if (p.post) {
    float total = 0.0f;
    for (int j = 0; j < jcount; ++j) {
      const int u = lane + 64 * j;
      float part = 0.0f;
      if (u < units) {
        load16<BT>(branch_at<BT>(p, row, u), v);
        part = squares16(part, v);
      }
      total = total + butterfly(part);
    }
    pinv = inv_rms(p, total, p.post_eps);
  }
  float ss = 0.0f;
  for (int j = 0; j < jcount; ++j) {
    const int u = lane + 64 * j;
    if (u < units) {
      uint4 xr[4];
      raw16<DT>(x_at(p, row, u), xr);
      load16<BT>(branch_at<BT>(p, row, u), v);
      float g[16];
      branch_factor(p, t, (int64_t)u * 16, g);
      update16<DT>(p, g, xr, v, pinv);
      store_x(p, row, u, xr);
      ss = squares16(ss, v);
    }
  }
  if (MODE == 0 && !p.pre) return;
  const float inv = inv_rms(p, butterfly(ss), p.eps);
  auto finish = [&](int u, bool store) {
    uint32_t bits[8];
    load16<DT>(out_at(p, row, u), v);
    modulate16<DT, kAnyTables, (MODE >= 2 && kPrescaled<DT>)>(v, bits, inv, p.weight, t.add, t.mul, (int64_t)u * 16);
    if (store && p.y) store_y(p, row, u, bits);
    if constexpr (MODE >= 2) rotate16<DT, MODE>(p, u, buf, lane & 15, v);
  };
  float s = 0.0f, rcp = 0.0f;
  if constexpr (MODE != 0) {
    float amax = 0.0f;
    for (int j = 0; j < jcount; ++j) {
      const int u = lane + 64 * j;
      if (u < units) {
        finish(u, false);
        amax = absmax16(amax, v);
      }
    }
    s = scale_of<DT, MODE>(wave_max(amax));
    rcp = 1.0f / s;
    if (lane == 0) p.qscale[row] = s;
  }
  for (int j = 0; j < jcount; ++j) {
    const int u = lane + 64 * j;
    if (u < units) {
      finish(u, true);
      if constexpr (MODE != 0) {
        if constexpr (MODE == 3) {
#pragma unroll
          for (int i = 0; i < 16; ++i) v[i] = round_to<DT>(v[i]);
        }
        store_codes(p, row, u, v, s, rcp);
      }
    }
  }
}

// Rows that a workgroup per row takes: three for each of 256 CUs (of which a CU holds
// two at a time where a row has six waves). More go to the staged kernel (us, split /
// staged: 5120 columns with post norm to rows, 512 rows 7.3 / 9.8, 768 11.0 / 10.9,
// 1536 21.2 / 16.2; 5376 columns with gate, modulation and rotation to codes, fp32
// branch, 512 rows 11.2 / 16.9, 768 15.7 / 19.4, 1024 25.1 / 21.2).
constexpr int64_t kSplitRows = 768;

template <int DT, int BT, int MODE>
static int launch_residual_norm(const ResNormParams& p, hipStream_t stream) {
  const int jneed = (int)(((p.cols >> 4) + 63) / 64);
  if (jneed > 6) {
    hipLaunchKernelGGL((residual_norm_wide_kernel<DT, BT, MODE>), dim3((unsigned)((p.rows + kResWaves - 1) / kResWaves)),
                       dim3(64 * kResWaves), MODE >= 2 ? sizeof(float) * kResWaves * kRotWave : 0, stream, p);
    return launch_status("w8a8_residual_norm");
  }
  auto of_j = [&](auto go) {
    switch (jneed) {
      case 1: go(std::integral_constant<int, 1>{}); break;
      case 2: go(std::integral_constant<int, 2>{}); break;
      case 3: go(std::integral_constant<int, 3>{}); break;
      case 4: go(std::integral_constant<int, 4>{}); break;
      case 5: go(std::integral_constant<int, 5>{}); break;
      default: go(std::integral_constant<int, 6>{}); break;
    }
  };
  if (p.rows <= kSplitRows) {
    of_j([&](auto j_tag) {
      constexpr int J = decltype(j_tag)::value;
      hipLaunchKernelGGL((residual_norm_split_kernel<DT, BT, MODE, J>), dim3((unsigned)p.rows), dim3(64 * J),
                         MODE >= 2 ? sizeof(float) * J * kRotWave : 0, stream, p);
    });
    return launch_status("w8a8_residual_norm");
  }
  const int tables = (p.gate || p.post_weight ? 1 : 0) + (p.weight ? 1 : 0) + (p.shift ? 2 : 0);
  const size_t lds = sizeof(float) * ((MODE >= 2 ? staged_waves(BT) * kRotWave : 0) + (size_t)tables * p.cols);
  // As many rows to a workgroup as give each CU a whole number of them, 60 at
  // most (a workgroup whose rows have two labels holds up the others less).
  const int64_t cus = current_device_cus(), rounds = (p.rows + 60 * cus - 1) / (60 * cus);
  const int per = (int)((p.rows + cus * rounds - 1) / (cus * rounds));
  of_j([&](auto j_tag) {
    constexpr int J = decltype(j_tag)::value;
    constexpr int JJ = J == 3 ? 4 : J == 5 ? 6 : J;
    hipLaunchKernelGGL((residual_norm_staged_kernel<DT, BT, MODE, JJ>), dim3((unsigned)((p.rows + per - 1) / per)),
                       dim3(64 * staged_waves(BT)), lds, stream, p, per);
  });
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
