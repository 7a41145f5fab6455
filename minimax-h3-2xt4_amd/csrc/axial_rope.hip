// Rotary positions with several axes: pair p of a row turns by
// phi = position[axis[p]] * inv_freq[p], Q and K heads alike, optionally after
// a per-head RMS norm with gain; and the same rotations as a table.
//
// The angle is needed modulo a revolution, so it is taken in fp64 (position
// 10^6 times one radian is 1.6 * 10^5 revolutions: fp64 leaves 10^-10 of one,
// fp32 would leave a hundredth) down to the nearest quarter; what is left is
// rounded to fp32, for its sine and cosine.
// Each angle serves all heads of its row: a workgroup takes a row, puts its
// angles into LDS and turns all its heads from there.
//
// A head is split into chunks of 2 V channels: V pairs (V channels of each
// side, or V adjacent pairs), or 2 V channels that are not turned. A lane
// takes one chunk (C of them where V is 1), so a turn needs no other lane, and
// a head's 2^n lanes meet in a butterfly for the norm's sum.
//
// Bound by memory where rows are many: q and k are read and written once.
#include "w8a8_device.h"
#include "w8a8_host.h"

#include <type_traits>

namespace w8a8 {

constexpr int kAxThreads = 256;
constexpr int kAxPairs = 128;   // the most that a row has

struct AxTable {
  const void* positions;
  int64_t row_stride, axis_stride;
  int pos_type, pairs, axes;
  const double* inv_freq;
  const int32_t* axis;
};

struct AxRopeParams {
  const void* x[2];
  void* out[2];
  int64_t in_row[2], in_head[2], out_row[2], out_head[2];
  const float* gain[2];
  int heads[2];
  AxTable table;
  int dim, lanes;
  float eps, inv_dim;
};

__device__ __forceinline__ double position_of(const AxTable& t, int64_t row, int axis) {
  const int64_t i = row * t.row_stride + axis * t.axis_stride;
  if (t.pos_type == W8A8_POS_I64) return (double)reinterpret_cast<const int64_t*>(t.positions)[i];
  if (t.pos_type == W8A8_POS_I32) return (double)reinterpret_cast<const int32_t*>(t.positions)[i];
  return (double)reinterpret_cast<const float*>(t.positions)[i];
}

// Cosine and sine of 2 pi t: whole turns and the nearest quarter are taken off
// (exact), which leaves |x| <= pi / 4, rounded here to fp32 (2^-25), where the
// Taylor series to x^9 and x^10 are within 2^-29 of sine and cosine. With the
// roundings of their sums both are within 1.3 * 2^-24. (Rounded before the
// quarter is off, the fraction alone would be 2^-23.3 off.)
__device__ __forceinline__ float2 cos_sin_turns(double t) {
  const double f = t - rint(t), n = rint(4.0 * f);
  const float x = (float)((f - 0.25 * n) * 6.28318530717958647693);
  const float z = x * x;
  float s = __builtin_fmaf(z, 1.0f / 362880.0f, -1.0f / 5040.0f);
  s = __builtin_fmaf(z, s, 1.0f / 120.0f);
  s = __builtin_fmaf(z, s, -1.0f / 6.0f);
  s = __builtin_fmaf(x * z, s, x);
  float c = __builtin_fmaf(z, -1.0f / 3628800.0f, 1.0f / 40320.0f);
  c = __builtin_fmaf(z, c, -1.0f / 720.0f);
  c = __builtin_fmaf(z, c, 1.0f / 24.0f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.0f);
  const int quarter = (int)n & 3;
  const float a = quarter & 1 ? s : c, b = quarter & 1 ? c : s;
  return make_float2(quarter == 1 || quarter == 2 ? -a : a, quarter >= 2 ? -b : b);
}

// (cos, sin) of a row's pair. An infinite or NaN position gives NaN.
__device__ __forceinline__ float2 rotation_of(const AxTable& t, int64_t row, int pair) {
  const int axis = min(max(t.axis[pair], 0), t.axes - 1);
  const double turns = position_of(t, row, axis) * t.inv_freq[pair] * 0.15915494309189533577;
  return cos_sin_turns(turns);
}

template <typename T, int N>
struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Run {
  T e[N];
};

template <int DT>
__device__ __forceinline__ float widen(uint32_t u) {
  if constexpr (DT == kF32) return __uint_as_float(u);
  else if constexpr (DT == kF16) return h2f((uint16_t)u);
  else return bf2f((uint16_t)u);
}
template <int DT, typename T>
__device__ __forceinline__ T narrow(float f) {
  if constexpr (DT == kF32) return __float_as_uint(f);
  else if constexpr (DT == kF16) return f2h(f);
  else return f2bf(f);
}

// ADJ: adjacent pairs. V: pairs of a chunk; C: chunks of a lane.
template <int DT, bool ADJ, int V, int C>
__global__ __launch_bounds__(kAxThreads)
void axial_rope_kernel(AxRopeParams p) {
  using T = std::conditional_t<DT == kF32, uint32_t, uint16_t>;
  __shared__ float2 angle[kAxPairs];
  const int pairs = p.table.pairs;
  const int64_t row = blockIdx.x;
  for (int i = threadIdx.x; i < pairs; i += kAxThreads) angle[i] = rotation_of(p.table, row, i);
  __syncthreads();

  const int lanes = p.lanes, lane = threadIdx.x & (lanes - 1);
  const int per_pass = kAxThreads / lanes, heads = p.heads[0] + p.heads[1];
  const int turned = pairs / V, chunks = p.dim / (2 * V);
  // (All lanes of a head run the same passes.)
  for (int head = threadIdx.x / lanes; head < heads; head += per_pass) {
    const int w = head >= p.heads[0] ? 1 : 0, h = head - (w ? p.heads[0] : 0);
    const T* src = reinterpret_cast<const T*>(p.x[w]) + row * p.in_row[w] + h * p.in_head[w];
    T* dst = reinterpret_cast<T*>(p.out[w]) + row * p.out_row[w] + h * p.out_head[w];
    float a[C][V], b[C][V];
    int at[C], bt[C];
    float ss = 0.0f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int ch = lane + c * lanes;
      const bool on = ch < chunks;
      const bool split_halves = !ADJ && ch < turned;
      at[c] = split_halves ? ch * V : ch < turned ? 2 * V * ch : 2 * pairs + (ch - turned) * 2 * V;
      bt[c] = at[c] + (split_halves ? pairs : V);
      Run<T, V> ra{}, rb{};
      if (on) {
        ra = *reinterpret_cast<const Run<T, V>*>(src + at[c]);
        rb = *reinterpret_cast<const Run<T, V>*>(src + bt[c]);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        a[c][i] = widen<DT>(ra.e[i]);
        b[c][i] = widen<DT>(rb.e[i]);
        ss = __builtin_fmaf(a[c][i], a[c][i], ss);
        ss = __builtin_fmaf(b[c][i], b[c][i], ss);
      }
    }
    const float* gain = p.gain[w];
    if (gain) {
      for (int off = lanes >> 1; off >= 1; off >>= 1) ss = ss + __shfl_xor(ss, off, 64);
      const float inv = 1.0f / __builtin_sqrtf(ss * p.inv_dim + p.eps);
#pragma unroll
      for (int c = 0; c < C; ++c) {
        if (lane + c * lanes < chunks) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            a[c][i] = a[c][i] * inv * gain[at[c] + i];
            b[c][i] = b[c][i] * inv * gain[bt[c] + i];
          }
        }
      }
    }
#pragma unroll
    for (int c = 0; c < C; ++c) {
      const int ch = lane + c * lanes;
      if (ch >= chunks) continue;
      Run<T, V> ra, rb;
      if (ch < turned) {
        const float2* rot = angle + ch * V;
        if constexpr (ADJ) {
          // The 2 V channels a[0..V), b[0..V) hold pairs (2 i, 2 i + 1).
          float v[2 * V];
#pragma unroll
          for (int i = 0; i < V; ++i) {
            v[i] = a[c][i];
            v[V + i] = b[c][i];
          }
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 cs = rot[i];
            const float u = v[2 * i], t = v[2 * i + 1];
            v[2 * i] = __builtin_fmaf(-t, cs.y, u * cs.x);
            v[2 * i + 1] = __builtin_fmaf(u, cs.y, t * cs.x);
          }
#pragma unroll
          for (int i = 0; i < V; ++i) {
            ra.e[i] = narrow<DT, T>(v[i]);
            rb.e[i] = narrow<DT, T>(v[V + i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float2 cs = rot[i];
            const float u = a[c][i], t = b[c][i];
            ra.e[i] = narrow<DT, T>(__builtin_fmaf(-t, cs.y, u * cs.x));
            rb.e[i] = narrow<DT, T>(__builtin_fmaf(u, cs.y, t * cs.x));
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          ra.e[i] = narrow<DT, T>(a[c][i]);
          rb.e[i] = narrow<DT, T>(b[c][i]);
        }
      }
      *reinterpret_cast<Run<T, V>*>(dst + at[c]) = ra;
      *reinterpret_cast<Run<T, V>*>(dst + bt[c]) = rb;
    }
  }
}

template <int DT, bool ADJ>
static int launch_axial(const AxRopeParams& p, int v, unsigned grid, hipStream_t s) {
  switch (v) {
    case 8: hipLaunchKernelGGL((axial_rope_kernel<DT, ADJ, 8, 1>), dim3(grid), dim3(kAxThreads), 0, s, p); break;
    case 4: hipLaunchKernelGGL((axial_rope_kernel<DT, ADJ, 4, 1>), dim3(grid), dim3(kAxThreads), 0, s, p); break;
    case 2: hipLaunchKernelGGL((axial_rope_kernel<DT, ADJ, 2, 1>), dim3(grid), dim3(kAxThreads), 0, s, p); break;
    default: hipLaunchKernelGGL((axial_rope_kernel<DT, ADJ, 1, 2>), dim3(grid), dim3(kAxThreads), 0, s, p); break;
  }
  return launch_status("w8a8_axial_rope");
}

// One pair of one row per thread.
template <int FQ>
__global__ __launch_bounds__(kAxThreads)
void axial_freqs_kernel(AxTable t, int64_t rows, int layout, void* freqs) {
  const int64_t i = (int64_t)blockIdx.x * kAxThreads + threadIdx.x;
  if (i >= rows * t.pairs) return;
  const int64_t row = i / t.pairs;
  const int pair = (int)(i - row * t.pairs);
  const float2 cs = rotation_of(t, row, pair);
  using T = std::conditional_t<FQ == kF32, uint32_t, uint16_t>;
  const Run<T, 2> first{{narrow<FQ, T>(cs.x), narrow<FQ, T>(-cs.y)}};
  const Run<T, 2> matrix_second{{narrow<FQ, T>(cs.y), narrow<FQ, T>(cs.x)}};
  const Run<T, 2> pairs_second{{narrow<FQ, T>(cs.x), narrow<FQ, T>(cs.y)}};
  Run<T, 2>* out = reinterpret_cast<Run<T, 2>*>(freqs) + row * 2 * t.pairs;
  if (layout == W8A8_ROPE_MATRICES) {
    out[2 * pair] = first;
    out[2 * pair + 1] = matrix_second;
  } else {
    out[pair] = first;
    out[t.pairs + pair] = pairs_second;
  }
}

// A [rows, heads, dim] view's memory.
struct HeadsView {
  const void* at;
  int64_t row, head, rows, heads, dim;   // (bytes, numbers of rows and heads, bytes)
};

static HeadsView view_of(const void* at, const int64_t* st, int64_t rows, int64_t heads, int64_t dim, int es) {
  return {at, st[0] * es, st[1] * es, rows, heads, dim * es};
}

// Whether two such views share no byte, as far as spans, rows (or heads, where they
// are the outer dimension) and heads between each other's tell.
static bool views_apart(const HeadsView& a, const HeadsView& b) {
  auto span = [](const HeadsView& v) { return (v.rows - 1) * v.row + (v.heads - 1) * v.head + v.dim; };
  auto by_rows = [&](const HeadsView& v) { return RowsOf{v.at, v.row, (v.heads - 1) * v.head + v.dim, span(v)}; };
  auto by_heads = [&](const HeadsView& v) { return RowsOf{v.at, v.head, (v.rows - 1) * v.row + v.dim, span(v)}; };
  // The inner stride alone, where the outer is a multiple of it; 0 (tells nothing) else.
  auto inner = [&](const HeadsView& v) {
    const int64_t s = v.row < v.head ? v.row : v.head;
    return RowsOf{v.at, s > 0 && v.row % s == 0 && v.head % s == 0 ? s : 0, v.dim, span(v)};
  };
  return apart(by_rows(a), by_rows(b)) || apart(by_heads(a), by_heads(b)) || apart(inner(a), inner(b));
}

}  // namespace w8a8

extern "C" int w8a8_axial_rope(const W8A8AxialRopeArgs* a) {
  using namespace w8a8;
  W8A8_REQUIRE(a != nullptr, "w8a8_axial_rope: null args");
  W8A8_REQUIRE(a->struct_size == sizeof(W8A8AxialRopeArgs), "w8a8_axial_rope: struct_size %u != %zu", a->struct_size,
               sizeof(W8A8AxialRopeArgs));
  W8A8_REQUIRE(a->dtype == W8A8_F16 || a->dtype == W8A8_BF16 || a->dtype == W8A8_F32,
               "w8a8_axial_rope: dtype %d not F16/BF16/F32", a->dtype);
  W8A8_REQUIRE(a->dim >= 2 && a->dim <= 256 && a->dim % 2 == 0, "w8a8_axial_rope: dim %d must be even in [2, 256]",
               a->dim);
  W8A8_REQUIRE(a->pairs >= 1 && a->pairs <= a->dim / 2, "w8a8_axial_rope: pairs %d outside [1, dim / 2]", a->pairs);
  W8A8_REQUIRE(a->axes >= 1 && a->axes <= 16, "w8a8_axial_rope: axes %d outside [1, 16]", a->axes);
  W8A8_REQUIRE(a->pairing == W8A8_ROPE_HALF || a->pairing == W8A8_ROPE_ADJACENT, "w8a8_axial_rope: unknown pairing");
  W8A8_REQUIRE(a->pos_type >= W8A8_POS_I32 && a->pos_type <= W8A8_POS_F32, "w8a8_axial_rope: unknown pos_type");
  W8A8_REQUIRE(a->rows >= 0 && a->rows < ((int64_t)1 << 31) && a->q_heads >= 1 && a->q_heads <= 4096 &&
                   a->k_heads >= 0 && a->k_heads <= 4096,
               "w8a8_axial_rope: rows or heads out of range");
  W8A8_REQUIRE((a->k != nullptr) == (a->k_out != nullptr) && (a->rows == 0 || (a->k != nullptr) == (a->k_heads > 0)),
               "w8a8_axial_rope: k, k_out and k_heads go together");
  W8A8_REQUIRE((a->q_gain != nullptr) == (a->k_gain != nullptr) || (a->k_heads == 0 && !a->k_gain),
               "w8a8_axial_rope: q_gain and k_gain go together");
  if (a->rows == 0) return W8A8_OK;
  const int es = elem_size(a->dtype);
  W8A8_REQUIRE(a->q && a->q_out && a->positions && a->inv_freq && a->axis, "w8a8_axial_rope: null buffer");
  const int pes = a->pos_type == W8A8_POS_I64 ? 8 : 4;
  W8A8_REQUIRE((uintptr_t)a->positions % pes == 0 && (uintptr_t)a->inv_freq % 8 == 0 && (uintptr_t)a->axis % 4 == 0 &&
                   (uintptr_t)a->q_gain % 4 == 0 && (uintptr_t)a->k_gain % 4 == 0,
               "w8a8_axial_rope: positions, inv_freq, axis or a gain misaligned");
  W8A8_REQUIRE(a->pos_strides[0] >= 0 && a->pos_strides[1] >= 0, "w8a8_axial_rope: negative position stride");
  const void* in[2] = {a->q, a->k};
  void* out[2] = {a->q_out, a->k_out};
  const int64_t* ist[2] = {a->q_strides, a->k_strides};
  const int64_t* ost[2] = {a->q_out_strides, a->k_out_strides};
  const int heads[2] = {a->q_heads, a->k_heads};
  // The widest chunk that the sizes, strides and addresses allow.
  int v = 8;
  while (v > 1 && (a->pairs % v || (a->dim - 2 * a->pairs) % (2 * v))) v >>= 1;
  AxRopeParams p{};
  HeadsView vin[2] = {}, vout[2] = {};
  for (int w = 0; w < 2; ++w) {
    if (!heads[w]) continue;
    W8A8_REQUIRE((uintptr_t)in[w] % es == 0 && (uintptr_t)out[w] % es == 0, "w8a8_axial_rope: misaligned tensor");
    W8A8_REQUIRE(ist[w][0] >= 0 && ist[w][1] >= 0 && ost[w][0] >= 0 && ost[w][1] >= 0,
                 "w8a8_axial_rope: negative stride");
    // Rows and heads of an output must not share memory: one stride steps over
    // the other's whole extent.
    const int64_t d = a->dim, r = ost[w][0], h = ost[w][1];
    const bool rows_outer = (heads[w] == 1 || h >= d) && (a->rows == 1 || r >= (heads[w] - 1) * h + d);
    const bool heads_outer = (a->rows == 1 || r >= d) && (heads[w] == 1 || h >= (a->rows - 1) * r + d);
    W8A8_REQUIRE(rows_outer || heads_outer, "w8a8_axial_rope: an output's heads overlap");
    const int64_t bits = (int64_t)((uintptr_t)in[w] | (uintptr_t)out[w]) |
                         ((ist[w][0] | ist[w][1] | ost[w][0] | ost[w][1]) * es);
    while (v > 1 && bits % (v * es < 16 ? v * es : 16)) v >>= 1;
    p.x[w] = in[w];
    p.out[w] = out[w];
    p.in_row[w] = ist[w][0];
    p.in_head[w] = ist[w][1];
    p.out_row[w] = ost[w][0];
    p.out_head[w] = ost[w][1];
    p.heads[w] = heads[w];
    vin[w] = view_of(in[w], ist[w], a->rows, heads[w], d, es);
    vout[w] = view_of(out[w], ost[w], a->rows, heads[w], d, es);
  }
  for (int o = 0; o < 2; ++o) {
    if (!heads[o]) continue;
    for (int i = 0; i < 2; ++i) {
      const bool same = i == o && out[o] == in[i] && ost[o][0] == ist[i][0] && ost[o][1] == ist[i][1];
      W8A8_REQUIRE(!heads[i] || same || views_apart(vout[o], vin[i]), "w8a8_axial_rope: an output overlaps an input");
    }
  }
  W8A8_REQUIRE(!heads[1] || views_apart(vout[0], vout[1]), "w8a8_axial_rope: q_out and k_out overlap");
  p.gain[0] = a->q_gain;
  p.gain[1] = a->k_gain;
  p.table = AxTable{a->positions, a->pos_strides[0], a->pos_strides[1], a->pos_type, a->pairs, a->axes, a->inv_freq, a->axis};
  p.dim = a->dim;
  p.eps = a->eps;
  p.inv_dim = (float)(1.0 / (double)a->dim);
  const int chunks = a->dim / (2 * v), lane_chunks = v == 1 ? 2 : 1;
  p.lanes = 1;
  while (p.lanes * lane_chunks < chunks) p.lanes *= 2;
  W8A8_REQUIRE(a->rows * kAxThreads < ((int64_t)1 << 32), "w8a8_axial_rope: too many rows for one launch");
  hipStream_t s = reinterpret_cast<hipStream_t>(a->stream);
  const bool adj = a->pairing == W8A8_ROPE_ADJACENT;
  const unsigned grid = (unsigned)a->rows;
  switch (a->dtype) {
    case W8A8_F16: return adj ? launch_axial<kF16, true>(p, v, grid, s) : launch_axial<kF16, false>(p, v, grid, s);
    case W8A8_BF16: return adj ? launch_axial<kBF16, true>(p, v, grid, s) : launch_axial<kBF16, false>(p, v, grid, s);
    default: return adj ? launch_axial<kF32, true>(p, v, grid, s) : launch_axial<kF32, false>(p, v, grid, s);
  }
}

extern "C" int w8a8_axial_freqs(const W8A8AxialFreqsArgs* a) {
  using namespace w8a8;
  W8A8_REQUIRE(a != nullptr, "w8a8_axial_freqs: null args");
  W8A8_REQUIRE(a->struct_size == sizeof(W8A8AxialFreqsArgs), "w8a8_axial_freqs: struct_size %u != %zu",
               a->struct_size, sizeof(W8A8AxialFreqsArgs));
  W8A8_REQUIRE(a->freq_dtype == W8A8_F16 || a->freq_dtype == W8A8_F32, "w8a8_axial_freqs: freq_dtype %d not F16/F32",
               a->freq_dtype);
  W8A8_REQUIRE(a->freq_layout == W8A8_ROPE_MATRICES || a->freq_layout == W8A8_ROPE_PAIRS,
               "w8a8_axial_freqs: unknown freq_layout");
  W8A8_REQUIRE(a->pos_type >= W8A8_POS_I32 && a->pos_type <= W8A8_POS_F32, "w8a8_axial_freqs: unknown pos_type");
  W8A8_REQUIRE(a->pairs >= 1 && a->pairs <= 128 && a->axes >= 1 && a->axes <= 16 && a->rows >= 0 &&
                   a->rows < ((int64_t)1 << 31),
               "w8a8_axial_freqs: rows, pairs or axes out of range");
  if (a->rows == 0) return W8A8_OK;
  const int pes = a->pos_type == W8A8_POS_I64 ? 8 : 4;
  W8A8_REQUIRE(a->positions && a->inv_freq && a->axis && a->freqs && aligned16(a->freqs) &&
                   (uintptr_t)a->positions % pes == 0 && (uintptr_t)a->inv_freq % 8 == 0 && (uintptr_t)a->axis % 4 == 0,
               "w8a8_axial_freqs: null or misaligned buffer");
  W8A8_REQUIRE(a->pos_strides[0] >= 0 && a->pos_strides[1] >= 0, "w8a8_axial_freqs: negative position stride");
  const int64_t blocks = (a->rows * a->pairs + kAxThreads - 1) / kAxThreads;
  W8A8_REQUIRE(blocks * kAxThreads < ((int64_t)1 << 32), "w8a8_axial_freqs: too many rows for one launch");
  const AxTable t{a->positions, a->pos_strides[0], a->pos_strides[1], a->pos_type, a->pairs, a->axes, a->inv_freq, a->axis};
  hipStream_t s = reinterpret_cast<hipStream_t>(a->stream);
  if (a->freq_dtype == W8A8_F32)
    hipLaunchKernelGGL((axial_freqs_kernel<kF32>), dim3((unsigned)blocks), dim3(kAxThreads), 0, s, t, a->rows,
                       a->freq_layout, a->freqs);
  else
    hipLaunchKernelGGL((axial_freqs_kernel<kF16>), dim3((unsigned)blocks), dim3(kAxThreads), 0, s, t, a->rows,
                       a->freq_layout, a->freqs);
  return launch_status("w8a8_axial_freqs");
}
