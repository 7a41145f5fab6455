// The normalize-and-modulate step shared by the norm kernels.
#pragma once

#include "w8a8_device.h"

namespace w8a8 {

__device__ __forceinline__ void load16_f32(const float* p, float (&v)[16]) {
  const float4* q = reinterpret_cast<const float4*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float4 t = q[i];
    v[4 * i] = t.x; v[4 * i + 1] = t.y; v[4 * i + 2] = t.z; v[4 * i + 3] = t.w;
  }
}

// Table flags of a kernel: kGain (weight present), kMod (shift/scale
// tables present), kAnyTables (decide per call from the pointers).
enum NormTables { kGain = 1, kMod = 2, kAnyTables = 4 };

// v: x on entry; on return the normalized, modulated value rounded to DT
// (as fp32; times 1/16 when SCALED), with its storage bits packed in bits.
template <int DT, int TB, bool SCALED>
__device__ __forceinline__ void modulate16(float (&v)[16], uint32_t (&bits)[8], float inv, const float* w,
                                           const float* sh, const float* sc, int64_t c0) {
  const bool gain = (TB & kGain) || ((TB & kAnyTables) && w);
  const bool mod = (TB & kMod) || ((TB & kAnyTables) && sh);
  float wv[16], shv[16], scv[16];
  if (gain) load16_f32(w + c0, wv);
  if (mod) {
    load16_f32(sc + c0, scv);
    load16_f32(sh + c0, shv);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    float t = DT == kF16 ? mul_mix(v[i], inv) : v[i] * inv;
    if (gain) t = t * wv[i];
    if (mod) {
      const float f = 1.0f + scv[i];
      t = t * f;
      t = t + shv[i];
    }
    v[i] = t;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    if constexpr (DT == kF16) {
      bits[i] = f2h2_of_f32(v[2 * i], v[2 * i + 1]);
      v[2 * i] = h2f((uint16_t)(bits[i] & 0xffffu));
      v[2 * i + 1] = h2f((uint16_t)(bits[i] >> 16));
    } else {
      const uint16_t lo = f2bf(v[2 * i]), hi = f2bf(v[2 * i + 1]);
      bits[i] = (uint32_t)lo | ((uint32_t)hi << 16);
      v[2 * i] = bf2f(lo);
      v[2 * i + 1] = bf2f(hi);
    }
  }
  if constexpr (SCALED) scale16(v);
}

}  // namespace w8a8
