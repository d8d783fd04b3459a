// What the kernels of rotary positions share (rope.hip, norm_rope.hip): a pair's
// cosine and sine, and values in and out of 32 bits.
#pragma once

#include "common.hpp"

namespace svdmlp {

__device__ __forceinline__ void turn(int64_t pos, double inv_freq, float scale, float* c, float* s) {
  double t = (double)pos * inv_freq * 0.15915494309189533577;  // turns
  t = 4.0 * (t - rint(t));                                     // quarter turns, -2..2
  const double q = rint(t);
  float sn, cs;
  sincospif((float)(t - q) * 0.5f, &sn, &cs);
  const int k = (int)q & 3;
  const float a = (k & 1) ? sn : cs, b = (k & 1) ? cs : sn;
  *c = scale * ((k == 1 || k == 2) ? -a : a);
  *s = scale * ((k & 2) ? -b : b);
}

template <bool BF16>
__device__ __forceinline__ float ld1(const void* p, int64_t i) {
  if constexpr (BF16) return bf16_bits_to_f32(static_cast<const uint16_t*>(p)[i]);
  else return static_cast<const float*>(p)[i];
}
template <bool BF16>
__device__ __forceinline__ void st1(void* p, int64_t i, float v) {
  if constexpr (BF16) static_cast<uint16_t*>(p)[i] = (uint16_t)f32_to_bf16_bits(v);
  else static_cast<float*>(p)[i] = v;
}

// One 16-byte piece as 4 or 8 floats and back.
template <bool BF16>
__device__ __forceinline__ void unpack(u32x4 v, float* f) {
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (BF16) {
      f[2 * w] = __uint_as_float(v[w] << 16);
      f[2 * w + 1] = __uint_as_float(v[w] & 0xffff0000u);
    } else {
      f[w] = __uint_as_float(v[w]);
    }
  }
}
template <bool BF16>
__device__ __forceinline__ u32x4 pack(const float* f) {
  u32x4 v;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    if constexpr (BF16) v[w] = pack_bf16x2(f[2 * w], f[2 * w + 1]);
    else v[w] = __float_as_uint(f[w]);
  }
  return v;
}

}  // namespace svdmlp
