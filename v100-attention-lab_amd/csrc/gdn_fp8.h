// Rounding to e4m3 with a scale, shared by the norm's 8-bit form, the quantisers
// and the 8-bit cache.
#pragma once

#include "gdn_row_io.h"

namespace gdn {
namespace fp8 {

constexpr float kFp8Max = 448.f;     // largest finite e4m3

// The larger of two; NaN where either is.
__device__ __forceinline__ float nan_max(float a, float b) { return a != a || a > b ? a : b; }
template <int W>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = W / 2; o >= 1; o >>= 1) v = nan_max(v, __shfl_xor(v, o, 64));
  return v;
}

// 4 values as e4m3 bytes, rounded to the nearest even; values are clamped to
// the type's range first (NaN stays NaN).
__device__ __forceinline__ float clamp_fp8(float v) {
  return v != v ? v : fminf(fmaxf(v, -kFp8Max), kFp8Max);
}
__device__ __forceinline__ uint32_t pack_fp8(float a, float b, float c, float d) {
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_fp8(a), clamp_fp8(b), 0, false);
  r = __builtin_amdgcn_cvt_pk_fp8_f32(clamp_fp8(c), clamp_fp8(d), r, true);
  return (uint32_t)r;
}
template <int V>
__device__ __forceinline__ void store_fp8(uint8_t* q, const float (&v)[V]) {
  if constexpr (V == 8) {
    *reinterpret_cast<uint2*>(q) =
        make_uint2(pack_fp8(v[0], v[1], v[2], v[3]), pack_fp8(v[4], v[5], v[6], v[7]));
  } else {
    static_assert(V == 1, "");
    *q = (uint8_t)(pack_fp8(v[0], 0.f, 0.f, 0.f) & 0xffu);
  }
}
// y / scale, rounded once, by the scale that is stored: the product with 1 / scale
// (one unit off at most), corrected by its remainder.  `up` keeps 1 / scale finite
// for the smallest scales.  A scale of 0 (a group of zeros) gives zeros, of infinity
// zeros and inf / inf.
struct Quant {
  float up, s, inv;
  __device__ __forceinline__ explicit Quant(float scale) {
    up = scale < 0x1p-100f ? 0x1p100f : 1.f;
    s = scale < __builtin_inff() ? scale * up : 0.f;
    inv = scale == 0.f ? 0.f : __builtin_amdgcn_rcpf(scale * up);
  }
  __device__ __forceinline__ float operator()(float y) const {
    y *= up;
    const float q = y * inv;
    return __builtin_fmaf(__builtin_fmaf(-q, s, y), inv, q);
  }
};

}  // namespace fp8
}  // namespace gdn
