// Element access shared by the row-wise operators (scan, norm): V consecutive
// elements of a 16-bit or fp32 row as one load or store, kept packed until
// they are used.
#pragma once

#include "gdn_fwd_kernel.h"

namespace gdn {
namespace rowio {

template <int BYTES>
struct Words;
template <>
struct Words<2> {
  typedef uint16_t T;
};
template <>
struct Words<4> {
  typedef uint32_t T;
};
template <>
struct Words<8> {
  typedef uint2 T;
};
template <>
struct Words<16> {
  typedef uint4 T;
};
struct __attribute__((aligned(16))) Quads2 {
  uint4 a, b;
};
template <>
struct Words<32> {
  typedef Quads2 T;
};

template <typename E>
__device__ __forceinline__ float to_f32(E e);
template <>
__device__ __forceinline__ float to_f32<f16>(f16 e) {
  return (float)e;
}
template <>
__device__ __forceinline__ float to_f32<bf16_t>(bf16_t e) {
  return bf16_bits_to_float(e.bits);
}
template <>
__device__ __forceinline__ float to_f32<float>(float e) {
  return e;
}
template <typename E>
__device__ __forceinline__ E from_f32(float x);
template <>
__device__ __forceinline__ f16 from_f32<f16>(float x) {
  return (f16)x;
}
template <>
__device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) {
  return bf16_t{float_to_bf16_bits(x)};
}
template <>
__device__ __forceinline__ float from_f32<float>(float x) {
  return x;
}

// V elements of type E, packed as they lie in memory.
template <typename E, int V>
struct Pack {
  typedef typename Words<V * sizeof(E)>::T Raw;
  Raw raw;
  __device__ __forceinline__ void load(const E* p) { raw = *reinterpret_cast<const Raw*>(p); }
  __device__ __forceinline__ void store(E* p) const { *reinterpret_cast<Raw*>(p) = raw; }
  __device__ __forceinline__ void zero() { raw = Raw{}; }
  // From here on the elements are unpacked again where they are used (the
  // compiler would keep them unpacked, in twice the registers).
  __device__ __forceinline__ void repack() {
    uint32_t w[(sizeof(Raw) + 3) / 4] = {};
    __builtin_memcpy(w, &raw, sizeof(Raw));
#pragma unroll
    for (auto& x : w) asm volatile("" : "+v"(x));
    __builtin_memcpy(&raw, w, sizeof(Raw));
  }
  __device__ __forceinline__ float get(int i) const {
    E e[V];
    __builtin_memcpy(e, &raw, sizeof(raw));
    return to_f32<E>(e[i]);
  }
  __device__ __forceinline__ void set(const float* x) {
    E e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<E>(x[i]);
    __builtin_memcpy(&raw, e, sizeof(raw));
  }
};

}  // namespace rowio

// gdn_fwd_kernel.h's dtype codes on the host.
inline bool scan_dtype_ok(int dt) { return dt == GDN_DTYPE_F32 || dt == GDN_DTYPE_F16 || dt == GDN_DTYPE_BF16; }
// Whether one launch holds that many workgroups: its threads are counted in 32
// bits, and a launch of more runs what is left of them without an error.
inline bool grid_fits(int64_t blocks, int threads) { return blocks * threads <= 0xffffffffLL; }
inline int dtype_bytes(int dt) { return dt == GDN_DTYPE_F32 ? 4 : 2; }

}  // namespace gdn
