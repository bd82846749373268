// What the kernels of 8-bit products share: their parameters and how a tile of sums
// becomes outputs (formats and formulas: include/dflash_int8.h).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "device_common.h"
#include "dflash_int8.h"
#include "host_common.h"

namespace dflash {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x2 u32x2_e2 __attribute__((aligned(2)));  // vectors at any element of 16 or 32 bits
typedef f32x4 f32x4_e4 __attribute__((aligned(4)));

inline int k_steps(int K) { return 2 * (int)ceil_div(K, 128); }
inline int channel_tiles(int N, int gated) {
  return gated ? 2 * (int)ceil_div(N / 2, 16) : (int)ceil_div(N, 16);
}

struct GemmI8 {
  const uint8_t* x;
  int64_t xs;
  const float* sx;
  const u32x4* w;
  const float* sw;
  void* out;
  int64_t os;
  int M, cols;  // output rows and columns
  int K, k_steps, tiles;
};

template <typename T>
struct Out;
template <>
struct Out<float> {
  static __device__ void store4(float* p, const float (&v)[4]) {
    *reinterpret_cast<f32x4_e4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
  }
  static __device__ float one(float v) { return v; }
};
template <>
struct Out<uint16_t> {  // bf16
  static __device__ void store4(uint16_t* p, const float (&v)[4]) {
    *reinterpret_cast<u32x2_e2*>(p) = u32x2{f32_to_bf16_rne(v[0]) | (uint32_t)f32_to_bf16_rne(v[1]) << 16,
                                            f32_to_bf16_rne(v[2]) | (uint32_t)f32_to_bf16_rne(v[3]) << 16};
  }
  static __device__ uint16_t one(float v) { return f32_to_bf16_rne(v); }
};
template <>
struct Out<_Float16> {
  static __device__ void store4(_Float16* p, const float (&v)[4]) {
    typedef _Float16 h4 __attribute__((ext_vector_type(4), aligned(2)));
    *reinterpret_cast<h4*>(p) = h4{(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  }
  static __device__ _Float16 one(float v) { return (_Float16)v; }
};

// 4 neighbouring output columns from col on of row m (those below cols).
template <typename T>
__device__ __forceinline__ void store_cols(const GemmI8& p, int m, int col, const float (&v)[4]) {
  T* o = static_cast<T*>(p.out) + (int64_t)m * p.os + col;
  if (col + 4 <= p.cols) {
    Out<T>::store4(o, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (col + e < p.cols) o[e] = Out<T>::one(v[e]);
  }
}

__device__ __forceinline__ float silu(float g) { return g / (1.f + expf(-g)); }

// Lane (r16, g) of a 16 x 16 tile of sums holds channels 4g .. 4g + 3 of the tile for
// row r16: the outputs of the channel tiles t and t + 1 (a gate and its up where
// GATED) for row m.
template <typename T, bool GATED>
__device__ __forceinline__ void store_pair(const GemmI8& p, int t, int g, int m, const i32x4& a, const i32x4& b,
                                           float sx) {
  const f32x4 sa = *reinterpret_cast<const f32x4*>(p.sw + 16 * t + 4 * g);
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)a[e] * sa[e] * sx;
  if (!GATED) store_cols<T>(p, m, 16 * t + 4 * g, v);
  if (t + 1 >= p.tiles) return;
  const f32x4 sb = *reinterpret_cast<const f32x4*>(p.sw + 16 * (t + 1) + 4 * g);
  if (GATED) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = silu(v[e]) * ((float)b[e] * sb[e] * sx);
    store_cols<T>(p, m, 8 * t + 4 * g, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = (float)b[e] * sb[e] * sx;
    store_cols<T>(p, m, 16 * (t + 1) + 4 * g, v);
  }
}

// Products of many rows (int8_prompt.hip).
template <typename T, bool GATED>
hipError_t launch_prompt_i8(const GemmI8& p, hipStream_t s);

}  // namespace dflash
