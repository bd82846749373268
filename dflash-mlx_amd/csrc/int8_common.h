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

// How a product runs: as a stream of the weight (int8.hip), or by tiles of 256 x 256 or
// 128 x 128 with K in so many splits (int8_prompt.hip).
struct PlanI8 {
  enum Kind { kStream, kNarrow, kWide } kind;
  int splits;
};

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
  PlanI8 plan;
  void* workspace;  // where the splits' sums go
  const uint16_t* raw;  // a single row that is not quantised yet (then not x and sx)
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
struct Out<uint16_t> {  // bf16, by the hardware's conversion (to nearest, ties to even)
  static __device__ void store4(uint16_t* p, const float (&v)[4]) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    *reinterpret_cast<u32x2_e2*>(p) =
        u32x2{__builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[0], v[1]}, bf16x2)),
              __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2], v[3]}, bf16x2))};
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

// 4 neighbouring output columns from col + 4 g on of a lane's row, at `off` (4 g
// counted) from rows; WHOLE: all of them are there.
template <typename T, bool WHOLE>
__device__ __forceinline__ void store_cols(const GemmI8& p, T* rows, uint32_t off, int col, int g, const float (&v)[4]) {
  T* o = rows + col + off;
  const int left = p.cols - col - 4 * g;
  if (WHOLE || left >= 4) {
    Out<T>::store4(o, v);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < left) o[e] = Out<T>::one(v[e]);
  }
}

// g / (1 + e^-g) with the hardware's exp2 and reciprocal, each within an ulp: what the
// rounding of -g log2(e) and of the constant leave out of the exponent (2^-24 of it each, a
// step of the result and more from |g| = 2 on) is added back while the power is finite.
// A quarter of the instructions of expf and a division.
__device__ __forceinline__ float silu(float g) {
  const float hi = -1.44269504f * g;
  const float lo = fmaf(-g, 1.92596303e-8f, fmaf(-g, 1.44269504f, -hi));  // log2(e) = 1.44269502... + 1.926e-8
  float e = __builtin_amdgcn_exp2f(hi);
  if (fabsf(hi) < 120.f) e = fmaf(e, 0.693147181f * lo, e);
  return g * __builtin_amdgcn_rcpf(1.f + e);
}

// Lane (r16, g) of a 16 x 16 tile of sums holds channels 4g .. 4g + 3 of the tile for
// row r16.  The scales of its channels of tile t (the last tile's, if there is none).
__device__ __forceinline__ f32x4 tile_scales(const GemmI8& p, int t, int g) {
  return *reinterpret_cast<const f32x4*>(p.sw + 16 * min(t, p.tiles - 1) + 4 * g);
}

// The outputs of the channel tiles t and t + 1 (a gate and its up where GATED; t is even
// and there) for the lane's row, whose column 4 g is at rows + off, with the tiles' and the
// row's scales.
template <typename T, bool GATED, bool WHOLE = false>
__device__ __forceinline__ void store_pair(const GemmI8& p, int t, int g, T* rows, uint32_t off, const i32x4& a, const i32x4& b,
                                           const f32x4& sa, const f32x4& sb, float sx) {
  float v[4], u[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (float)a[e] * sa[e] * sx, u[e] = (float)b[e] * sb[e] * sx;
  if (GATED) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = silu(v[e]) * u[e];
    store_cols<T, WHOLE>(p, rows, off, 8 * t, g, v);
  } else {
    store_cols<T, WHOLE>(p, rows, off, 16 * t, g, v);
    if (WHOLE || t + 1 < p.tiles) store_cols<T, WHOLE>(p, rows, off, 16 * (t + 1), g, u);
  }
}

// Products by tiles (int8_prompt.hip).
template <typename T, bool GATED>
hipError_t launch_prompt_i8(const GemmI8& p, hipStream_t s);

}  // namespace dflash
