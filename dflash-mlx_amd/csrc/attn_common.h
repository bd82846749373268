// Device helpers of the attention kernels: of the bf16 cache's (model_ops.hip) and of
// the 8-bit cache's (kv8.hip, attn_q8.hip).  Rotation, norm_rotate and the sums and
// roundings that they use are the bf16 cache's alone.
#pragma once

#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "device_common.h"

namespace dflash {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ u32x4 ld16(const void* p) { return *reinterpret_cast<const u32x4*>(p); }

__device__ __forceinline__ void unpack8(u32x4 w, float* f) {
  f[0] = bf16_lo(w.x); f[1] = bf16_hi(w.x);
  f[2] = bf16_lo(w.y); f[3] = bf16_hi(w.y);
  f[4] = bf16_lo(w.z); f[5] = bf16_hi(w.z);
  f[6] = bf16_lo(w.w); f[7] = bf16_hi(w.w);
}

__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return (uint32_t)f32_to_bf16_rne(a) | ((uint32_t)f32_to_bf16_rne(b) << 16);
}

__device__ __forceinline__ u32x4 pack8(const float* f) {
  return u32x4{pack2(f[0], f[1]), pack2(f[2], f[3]), pack2(f[4], f[5]), pack2(f[6], f[7])};
}

__device__ __forceinline__ float bf16_round(float x) { return bf16_bits_to_f32(f32_to_bf16_rne(x)); }

__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

constexpr int kHD = 128;  // attention head dim supported by these kernels

// pos * base^(-2i/rot) reduced to [0, 2*pi), computed in fp64.
__device__ __forceinline__ float rope_angle(int pos, int i, int rot, double log2_base) {
  const double inv_freq = exp2(-(double)(2 * i) / (double)rot * log2_base);
  const double a = (double)pos * inv_freq;
  const double two_pi = 6.283185307179586476925286766559;
  return (float)(a - two_pi * floor(a / two_pi));
}

// Rotation of a lane's features 2l and 2l + 1 at position pos (sine and cosine
// of both; only lanes below rot / 2 rotate).
struct Rotation {
  float s0, c0, s1, c1;
};

__device__ __forceinline__ Rotation rotation_of(int pos, int d0, int rot, double log2_base) {
  Rotation r{0.f, 1.f, 0.f, 1.f};
  if (d0 < rot) {
    const int half = rot >> 1;
    const int i0 = d0 < half ? d0 : d0 - half;
    // Angles in fp64, reduced modulo 2*pi before the fp32 sincos: at
    // positions of several thousand an fp32 angle would carry ~1e-4 rad of
    // rounding.
    sincosf(rope_angle(pos, i0, rot, log2_base), &r.s0, &r.c0);
    sincosf(rope_angle(pos, i0 + 1, rot, log2_base), &r.s1, &r.c1);
  }
  return r;
}

// A head's row (this lane's two features of it): RMSNorm and rotary by rotation(),
// packed.  x c and the product p s round once each, whatever the compiler would
// contract where this is inlined: every kernel rotates to the same bits.
template <class Rot>
__device__ __forceinline__ uint32_t norm_rotate(uint32_t xv, uint32_t wv, Rot rotation, int d0, int rot,
                                                float eps) {
  float x0 = bf16_lo(xv), x1 = bf16_hi(xv);
  const float ss = wave_sum(x0 * x0 + x1 * x1);
  const float inv = 1.f / sqrtf(ss / (float)kHD + eps);
  x0 = x0 * inv * bf16_lo(wv);
  x1 = x1 * inv * bf16_hi(wv);
  if (rot > 0) {
    const float p0 = __shfl_xor(x0, rot >> 2, 64);
    const float p1 = __shfl_xor(x1, rot >> 2, 64);
    if (d0 < rot) {
      const Rotation r = rotation();
      const float q0 = p0 * r.s0, q1 = p1 * r.s1;
      const bool low = d0 < (rot >> 1);
      x0 = fmaf(x0, r.c0, low ? -q0 : q0);
      x1 = fmaf(x1, r.c1, low ? -q1 : q1);
    }
  }
  return pack2(x0, x1);
}

typedef float f32x16 __attribute__((ext_vector_type(16)));

// x of this lane and of lane ^ 32.
__device__ __forceinline__ f32x2 both_halves(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return f32x2{__uint_as_float(r[0]), __uint_as_float(r[1])};
}

__device__ __forceinline__ u32x4 cvt8_bf16(const float* v) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  uint32_t o[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    o[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{v[2 * i], v[2 * i + 1]}, bf16x2));
  return u32x4{o[0], o[1], o[2], o[3]};
}

}  // namespace
}  // namespace dflash
