// The 8-bit key/value cache (include/dflash_kv8.h): its device view, the
// quantisation of a block, and the codes' conversion back.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_common.h"
#include "device_common.h"
#include "dflash_kv8.h"
#include "host_common.h"

namespace dflash {
namespace {

constexpr int kBlk = 64;      // positions that share a scale
constexpr int kSlots = 128;   // tail slots: two blocks
constexpr int kMaxDraft = 16; // tokens of a draft append
constexpr int kBlkBytes = kBlk * kHD;

struct Kv8 {
  uint8_t* k;
  uint8_t* v;
  float* ks;
  float* vs;
  uint16_t* tk;
  uint16_t* tv;
  int B, Hkv, Smax, nblk;

  // Head bh = b * Hkv + h: its block blk's keys [64][128] and values [128][64],
  // its tail's keys [slot][128] and values [128][slot].
  __device__ uint8_t* keys(int64_t bh, int blk) const { return k + (bh * nblk + blk) * kBlkBytes; }
  __device__ uint8_t* values(int64_t bh, int blk) const { return v + (bh * nblk + blk) * kBlkBytes; }
  __device__ uint16_t* tail_keys(int64_t bh) const { return tk + bh * (kSlots * kHD); }
  __device__ uint16_t* tail_values(int64_t bh) const { return tv + bh * (kHD * kSlots); }
};

inline int check_cache(const dflash_kv8_cache* c, Kv8* out) {
  if (c == nullptr) return DFLASH_ERR_NULL;
  if (c->type != DFLASH_KV_INT8 && c->type != DFLASH_KV_E4M3) return DFLASH_ERR_UNSUPPORTED;
  if (c->B < 0 || c->Hkv <= 0 || c->Smax <= 0 || c->Smax % kBlk != 0) return DFLASH_ERR_SHAPE;
  if ((int64_t)c->B * c->Hkv > INT32_MAX) return DFLASH_ERR_SHAPE;
  *out = Kv8{static_cast<uint8_t*>(c->k_codes), static_cast<uint8_t*>(c->v_codes), c->k_scale, c->v_scale,
             static_cast<uint16_t*>(c->tail_k), static_cast<uint16_t*>(c->tail_vt), c->B, c->Hkv, c->Smax,
             c->Smax / kBlk};
  if (c->B == 0) return DFLASH_OK;
  const void* ptrs[] = {c->k_codes, c->v_codes, c->k_scale, c->v_scale, c->tail_k, c->tail_vt};
  for (const void* p : ptrs) {
    if (p == nullptr) return DFLASH_ERR_NULL;
    if ((uintptr_t)p & 15) return DFLASH_ERR_ALIGN;
  }
  return DFLASH_OK;
}

// A block's scale and its values' multiplier.  a: the largest magnitude's bits
// (as an integer maximum of |x|'s bits, so NaN and infinity stand above all).
template <int TYPE>
__device__ __forceinline__ f32x2 block_scale(uint32_t a_bits) {
  if (a_bits >= 0x7f800000u) return f32x2{__uint_as_float(0x7fc00000u), 0.f};
  const float a = fmaxf(__uint_as_float(a_bits), 0x1p-100f);
  if (TYPE == DFLASH_KV_INT8) return f32x2{a / 127.f, 127.f / a};
  // a = 1.m 2^e, 448 = 1.75 2^8: 2^(e-8), or 2^(e-7) where 1.m > 1.75
  const uint32_t u = __float_as_uint(a);
  const uint32_t e = (u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1u : 0u);
  return f32x2{__uint_as_float(e << 23), __uint_as_float((254u - e) << 23)};
}

// Four codes.  mul 0 (a block with a NaN or an infinity): codes 0.
template <int TYPE>
__device__ __forceinline__ uint32_t quantise4(float x0, float x1, float x2, float x3, float mul) {
  if (mul == 0.f) return 0u;
  if (TYPE == DFLASH_KV_INT8) {
    const int a = (int)rintf(x0 * mul), b = (int)rintf(x1 * mul);
    const int c = (int)rintf(x2 * mul), d = (int)rintf(x3 * mul);
    return (a & 255) | ((b & 255) << 8) | ((c & 255) << 16) | ((uint32_t)d << 24);
  }
  int r = __builtin_amdgcn_cvt_pk_fp8_f32(x0 * mul, x1 * mul, 0, false);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x2 * mul, x3 * mul, r, true);
}

// Eight codes from 16 bytes of bf16.
template <int TYPE>
__device__ __forceinline__ u32x2 quantise8(u32x4 w, float mul) {
  float f[8];
  unpack8(w, f);
  return u32x2{quantise4<TYPE>(f[0], f[1], f[2], f[3], mul), quantise4<TYPE>(f[4], f[5], f[6], f[7], mul)};
}

// Four codes as fp32: exact.
template <int TYPE>
__device__ __forceinline__ f32x4 codes_f32(uint32_t c) {
  if (TYPE == DFLASH_KV_INT8)
    return f32x4{(float)(int8_t)c, (float)(int8_t)(c >> 8), (float)(int8_t)(c >> 16), (float)(int8_t)(c >> 24)};
  const f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, false), b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c, true);
  return f32x4{a.x, a.y, b.x, b.y};
}

// Byte N of c, signed, as fp32, in one instruction.  (Written out: from plain C the
// compiler takes a loaded word apart byte by byte where it is loaded and carries 16
// registers where 4 do, and converts in two.)
template <int N>
__device__ __forceinline__ uint32_t signed_byte_f32(uint32_t c) {
  uint32_t f;
  if (N == 0)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_0" : "=v"(f) : "v"(c));
  if (N == 1)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_1" : "=v"(f) : "v"(c));
  if (N == 2)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_2" : "=v"(f) : "v"(c));
  if (N == 3)
    asm("v_cvt_f32_i32_sdwa %0, sext(%1) dst_sel:DWORD dst_unused:UNUSED_PAD src0_sel:BYTE_3" : "=v"(f) : "v"(c));
  return f;
}

// Four codes as two packed bf16 pairs: exact, both types have at most 8 significant bits.
template <int TYPE>
__device__ __forceinline__ u32x2 codes_bf16(uint32_t c) {
  if (TYPE == DFLASH_KV_INT8)  // integers: the low half of the fp32 bits is zero
    return u32x2{__builtin_amdgcn_perm(signed_byte_f32<1>(c), signed_byte_f32<0>(c), 0x07060302u),
                 __builtin_amdgcn_perm(signed_byte_f32<3>(c), signed_byte_f32<2>(c), 0x07060302u)};
  return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, false)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c, 1.f, true))};
}

// What eight codes stand for, rounded to bf16.
template <int TYPE>
__device__ __forceinline__ u32x4 values_bf16(u32x2 q, float scale) {
  const f32x4 a = codes_f32<TYPE>(q.x) * scale, b = codes_f32<TYPE>(q.y) * scale;
  const float f[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  return cvt8_bf16(f);
}

// Largest magnitude's bits of two packed bf16, as fp32 bits.
__device__ __forceinline__ uint32_t abs_bits2(uint32_t w) {
  return max(w & 0x7fff0000u, (w << 16) & 0x7fff0000u);
}
__device__ __forceinline__ uint32_t abs_bits16(u32x4 w) {
  return max(max(abs_bits2(w.x), abs_bits2(w.y)), max(abs_bits2(w.z), abs_bits2(w.w)));
}

__device__ __forceinline__ uint32_t wave_max_u32(uint32_t x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x = max(x, (uint32_t)__shfl_xor((int)x, off, 64));
  return x;
}

// Maximum over a 256-thread workgroup (red: 4 words of LDS; ends after a barrier,
// and no thread writes red again before the next one).
__device__ __forceinline__ uint32_t group_max_u32(uint32_t x, uint32_t* red) {
  x = wave_max_u32(x);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = x;
  __syncthreads();
  x = max(max(red[0], red[1]), max(red[2], red[3]));
  __syncthreads();
  return x;
}

}  // namespace
}  // namespace dflash
