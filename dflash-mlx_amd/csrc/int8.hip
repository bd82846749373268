// Projections in 8-bit integers: quantisation of rows, packing of weights and the
// product (include/dflash_int8.h has the formats and formulas).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "device_common.h"
#include "dflash_int8.h"
#include "host_common.h"
#include "int8_common.h"

namespace dflash {
namespace {

typedef u32x4 u32x4_e2 __attribute__((aligned(2)));  // a vector at any element of 16 bits

// ------------------------------------------------------------------ quantise

template <bool BF16>
__device__ __forceinline__ float value16(uint32_t bits) {
  return BF16 ? bf16_bits_to_f32(bits) : f16_bits_to_f32((uint16_t)bits);
}

// One row's largest magnitude as the 16-bit pattern without its sign (the order of
// the patterns is that of the magnitudes, a NaN above an infinity above the rest) to
// its scale, and to what makes a code: 127 x / a = (x * times) / a1 with a = a1 2^e,
// 1 <= a1 < 2, and times = 127 / 2^e, which neither overflows nor rounds.
struct RowScale {
  float times, a1, inv, scale;
  bool finite;
};
template <bool BF16>
__device__ __forceinline__ RowScale row_scale(uint32_t largest) {
  RowScale r;
  r.finite = largest < (BF16 ? 0x7f80u : 0x7c00u);
  const float a = r.finite ? fmaxf(value16<BF16>(largest), 0x1p-100f) : 1.f;
  const uint32_t bits = __float_as_uint(a);
  r.times = __uint_as_float(((260u - (bits >> 23)) << 23) | 0x7e0000u);  // 127 = 0x7e0000 / 2^23 + 1 times 2^6
  r.a1 = __uint_as_float((bits & 0x7fffffu) | 0x3f800000u);
  r.inv = 1.f / r.a1;
  r.scale = r.finite ? a / 127.f : __builtin_nanf("");
  return r;
}

// rint(127 x / a).  One correction makes a quotient that fp32 can hold exact, ties
// among them (the numerator and the residual are exact: x and a have at most 11
// bits), and any other quotient is further from a tie, 1 / (2 mantissa of a) = 2^-12
// of its last place and 2^-20 of itself, than the corrected one is from it (2^-23).
__device__ __forceinline__ int code_of(float x, const RowScale& r) {
  const float y = x * r.times, q = y * r.inv;
  return (int)rintf(fmaf(fmaf(-q, r.a1, y), r.inv, q));
}

template <bool BF16>
__device__ __forceinline__ u32x2 codes8(u32x4 v, const RowScale& r) {
  uint32_t o[2] = {0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    o[e >> 2] |= (uint32_t)(code_of(value16<BF16>((v[e >> 1] >> (16 * (e & 1))) & 0xffffu), r) & 0xff) << (8 * (e & 3));
  return r.finite ? u32x2{o[0], o[1]} : u32x2{0, 0};
}

__device__ __forceinline__ uint32_t largest8(u32x4 v, uint32_t m) {
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max(v[i] & 0x7fffu, (v[i] >> 16) & 0x7fffu));
  return m;
}

// Elements 8c .. 8c + 7 of a row of K (zeros past its end).
__device__ __forceinline__ u32x4 load_row8(const uint16_t* x, int c, int K) {
  if (8 * c + 8 <= K) return *reinterpret_cast<const u32x4_e2*>(x + 8 * c);
  u32x4 v{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (8 * c + e < K) v[e >> 1] |= (uint32_t)x[8 * c + e] << (16 * (e & 1));
  return v;
}

constexpr int kQThreads = 256;

// A workgroup a row.
template <bool BF16>
__global__ __launch_bounds__(kQThreads) void quantize_rows_kernel(const uint16_t* x, int64_t xs, uint8_t* codes,
                                                                  int64_t cs, float* scale, int K) {
  __shared__ uint32_t best[kQThreads / 64];
  const uint16_t* xr = x + (int64_t)blockIdx.x * xs;
  const int chunks = 2 * ((K + 15) >> 4);  // pieces of 8, up to K rounded up to 16
  uint32_t m = 0;
  for (int c = threadIdx.x; c < chunks; c += kQThreads) m = largest8(load_row8(xr, c, K), m);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kQThreads / 64; ++w) m = max(m, best[w]);
  const RowScale r = row_scale<BF16>(m);
  uint8_t* cr = codes + (int64_t)blockIdx.x * cs;
  for (int c = threadIdx.x; c < chunks; c += kQThreads)
    *reinterpret_cast<u32x2*>(cr + 8 * c) = codes8<BF16>(load_row8(xr, c, K), r);
  if (threadIdx.x == 0) scale[blockIdx.x] = r.scale;
}

// ---------------------------------------------------------------------- pack

// A thread a lane's 16 bytes of a fragment.
__global__ __launch_bounds__(256) void pack_kernel(const int8_t* codes, int64_t rs, const float* scale, u32x4* packed,
                                                   float* packed_scale, int N, int K, int gated, int tiles) {
  const int lane = threadIdx.x & 63;
  const int tile = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (tile >= tiles) return;
  const int ks = blockIdx.y;
  const int half = N / 2;
  const int j = gated ? 16 * (tile >> 1) + (lane & 15) : 16 * tile + (lane & 15);  // channel, of its half if gated
  const int n = gated && (tile & 1) ? half + j : j;
  const bool live = j < (gated ? half : N);
  const int k0 = 64 * ks + 16 * (lane >> 4);
  u32x4 v{0, 0, 0, 0};
  if (live)
    for (int e = 0; e < 16; ++e)
      if (k0 + e < K) v[e >> 2] |= (uint32_t)(uint8_t)codes[n * rs + k0 + e] << (8 * (e & 3));
  packed[((int64_t)ks * tiles + tile) * 64 + lane] = v;
  if (ks == 0 && lane < 16) packed_scale[16 * tile + lane] = live ? scale[n] : 0.f;
}

// ------------------------------------------------------------------- product

// A wave takes two channel tiles and MT row tiles over all of K.
template <typename T, bool GATED, int MT>
__global__ __launch_bounds__(256) void gemm_i8_kernel(const GemmI8 p) {
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int t = 2 * (blockIdx.x * 4 + (threadIdx.x >> 6));
  if (t >= p.tiles) return;
  const int m0 = blockIdx.y * 16 * MT;
  const int t1 = min(t + 1, p.tiles - 1);
  const int last = (p.K - 1) >> 4;  // the row's last 16-byte piece; the weight is 0 behind K
  i32x4 acc[2][MT] = {};
  for (int ks = 0; ks < p.k_steps; ++ks) {
    const u32x4* w = p.w + (int64_t)ks * p.tiles * 64 + lane;
    const i32x4 a0 = __builtin_bit_cast(i32x4, w[(int64_t)t * 64]);
    const i32x4 a1 = __builtin_bit_cast(i32x4, w[(int64_t)t1 * 64]);
    const int piece = min(4 * ks + g, last);
#pragma unroll
    for (int j = 0; j < MT; ++j) {
      const int m = min(m0 + 16 * j + r16, p.M - 1);
      const i32x4 b = *reinterpret_cast<const i32x4*>(p.x + (int64_t)m * p.xs + 16 * piece);
      acc[0][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a0, b, acc[0][j], 0, 0, 0);
      acc[1][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a1, b, acc[1][j], 0, 0, 0);
    }
  }
#pragma unroll
  for (int j = 0; j < MT; ++j) {
    const int m = m0 + 16 * j + r16;
    if (m < p.M)
      store_pair<T, GATED>(p, t, g, static_cast<T*>(p.out) + (int64_t)m * p.os, 4 * g, acc[0][j], acc[1][j], tile_scales(p, t, g), tile_scales(p, t + 1, g), p.sx[m]);
  }
}

template <typename T, bool GATED>
hipError_t launch_gemm(const GemmI8& p, hipStream_t s) {
  if (p.M > 256) return launch_prompt_i8<T, GATED>(p, s);
  const unsigned gx = (unsigned)ceil_div(p.tiles, 8);
  if (p.M <= 16)
    hipLaunchKernelGGL((gemm_i8_kernel<T, GATED, 1>), dim3(gx, 1), dim3(256), 0, s, p);
  else
    hipLaunchKernelGGL((gemm_i8_kernel<T, GATED, 4>), dim3(gx, (unsigned)ceil_div(p.M, 64)), dim3(256), 0, s, p);
  return hipGetLastError();
}

template <typename T>
hipError_t launch_gemm(const GemmI8& p, int gated, hipStream_t s) {
  return gated ? launch_gemm<T, true>(p, s) : launch_gemm<T, false>(p, s);
}

bool bad_weight(int N, int K, int gated) {
  return N <= 0 || K <= 0 || K > DFLASH_I8_MAX_K || N > INT32_MAX - 64 || (gated && N % 2);
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" size_t dflash_weight_i8_bytes(int N, int K, int gated) {
  return bad_weight(N, K, gated) ? 0 : (size_t)k_steps(K) * channel_tiles(N, gated) * 1024;
}

extern "C" size_t dflash_weight_i8_scales(int N, int gated) {
  return bad_weight(N, 1, gated) ? 0 : (size_t)16 * channel_tiles(N, gated);
}

extern "C" int dflash_weight_pack_i8(const void* codes, int64_t row_stride, const float* scale, void* packed_codes,
                                     float* packed_scale, int N, int K, int gated, void* stream) {
  if (bad_weight(N, K, gated) || (N > 1 && row_stride < K)) return DFLASH_ERR_SHAPE;
  if (codes == nullptr || scale == nullptr || packed_codes == nullptr || packed_scale == nullptr) return DFLASH_ERR_NULL;
  if ((uintptr_t)scale % 4 || (uintptr_t)packed_codes % 16 || (uintptr_t)packed_scale % 16) return DFLASH_ERR_ALIGN;
  const int tiles = channel_tiles(N, gated);
  hipLaunchKernelGGL(pack_kernel, dim3((unsigned)ceil_div(tiles, 4), (unsigned)k_steps(K)), dim3(256), 0,
                     static_cast<hipStream_t>(stream), static_cast<const int8_t*>(codes), row_stride, scale,
                     static_cast<u32x4*>(packed_codes), packed_scale, N, K, gated, tiles);
  return to_status(hipGetLastError());
}

extern "C" int dflash_quantize_rows_i8(const void* x, int x_dtype, int64_t x_row_stride, void* codes,
                                       int64_t codes_row_stride, float* scale, int M, int K, void* stream) {
  if (M < 0 || K <= 0 || K > DFLASH_I8_MAX_K || x_row_stride < 0) return DFLASH_ERR_SHAPE;
  if (codes_row_stride < 16 * ceil_div(K, 16)) return DFLASH_ERR_SHAPE;
  if (M == 0) return DFLASH_OK;
  if (x == nullptr || codes == nullptr || scale == nullptr) return DFLASH_ERR_NULL;
  if (x_dtype != DFLASH_DTYPE_BF16 && x_dtype != DFLASH_DTYPE_F16) return DFLASH_ERR_UNSUPPORTED;
  if ((uintptr_t)x % 2 || (uintptr_t)codes % 16 || codes_row_stride % 16 || (uintptr_t)scale % 4)
    return DFLASH_ERR_ALIGN;
  const auto kernel = x_dtype == DFLASH_DTYPE_BF16 ? quantize_rows_kernel<true> : quantize_rows_kernel<false>;
  hipLaunchKernelGGL(kernel, dim3((unsigned)M), dim3(kQThreads), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint16_t*>(x), x_row_stride, static_cast<uint8_t*>(codes), codes_row_stride,
                     scale, K);
  return to_status(hipGetLastError());
}

extern "C" int dflash_gemm_i8(const void* x, int64_t x_row_stride, const float* x_scale, const void* packed_codes,
                              const float* packed_scale, void* out, int out_dtype, int64_t out_row_stride, int M,
                              int N, int K, int gated, void* stream) {
  if (M < 0 || bad_weight(N, K, gated)) return DFLASH_ERR_SHAPE;
  GemmI8 p{};
  p.cols = gated ? N / 2 : N;
  if (M > 1 && (x_row_stride < 16 * ceil_div(K, 16) || out_row_stride < p.cols)) return DFLASH_ERR_SHAPE;
  // the prompt kernel's offsets in a block of rows are 32-bit, its tiles counted in an int
  if (x_row_stride > (1 << 23) || out_row_stride > (1 << 26) || ceil_div(M, 256) * ceil_div(N, 128) > INT32_MAX / 2) return DFLASH_ERR_SHAPE;
  if (M == 0) return DFLASH_OK;
  if (x == nullptr || x_scale == nullptr || packed_codes == nullptr || packed_scale == nullptr || out == nullptr)
    return DFLASH_ERR_NULL;
  const bool f32 = out_dtype == DFLASH_DTYPE_F32;
  if (!f32 && out_dtype != DFLASH_DTYPE_BF16 && out_dtype != DFLASH_DTYPE_F16) return DFLASH_ERR_UNSUPPORTED;
  if ((uintptr_t)x % 16 || x_row_stride % 16 || (uintptr_t)x_scale % 4 || (uintptr_t)packed_codes % 16 ||
      (uintptr_t)packed_scale % 16 || (uintptr_t)out % (f32 ? 4 : 2))
    return DFLASH_ERR_ALIGN;
  p.x = static_cast<const uint8_t*>(x), p.xs = x_row_stride, p.sx = x_scale;
  p.w = static_cast<const u32x4*>(packed_codes), p.sw = packed_scale;
  p.out = out, p.os = out_row_stride;
  p.M = M, p.K = K, p.k_steps = k_steps(K), p.tiles = channel_tiles(N, gated);
  hipStream_t s = static_cast<hipStream_t>(stream);
  return to_status(f32                                ? launch_gemm<float>(p, gated, s)
                   : out_dtype == DFLASH_DTYPE_BF16 ? launch_gemm<uint16_t>(p, gated, s)
                                                      : launch_gemm<_Float16>(p, gated, s));
}
