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

// A workgroup of NT threads a row, which they keep in registers: one trip to memory for
// rows of up to 32 NT values, and another to the L2 for longer ones.
template <bool BF16, int NT>
__global__ __launch_bounds__(NT) void quantize_rows_kernel(const uint16_t* x, int64_t xs, uint8_t* codes, int64_t cs,
                                                           float* scale, int K) {
  constexpr int R = 4;
  __shared__ uint32_t best[NT / 64];
  const uint16_t* xr = x + (int64_t)blockIdx.x * xs;
  uint8_t* cr = codes + (int64_t)blockIdx.x * cs;
  const int chunks = 2 * ((K + 15) >> 4);  // pieces of 8, up to K rounded up to 16
  u32x4 held[R] = {};
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (const int c = threadIdx.x + i * NT; c < chunks) held[i] = load_row8(xr, c, K);
#pragma unroll
  for (int i = 0; i < R; ++i) m = largest8(held[i], m);
  for (int c = threadIdx.x + R * NT; c < chunks; c += NT) m = largest8(load_row8(xr, c, K), m);
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
  if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) m = max(m, best[w]);
  const RowScale r = row_scale<BF16>(m);
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (const int c = threadIdx.x + i * NT; c < chunks) *reinterpret_cast<u32x2*>(cr + 8 * c) = codes8<BF16>(held[i], r);
  for (int c = threadIdx.x + R * NT; c < chunks; c += NT)
    *reinterpret_cast<u32x2*>(cr + 8 * c) = codes8<BF16>(load_row8(xr, c, K), r);
  if (threadIdx.x == 0) scale[blockIdx.x] = r.scale;
}

// The residual add and RMSNorm with the row quantised in the same registers.  The norm is
// rounded to bf16 first, as the projections' rows are otherwise.  A launch, and the normed
// rows' way to memory and back, less before every projection of a layer's input: of few
// rows, where every launch is bound by its latency, 4.9 us for 16 rows of 2560 against 4.1 +
// 4.0 (a verify step of 16 tokens 2.49 -> 2.35 ms).  Four eights a thread: rows of up to 32 NT.
template <int NT>
__global__ __launch_bounds__(NT) void add_rmsnorm_i8_kernel(const u32x4* h, const u32x4* r, const u32x4* w, u32x4* h_out,
                                                            u32x4* capture, int64_t capture_stride, uint8_t* codes,
                                                            int64_t cs, float* scale, int H, float eps) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  constexpr int R = 4;
  __shared__ float sums[NT / 64];
  __shared__ uint32_t best[NT / 64];
  const int chunks = H >> 3, wave = threadIdx.x >> 6;
  const int64_t at = (int64_t)blockIdx.x * chunks;
  auto pack = [](float a, float b) { return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2)); };
  u32x4 held[R] = {}, weight[R] = {};
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int c = threadIdx.x + i * NT;
    if (c >= chunks) continue;
    u32x4 v = h[at + c];
    weight[i] = w[c];
    if (r != nullptr) {
      const u32x4 a = r[at + c];
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] = pack(bf16_lo(v[e]) + bf16_lo(a[e]), bf16_hi(v[e]) + bf16_hi(a[e]));
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) sum = fmaf(bf16_lo(v[e]), bf16_lo(v[e]), fmaf(bf16_hi(v[e]), bf16_hi(v[e]), sum));
    h_out[at + c] = v;
    if (capture != nullptr) capture[blockIdx.x * (capture_stride >> 3) + c] = v;
    held[i] = v;
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) sum += __shfl_xor(sum, off, 64);
  if ((threadIdx.x & 63) == 0) sums[wave] = sum;
  __syncthreads();
  sum = 0.f;
#pragma unroll
  for (int k = 0; k < NT / 64; ++k) sum += sums[k];
  const float inv = 1.f / sqrtf(sum / (float)H + eps);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      held[i][e] = pack(bf16_lo(held[i][e]) * inv * bf16_lo(weight[i][e]), bf16_hi(held[i][e]) * inv * bf16_hi(weight[i][e]));
    m = largest8(held[i], m);
  }
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) m = max(m, (uint32_t)__shfl_xor((int)m, off, 64));
  if ((threadIdx.x & 63) == 0) best[wave] = m;
  __syncthreads();
#pragma unroll
  for (int k = 0; k < NT / 64; ++k) m = max(m, best[k]);
  const RowScale rs = row_scale<true>(m);
  uint8_t* cr = codes + (int64_t)blockIdx.x * cs;
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (const int c = threadIdx.x + i * NT; c < chunks) *reinterpret_cast<u32x2*>(cr + 8 * c) = codes8<true>(held[i], rs);
  if (threadIdx.x == 0) scale[blockIdx.x] = rs.scale;
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
  typedef u32x4 u32x4_e1 __attribute__((aligned(1)));
  if (live && k0 + 16 <= K)
    v = *reinterpret_cast<const u32x4_e1*>(codes + n * rs + k0);
  else if (live)
    for (int e = 0; e < 16; ++e)
      if (k0 + e < K) v[e >> 2] |= (uint32_t)(uint8_t)codes[n * rs + k0 + e] << (8 * (e & 3));
  packed[((int64_t)ks * tiles + tile) * 64 + lane] = v;
  if (ks == 0 && lane < 16) packed_scale[16 * tile + lane] = live ? scale[n] : 0.f;
}

// ------------------------------------------------------------------- product

// Few rows: the weight is streamed once.  A workgroup takes VT channel tiles and all
// rows; its KW waves share K, each with a stretch of its own: no barrier while they
// stream, weights D k-steps ahead in registers, rows (which every workgroup reads) from
// the L2.  Their sums meet in LDS, integers, so their order does not matter.
//
// RAW (1 bf16, 2 fp16): a single row comes as it is, and every workgroup quantises it for
// itself into LDS while its first weights are on their way: 0.2 to 1.5 us where a launch
// before takes 2.6 (1 x 2560 x 9216 7.6 us in all, 18432 x 2560 gated 10.2; a verify step of
// one token 1.88 -> 1.78 ms).  Two rows take 2.1 to 2.8 so and four 2.3 to 4.7: no gain.
template <typename T, bool GATED, int MT, int VT, int KW, int D, int RAW>
__global__ __launch_bounds__(64 * KW) void stream_i8_kernel(const GemmI8 p) {
  __shared__ i32x4 sums[KW][VT * MT][64];
  extern __shared__ __attribute__((aligned(16))) uint8_t codes_s[];
  __shared__ uint32_t best_s[KW];
  float raw_scale = 0.f;
  static_assert(!RAW || MT == 1, "a single row");
  const int lane = threadIdx.x & 63, r16 = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int t0 = VT * blockIdx.x;
  const int all = (p.K + 63) >> 6, per = (all + KW - 1) / KW;
  const int k0 = min(wave * per, all), n = min(per, all - k0);
  const int last = (p.K - 1) >> 4;  // a row's last 16-byte piece; the weight is 0 behind K
  const u32x4* w[VT];
  const uint8_t* x[MT];
  constexpr int kHeld = 3;
  u32x4 held[kHeld] = {};
  const int chunks = 2 * (last + 1);
  if (RAW) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (const int c = threadIdx.x + i * 64 * KW; c < chunks) held[i] = load_row8(p.raw, c, p.K);
  }
#pragma unroll
  for (int v = 0; v < VT; ++v)
    w[v] = p.w + ((int64_t)k0 * p.tiles + min(t0 + v, p.tiles - 1)) * 64 + lane;
#pragma unroll
  for (int j = 0; j < MT; ++j)
    x[j] = RAW ? codes_s : p.x + (int64_t)min(16 * j + r16, p.M - 1) * p.xs;
  struct Stage {
    i32x4 a[VT], b[MT];
  } ring[D];
  auto load_rows = [&](Stage& s, int i) __attribute__((always_inline)) {
    const int piece = min(4 * (k0 + i) + g, last);
#pragma unroll
    for (int j = 0; j < MT; ++j) s.b[j] = *reinterpret_cast<const i32x4*>(x[j] + 16 * piece);
  };
  auto load = [&](Stage& s, int i) __attribute__((always_inline)) {
#pragma unroll
    for (int v = 0; v < VT; ++v)
      s.a[v] = __builtin_bit_cast(i32x4, __builtin_nontemporal_load(w[v] + (int64_t)i * p.tiles * 64));
    if (!RAW) load_rows(s, i);
  };
  i32x4 acc[VT][MT] = {};
  auto multiply = [&](Stage& s, int i) __attribute__((always_inline)) {
    if (RAW) load_rows(s, i);
#pragma unroll
    for (int v = 0; v < VT; ++v)
#pragma unroll
      for (int j = 0; j < MT; ++j)
        acc[v][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(s.a[v], s.b[j], acc[v][j], 0, 0, 0);
  };
  // Loads past the stretch read its last step again, so that every turn has as many in flight.
  if (n > 0) {
#pragma unroll
    for (int d = 0; d < D; ++d) load(ring[d], min(d, n - 1));
  }
  if (RAW) {
    uint32_t most = 0;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) most = largest8(held[i], most);
    for (int c = threadIdx.x + kHeld * 64 * KW; c < chunks; c += 64 * KW) most = largest8(load_row8(p.raw, c, p.K), most);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, off, 64));
    if (lane == 0) best_s[wave] = most;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < KW; ++k) most = max(most, best_s[k]);
    const RowScale r = row_scale<RAW == 1>(most);
    raw_scale = r.scale;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (const int c = threadIdx.x + i * 64 * KW; c < chunks)
        *reinterpret_cast<u32x2*>(codes_s + 8 * c) = codes8<RAW == 1>(held[i], r);
    for (int c = threadIdx.x + kHeld * 64 * KW; c < chunks; c += 64 * KW)
      *reinterpret_cast<u32x2*>(codes_s + 8 * c) = codes8<RAW == 1>(load_row8(p.raw, c, p.K), r);
    __syncthreads();
  }
  if (n > 0) {
    int i = 0;
    for (; i + D <= n; i += D) {
#pragma unroll
      for (int d = 0; d < D; ++d) {
        multiply(ring[d], i + d);
        load(ring[d], min(i + D + d, n - 1));
      }
    }
#pragma unroll
    for (int d = 0; d < D; ++d)
      if (i + d < n) multiply(ring[d], i + d);
  }
  // Wave k adds up and stores the pairs (of channel tiles, by row tile) k, k + KW, ...
#pragma unroll
  for (int v = 0; v < VT; ++v)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[wave][v * MT + j][lane] = acc[v][j];
  constexpr int kPair = VT > 1 ? 2 : 1;
  __syncthreads();
  for (int q = wave; q < VT / kPair * MT; q += KW) {
    const int v = q / MT * kPair, j = q % MT, t = t0 + v, m = 16 * j + r16;
    i32x4 a = sums[0][v * MT + j][lane], b = sums[0][(v + kPair - 1) * MT + j][lane];
#pragma unroll
    for (int k = 1; k < KW; ++k) {
      a += sums[k][v * MT + j][lane];
      if (VT > 1) b += sums[k][(v + kPair - 1) * MT + j][lane];
    }
    if (t < p.tiles && m < p.M) {
      T* row = static_cast<T*>(p.out) + (int64_t)m * p.os;
      const f32x4 sa = tile_scales(p, t, g);
      const float sx = RAW ? raw_scale : p.sx[m];
      if (VT > 1) {
        store_pair<T, GATED>(p, t, g, row, 4 * g, a, b, sa, tile_scales(p, t + 1, g), sx);
      } else {
        float o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = (float)a[e] * sa[e] * sx;
        store_cols<T, false>(p, row, 4 * g, 16 * t, g, o);
      }
    }
  }
}

template <typename T, bool GATED, int MT, int VT, int KW, int RAW>
hipError_t launch_stream(const GemmI8& p, hipStream_t s) {
  hipLaunchKernelGGL((stream_i8_kernel<T, GATED, MT, VT, KW, 4, RAW>), dim3((unsigned)ceil_div(p.tiles, VT)),
                     dim3(64 * KW), RAW ? 16 * (unsigned)ceil_div(p.K, 16) : 0, s, p);
  return hipGetLastError();
}

// Measured in replayed graphs over weights that are not in the cache (MI355X, us, the
// launch's gap with it), 16 rows, one channel tile and 8 waves / two and 4 / four and 4:
// 2560 x 9216 9.3 / 12.3 / 17.0, 2560 x 4096 6.1 / 7.0 / 9.3, 5120 x 2560 7.7 / 5.7 / 7.2,
// 18432 x 2560 gated - / 13.2 / 13.4, 151936 x 2560 117 / 80 / 71.
template <typename T, bool GATED, int MT, int RAW = 0>
hipError_t launch_rows(const GemmI8& p, hipStream_t s) {
  if (p.tiles <= 256) return launch_stream<T, GATED, MT, GATED ? 2 : 1, 8, RAW>(p, s);
  if (p.tiles <= 2048) return launch_stream<T, GATED, MT, 2, 4, RAW>(p, s);
  return launch_stream<T, GATED, MT, 4, 4, RAW>(p, s);
}

// A row that the streaming workgroups quantise for themselves: their LDS holds its codes.
constexpr int kRawK = 40960;

template <typename T, bool GATED>
hipError_t launch_gemm(const GemmI8& p, hipStream_t s) {
  if (p.plan.kind != PlanI8::kStream) return launch_prompt_i8<T, GATED>(p, s);
  if (p.M <= 16) return launch_rows<T, GATED, 1>(p, s);
  if (p.M <= 32) return launch_rows<T, GATED, 2>(p, s);
  return launch_rows<T, GATED, 4>(p, s);
}

template <typename T>
hipError_t launch_gemm(const GemmI8& p, int gated, hipStream_t s) {
  return gated ? launch_gemm<T, true>(p, s) : launch_gemm<T, false>(p, s);
}

// The plan of the least estimated time, in us, fitted to times of replayed graphs (MI355X).
//   stream: its bytes, the weight's and the rows' for every group of channel tiles, at 5.8
//     TB/s, for up to 64 rows;
//   wide: 0.62 a k-step of 64 and 8 a tile's outputs, a round of the compute units;
//   narrow: 0.45 a k-step where two workgroups share a unit, 0.27 alone, and 4 a tile; the
//     splits' sums are written and read at 4 TB/s by a launch of 2.5.
// Of the measured times of 23 products of 17 to 4096 rows, 2560 to 151936 channels and 1001 to
// 9216 features, weights not in the cache, the estimate is 0.95 to 1.1 for streams and 256 x 256
// tiles and 0.9 to 1.25 for 128 x 128 tiles of whole K; 1.25 to 1.4 where K is split (64 x 2560 x
// 9216 in 12: 17.7 for 13.5); and too short where a narrow launch waits for its weight: 63 for 78
// to 95 us of 17 and 64 x 151936 x 2560, 12.3 for 16.5 of 700 x 5003 x 1001.
PlanI8 plan_i8(int M, int tiles, int k_steps) {
  PlanI8 best{PlanI8::kStream, 1};
  if (M <= 16) return best;
  const double cus = std::max(device_cus(), 1);
  double least = 1e30;
  if (M <= 64) {
    const int vt = tiles <= 256 ? 1 : tiles <= 2048 ? 2 : 4;
    const double rows = (double)ceil_div(tiles, vt) * 16 * ceil_div(M, 16);
    least = 3 + (rows + 16. * tiles) * 64 * k_steps / 5.8e6;
  }
  const double wide = 4 + ceil_div(ceil_div(tiles, 16) * ceil_div(M, 256), (int64_t)cus) * (0.62 * k_steps + 8);
  if (wide < least) least = wide, best = {PlanI8::kWide, 1};
  const int64_t narrow_tiles = ceil_div(tiles, 8) * ceil_div(M, 128);
  for (int n = 1; n <= 16 && 4 * n <= k_steps; ++n) {
    const int steps = 2 * (int)ceil_div(k_steps / 2, n);
    if (n > 1 && narrow_tiles * n > 2 * cus) break;
    const int64_t units = narrow_tiles * n, whole = units / (int64_t)(2 * cus), rest = units % (int64_t)(2 * cus);
    double t = 4 + whole * (0.45 * steps + 4) + (rest == 0 ? 0 : rest <= cus ? 0.27 * steps + 4 : 0.45 * steps + 4);
    if (n > 1) t += 2.5 + 8. * n * M * 16 * tiles / 4e6;
    if (t < least) least = t, best = {PlanI8::kNarrow, (int)ceil_div(k_steps, steps)};
  }
  return best;
}

bool bad_weight(int N, int K, int gated) {
  return N <= 0 || K <= 0 || K > DFLASH_I8_MAX_K || N > DFLASH_I8_MAX_N || (gated && N % 2);
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
  const bool bf = x_dtype == DFLASH_DTYPE_BF16;
  // Few rows leave most of the device idle, whose threads then share a row.
  const bool wide = M <= 512 && K > 2048;
  const auto kernel = wide ? (bf ? quantize_rows_kernel<true, 1024> : quantize_rows_kernel<false, 1024>)
                           : (bf ? quantize_rows_kernel<true, 256> : quantize_rows_kernel<false, 256>);
  hipLaunchKernelGGL(kernel, dim3((unsigned)M), dim3(wide ? 1024 : 256), 0, static_cast<hipStream_t>(stream),
                     static_cast<const uint16_t*>(x), x_row_stride, static_cast<uint8_t*>(codes), codes_row_stride,
                     scale, K);
  return to_status(hipGetLastError());
}

extern "C" int dflash_add_rmsnorm_i8(const void* h, const void* r, const void* weight, void* h_out, void* capture,
                                     int64_t capture_stride, void* codes, int64_t codes_row_stride, float* scale,
                                     int M, int H, float eps, void* stream) {
  if (M < 0 || H <= 0 || H % 16 || H > 32768 || codes_row_stride < H) return DFLASH_ERR_SHAPE;
  if (capture != nullptr && capture_stride < H) return DFLASH_ERR_SHAPE;
  if (M == 0) return DFLASH_OK;
  if (h == nullptr || weight == nullptr || h_out == nullptr || codes == nullptr || scale == nullptr) return DFLASH_ERR_NULL;
  for (const void* a : {h, r, weight, (const void*)h_out, (const void*)capture, (const void*)codes})
    if ((uintptr_t)a % 16) return DFLASH_ERR_ALIGN;
  if (codes_row_stride % 16 || (capture != nullptr && capture_stride % 8) || (uintptr_t)scale % 4) return DFLASH_ERR_ALIGN;
  const bool wide = H > 8192 || (M <= 512 && H > 2048);  // as above, and 256 threads hold 8192
  hipLaunchKernelGGL(wide ? add_rmsnorm_i8_kernel<1024> : add_rmsnorm_i8_kernel<256>, dim3((unsigned)M),
                     dim3(wide ? 1024 : 256), 0, static_cast<hipStream_t>(stream), static_cast<const u32x4*>(h),
                     static_cast<const u32x4*>(r), static_cast<const u32x4*>(weight), static_cast<u32x4*>(h_out),
                     static_cast<u32x4*>(capture), capture_stride, static_cast<uint8_t*>(codes), codes_row_stride,
                     scale, H, eps);
  return to_status(hipGetLastError());
}

extern "C" size_t dflash_gemm_i8_workspace_bytes(int M, int N, int K, int gated) {
  if (M <= 0 || bad_weight(N, K, gated)) return 0;
  const int tiles = channel_tiles(N, gated), splits = plan_i8(M, tiles, k_steps(K)).splits;
  return splits > 1 ? (size_t)splits * M * tiles * 64 : 0;
}

extern "C" int dflash_gemm_i8(const void* x, int64_t x_row_stride, const float* x_scale, const void* packed_codes,
                              const float* packed_scale, void* out, int out_dtype, int64_t out_row_stride, int M,
                              int N, int K, int gated, void* workspace, size_t workspace_bytes, void* stream) {
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
  p.plan = plan_i8(M, p.tiles, p.k_steps);
  if (p.plan.splits > 1 && workspace_bytes < (size_t)p.plan.splits * M * p.tiles * 64) return DFLASH_ERR_WORKSPACE;
  if (p.plan.splits > 1 && workspace == nullptr) return DFLASH_ERR_NULL;
  if ((uintptr_t)workspace % 16) return DFLASH_ERR_ALIGN;
  p.workspace = workspace;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return to_status(f32                                ? launch_gemm<float>(p, gated, s)
                   : out_dtype == DFLASH_DTYPE_BF16 ? launch_gemm<uint16_t>(p, gated, s)
                                                      : launch_gemm<_Float16>(p, gated, s));
}

namespace {
// Where a linear's codes, scales and splits' sums lie in its workspace.
size_t codes_bytes(int M, int K) { return (size_t)M * 16 * ceil_div(K, 16); }
size_t scales_bytes(int M) { return 16 * (size_t)ceil_div(M, 4); }
}  // namespace

extern "C" size_t dflash_linear_i8_workspace_bytes(int M, int N, int K, int gated) {
  if (M <= 0 || bad_weight(N, K, gated)) return 0;
  return codes_bytes(M, K) + scales_bytes(M) + dflash_gemm_i8_workspace_bytes(M, N, K, gated);
}

extern "C" int dflash_linear_i8(const void* x, int x_dtype, int64_t x_row_stride, const void* packed_codes,
                                const float* packed_scale, void* out, int out_dtype, int64_t out_row_stride, int M,
                                int N, int K, int gated, void* workspace, size_t workspace_bytes, void* stream) {
  if (M < 0 || bad_weight(N, K, gated)) return DFLASH_ERR_SHAPE;
  const int cols = gated ? N / 2 : N;
  if (x_row_stride < 0 || (M > 1 && out_row_stride < cols) || out_row_stride > (1 << 26)) return DFLASH_ERR_SHAPE;
  if (M == 0) return DFLASH_OK;
  // what the product would refuse is refused before anything is launched
  if (packed_codes == nullptr || packed_scale == nullptr || out == nullptr || workspace == nullptr) return DFLASH_ERR_NULL;
  const bool f32 = out_dtype == DFLASH_DTYPE_F32;
  if (!f32 && out_dtype != DFLASH_DTYPE_BF16 && out_dtype != DFLASH_DTYPE_F16) return DFLASH_ERR_UNSUPPORTED;
  if ((uintptr_t)packed_codes % 16 || (uintptr_t)packed_scale % 16 || (uintptr_t)out % (f32 ? 4 : 2) ||
      (uintptr_t)workspace % 16)
    return DFLASH_ERR_ALIGN;
  if (workspace_bytes < dflash_linear_i8_workspace_bytes(M, N, K, gated)) return DFLASH_ERR_WORKSPACE;
  if (M == 1 && K <= kRawK) {
    if (x == nullptr) return DFLASH_ERR_NULL;
    if (x_dtype != DFLASH_DTYPE_BF16 && x_dtype != DFLASH_DTYPE_F16) return DFLASH_ERR_UNSUPPORTED;
    if ((uintptr_t)x % 2) return DFLASH_ERR_ALIGN;
    GemmI8 p{};
    p.raw = static_cast<const uint16_t*>(x);
    p.w = static_cast<const u32x4*>(packed_codes), p.sw = packed_scale;
    p.out = out, p.os = out_row_stride, p.cols = cols;
    p.M = M, p.K = K, p.k_steps = k_steps(K), p.tiles = channel_tiles(N, gated);
    const bool bf = x_dtype == DFLASH_DTYPE_BF16;
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto launch = [&](auto t) {
      using T = decltype(t);
      return gated ? (bf ? launch_rows<T, true, 1, 1>(p, s) : launch_rows<T, true, 1, 2>(p, s))
                   : (bf ? launch_rows<T, false, 1, 1>(p, s) : launch_rows<T, false, 1, 2>(p, s));
    };
    return to_status(f32 ? launch(0.f) : out_dtype == DFLASH_DTYPE_BF16 ? launch(uint16_t{}) : launch(_Float16{}));
  }
  char* ws = static_cast<char*>(workspace);
  const size_t cb = codes_bytes(M, K), sb = scales_bytes(M);
  float* scale = reinterpret_cast<float*>(ws + cb);
  const int64_t cs = 16 * ceil_div(K, 16);
  const int e = dflash_quantize_rows_i8(x, x_dtype, x_row_stride, ws, cs, scale, M, K, stream);
  if (e) return e;
  return dflash_gemm_i8(ws, cs, scale, packed_codes, packed_scale, out, out_dtype, out_row_stride, M, N, K, gated,
                        ws + cb + sb, workspace_bytes - cb - sb, stream);
}
