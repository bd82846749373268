// 8-bit products of many rows: a prompt's projections.
//
// A workgroup of 12 waves computes 256 channels x 256 rows: 8 waves multiply, 4 load,
// both operands staged in LDS by direct global -> LDS loads.
//   - Compute wave w < 8 (wr = w / 2, wc = w % 2) owns channel tiles 4 wr .. 4 wr + 3
//     against row tiles 8 wc .. 8 wc + 7: 32 accumulator tiles, 32 products of 16 x 16 x
//     64 a k-step of 64.
//   - Weight stages: one k-step's 16 fragments (16 KB, contiguous in the packed weight),
//     by loader waves 8 and 9; three slots.
//   - Row stages: 128 bytes of each of the 256 rows (32 KB), by loader waves 10 and 11
//     in chunks of 128 rows, each load 8 whole rows of 128 bytes; three slots.  A block
//     of 8 rows takes 1 KB of LDS, 16-byte piece c of row r at slot 8 r + (c ^ r), so the
//     8 lanes that read one piece of 8 rows touch all banks once.
//   - One barrier a k-step, which all 12 waves keep.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "int8_common.h"
#include "lds_dma.h"

namespace dflash {
namespace {

constexpr int kRows = 256, kChannels = 256;
constexpr int kBand = 16;                  // channel tiles of 256 per band of the tile walk
constexpr int kThreads = 768;
constexpr int kWeightSlot = 16384, kRowSlot = 32768;
constexpr int kRowBase = 3 * kWeightSlot;
constexpr int kScaleBase = kRowBase + 3 * kRowSlot;
constexpr int kScaleSlot = 4 * (kChannels + kRows);     // a tile's channel and row scales
constexpr int kLdsU4 = (kScaleBase + 4 * kScaleSlot) / 16;  // 152 KB

struct PromptI8 {
  GemmI8 g;
  int n_tiles, m_tiles, total, per_xcd;
};

__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Wait until at most n chunks (8 loads each) of this wave are outstanding.
__device__ __forceinline__ void wait_chunks(int n) {
  if (n <= 0) wait_vm<0>();
  else if (n == 1) wait_vm<8>();
  else if (n == 2) wait_vm<16>();
  else wait_vm<24>();
}

// One k-step of a wave's 4 x 8 tiles, the rows in two halves of four.
__device__ __forceinline__ void multiply(const i32x4* wst, const i32x4* xst, int wr, int wc, int lane, int boff,
                                         i32x4 (&acc)[4][8]) {
  i32x4 a[4], b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) a[i] = wst[(4 * wr + i) * 64 + lane];
#pragma unroll
  for (int jh = 0; jh < 2; ++jh) {
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = xst[boff + 2 * (8 * wc + 4 * jh + j) * 64];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        acc[i][4 * jh + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[i], b[j], acc[i][4 * jh + j], 0, 0, 0);
  }
}

// Tile t of a workgroup has its scales in one of four slots: a loader is at most two tiles
// (four steps of at least two a tile) ahead of the tile whose outputs are being stored.
__device__ __forceinline__ uint32_t scales_at(int t) { return kScaleBase + (t & 3) * kScaleSlot; }

// The tiles of a workgroup: every n_slots-th of its XCD's range.
struct Walk {
  int u, end, stride;
  __device__ bool done() const { return u >= end; }
};

template <typename T, bool GATED>
__global__ __launch_bounds__(kThreads, 1) void prompt_i8_kernel(const PromptI8 q) {
  __shared__ __attribute__((aligned(16))) i32x4 lds[kLdsU4];
  const GemmI8& p = q.g;
  const int xcd = (int)(blockIdx.x & 7);
  Walk walk{xcd * q.per_xcd + (int)(blockIdx.x >> 3), min(q.total, (xcd + 1) * q.per_xcd), (int)(gridDim.x >> 3)};
  if (walk.done()) return;
  const int units = (walk.end - walk.u + walk.stride - 1) / walk.stride;
  // (channel tile, row tile) of unit u, in tiles of 256
  auto tile_of = [&](int u, int& nt, int& mt) {
    const int band_tiles = kBand * q.m_tiles;
    const int band = u / band_tiles;
    const int in_band = u - band * band_tiles;
    const int gsz = min(kBand, q.n_tiles - band * kBand);
    mt = in_band / gsz;
    nt = band * kBand + (in_band - mt * gsz);
  };

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int steps = p.k_steps;  // even
  const int all = units * steps;
  const uint32_t l0 = lds_addr(lds);

  // K-steps are counted through all of a workgroup's tiles.  Step i multiplies weight slot
  // i % 3 and row slot (i / 2) % 3.  Before it each loader's loads of what it needs are done
  // and every wave has passed the barrier, which also frees the slots read at step i - 1
  // for what the loaders issue next: while a tile's outputs are stored, the next tile's
  // first steps are on their way.  A tile's scales are loaded before its first step; the
  // waits count steps' loads alone, so that these only make them wait for more.
  if (wave >= 10) {
    // Row loader a: chunk j = 2 v + r (128 bytes of rows 128 r .. + 127 of a tile) into slot
    // v % 3, blocks 16 r + 8 a .. + 7 of 8 rows each.  Chunk j is issued at step j - 4: its
    // slot last held pair v - 3, multiplied up to step 2 v - 5.
    const int a = wave - 10;
    const int piece = (lane & 7) ^ (lane >> 3);
    const int last = (p.K - 1) >> 4;  // a row's last piece: the weight is 0 behind it
    uint32_t off[2][8];
    const uint8_t* xb;
    int tile = 0;
    auto begin = [&](int u) {
      int nt, mt;
      tile_of(u, nt, mt);
      const int m0 = mt * kRows;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int m = 128 * a + 64 * h;
        dma4(p.sx, 4 * (uint32_t)min(m0 + m + lane, p.M - 1), l0 + scales_at(tile) + 4 * (kChannels + m));
      }
      ++tile;
      xb = p.x + (int64_t)m0 * p.xs;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < 8; ++i)
          off[r][i] = (uint32_t)((int64_t)(min(m0 + 128 * r + 8 * (8 * a + i) + (lane >> 3), p.M - 1) - m0) * p.xs);
    };
    begin(walk.u);
    int j = 0, v8 = 0, slot = 0;  // the next chunk, the first piece and the slot of its pair
    int in_tile = 0;              // its step in its tile
    auto chunk = [&]() {
      const uint32_t at = 16 * (uint32_t)min(v8 + piece, last);
      const uint32_t dst = l0 + kRowBase + slot * kRowSlot + (16 * (j & 1) + 8 * a) * 1024;
      if (j & 1) {
#pragma unroll
        for (int i = 0; i < 8; ++i) dma16(xb, off[1][i] + at, dst + i * 1024);
        slot = slot == 2 ? 0 : slot + 1;
        v8 += 8;
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) dma16(xb, off[0][i] + at, dst + i * 1024);
      }
      ++j;
      if (++in_tile == steps && j < all) {
        in_tile = 0;
        v8 = 0;
        walk.u += walk.stride;
        begin(walk.u);
      }
    };
    while (j < 4 && j < all) chunk();
    for (int i = 0; i < all; ++i) {
      wait_chunks(min(i + 4, all) - (2 * (i >> 1) + 2));  // pair i / 2 needs chunks < 2 (i / 2) + 2
      barrier();
      if (j < all) chunk();
    }
    return;
  }
  if (wave >= 8) {
    // Weight loader l: fragments 8 l .. + 7 of step i + 2 after barrier i (tiles past the
    // last are clamped to it; their sums are never stored).
    const int l = wave - 8;
    const uint32_t voff = (uint32_t)(lane * 16);
    int t0 = 0, ks = 0, slot = 0, issued = 0, tile = 0;
    auto begin = [&](int u) {
      int nt, mt;
      tile_of(u, nt, mt);
      t0 = nt * (kChannels / 16);
      ks = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int n = 128 * l + 64 * h;
        dma4(p.sw, 4 * (uint32_t)min(16 * t0 + n + lane, 16 * p.tiles - 1), l0 + scales_at(tile) + 4 * n);
      }
      ++tile;
    };
    begin(walk.u);
    auto stage = [&]() {
      const u32x4* w = p.w + (int64_t)ks * p.tiles * 64;
      const uint32_t dst = l0 + slot * kWeightSlot;
#pragma unroll
      for (int i = 0; i < 8; ++i)
        dma16(w + (int64_t)min(t0 + 8 * l + i, p.tiles - 1) * 64, voff, dst + (8 * l + i) * 1024);
      slot = slot == 2 ? 0 : slot + 1;
      ++issued;
      if (++ks == steps && issued < all) {
        walk.u += walk.stride;
        begin(walk.u);
      }
    };
    stage();
    stage();
    for (int i = 0; i < all; ++i) {
      if (i + 1 < all) wait_vm<8>();
      else wait_vm<0>();
      barrier();
      if (issued < all) stage();
    }
    return;
  }

  const int wr = wave >> 1, wc = wave & 1;
  const int r16 = lane & 15, g = lane >> 4, rr = r16 & 7;
  const int boff0 = (r16 >> 3) * 64 + 8 * rr + (g ^ rr);
  const int boff1 = (r16 >> 3) * 64 + 8 * rr + ((4 + g) ^ rr);
  int ws = 0, xs = 0, tile = 0;  // slots
  for (; !walk.done(); walk.u += walk.stride) {
    int nt, mt;
    tile_of(walk.u, nt, mt);
    const int t0 = nt * (kChannels / 16) + 4 * wr, m0 = mt * kRows + 128 * wc;
    if (t0 >= p.tiles) {  // the wave's sums would never be stored
      for (int i = 0; i < steps; ++i) barrier();
      ws = (ws + steps) % 3;
      xs = (xs + steps / 2) % 3;
      ++tile;
      continue;
    }
    i32x4 acc[4][8] = {};
    for (int i = 0; i < steps; i += 2) {
      barrier();
      const i32x4* xst = lds + kRowBase / 16 + xs * (kRowSlot / 16);
      multiply(lds + ws * (kWeightSlot / 16), xst, wr, wc, lane, boff0, acc);
      ws = ws == 2 ? 0 : ws + 1;
      barrier();
      multiply(lds + ws * (kWeightSlot / 16), xst, wr, wc, lane, boff1, acc);
      ws = ws == 2 ? 0 : ws + 1;
      xs = xs == 2 ? 0 : xs + 1;
    }
    // No load from memory here: one behind a store would wait for the store.
    const float* sw = reinterpret_cast<const float*>(lds) + scales_at(tile) / 4 + 64 * wr + 4 * g;
    const float* sx = reinterpret_cast<const float*>(lds) + scales_at(tile) / 4 + kChannels + 128 * wc + r16;
    ++tile;
    // Where the wave's outputs are all there, an address is a uniform row block's and the
    // lane's offset in it, which no store changes.
    const uint32_t off = (uint32_t)r16 * (uint32_t)p.os + 4 * g;
    auto store = [&](auto WHOLE) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int m = m0 + 16 * j;
        if (!decltype(WHOLE)::value && m + r16 >= p.M) continue;
        T* rows = static_cast<T*>(p.out) + (int64_t)m * p.os;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int t = t0 + 2 * h;
          if (!decltype(WHOLE)::value && t >= p.tiles) continue;
          const f32x4 sa = *reinterpret_cast<const f32x4*>(sw + 32 * h), sb = *reinterpret_cast<const f32x4*>(sw + 32 * h + 16);
          store_pair<T, GATED, decltype(WHOLE)::value>(p, t, g, rows, off, acc[2 * h][j], acc[2 * h + 1][j], sa, sb, sx[16 * j]);
        }
      }
    };
    if (m0 + 128 <= p.M && (GATED ? 8 : 16) * (t0 + 4) <= p.cols)
      store(std::true_type{});
    else
      store(std::false_type{});
  }
}

}  // namespace

template <typename T, bool GATED>
hipError_t launch_prompt_i8(const GemmI8& p, hipStream_t s) {
  PromptI8 q{};
  q.g = p;
  q.n_tiles = (int)ceil_div(p.tiles, kChannels / 16);
  q.m_tiles = (int)ceil_div(p.M, kRows);
  q.total = q.n_tiles * q.m_tiles;
  q.per_xcd = (int)ceil_div(q.total, 8);
  const int slots = std::max(device_cus() / 8, 1);  // a workgroup's LDS takes a compute unit
  hipLaunchKernelGGL((prompt_i8_kernel<T, GATED>), dim3((unsigned)(8 * std::min(q.per_xcd, slots))), dim3(kThreads), 0, s, q);
  return hipGetLastError();
}

template hipError_t launch_prompt_i8<float, false>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<float, true>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<uint16_t, false>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<uint16_t, true>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<_Float16, false>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<_Float16, true>(const GemmI8&, hipStream_t);

}  // namespace dflash
