// 8-bit products of many rows: a prompt's projections, or a few draft blocks'.
//
// A workgroup computes a tile of 64 WR channels x 16 RT WC rows; both operands are staged in
// LDS by direct global -> LDS loads of waves that do nothing else.
//   - Compute wave (wr, wc) owns channel tiles 4 wr .. 4 wr + 3 against row tiles RT wc ..
//     RT wc + RT - 1: 4 RT products of 16 x 16 x 64 a k-step of 64.
//   - Weight stages: one k-step's 4 WR fragments (contiguous in the packed weight), 8 a
//     loader wave; three slots.
//   - Row stages: 128 bytes of each of the rows, in two chunks of half the rows, 8 loads a
//     loader wave each, a load 8 whole rows of 128 bytes; three slots.  A block of 8 rows
//     takes 1 KB of LDS, 16-byte piece c of row r at slot 8 r + (c ^ r), so the 8 lanes that
//     read one piece of 8 rows touch all banks once.
//   - One barrier a k-step, which all waves keep.
//   - Products of few tiles split K over workgroups, whose sums (integers: the same bits)
//     another launch adds up.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "int8_common.h"
#include "lds_dma.h"

namespace dflash {
namespace {

constexpr int kBandChannels = 4096;  // channels per band of the tile walk

// A tile's shape and what follows from it.
template <int WR_, int WC_, int RT_, int WS_, int RS_, int LPL_, bool SPLITS_>
struct Shape {
  // RT: row tiles of 16 a wave; WS, RS: slots of weights and rows
  static constexpr int WR = WR_, WC = WC_, RT = RT_, WS = WS_, RS = RS_;
  static constexpr int LPL = LPL_;  // loads a loader wave and step
  static constexpr bool kSplits = SPLITS_;  // may K be split over workgroups
  static constexpr int kRows = 16 * RT * WC, kChannels = 64 * WR, kBand = kBandChannels / kChannels;
  static constexpr int kCompute = WR * WC, kWeightLoaders = 4 * WR / LPL, kRowLoaders = kRows / 16 / LPL;
  static constexpr int kGroup = kCompute + kWeightLoaders + kRowLoaders;  // waves
  static constexpr int kThreads = 64 * kGroup;
  static constexpr int kWavesPerSimd = kCompute == 8 ? 3 : 4;  // one workgroup a compute unit, or two
  static constexpr int kWeightSlot = 4096 * WR, kRowSlot = 128 * kRows;
  static constexpr int kWeightLead = WS - 1, kRowLead = 2 * (RS - 1);  // k-steps that the loaders are ahead
  static constexpr int kRowBase = WS * kWeightSlot;
  static constexpr int kScaleBase = kRowBase + RS * kRowSlot;
  static constexpr int kScaleSlot = 4 * (kChannels + kRows);  // a tile's channel and row scales
  // The slot of tile t is written kRowLead + 1 steps before tile t begins at the earliest, and
  // its last tile's outputs are stored before the tile after that has begun; a tile has two
  // steps at least.
  static constexpr int kScaleSlots = 2 * 3 >= kRowLead + 1 ? 4 : 8;
  static_assert(2 * (kScaleSlots - 1) >= kRowLead + 1 && kRowLead <= 6 && kWeightLead <= 6, "leads");
  static constexpr int kLdsU4 = (kScaleBase + kScaleSlots * kScaleSlot) / 16;
};

// 256 x 256: half the bytes per product; 128 of its 168 registers are sums, and 6 that the
// outputs need wait in scratch (written once, read once a tile).
// 128 x 128: two workgroups a compute unit, one's
// products beside the other's waits; four loads a loader wave, whose issue the small tile's
// k-step waited for (40 against 48 us for a step chain of 144).
using Wide = Shape<4, 2, 8, 3, 3, 8, false>;
using Narrow = Shape<2, 2, 4, 3, 3, 4, true>;

struct PromptI8 {
  GemmI8 g;
  int n_tiles, m_tiles, tiles, total, per_xcd;
  int split_steps;  // k-steps of a split (even); p.k_steps: no split
  int32_t* part;    // split: [split][M][16 tiles of channels] sums
};

__device__ __forceinline__ void barrier() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// Wait until at most n groups of LPL loads of this wave are outstanding (n <= 6).
template <int LPL>
__device__ __forceinline__ void wait_groups(int n) {
  if (n <= 0) wait_vm<0>();
  else if (n == 1) wait_vm<LPL>();
  else if (n == 2) wait_vm<2 * LPL>();
  else if (n == 3) wait_vm<3 * LPL>();
  else if (n == 4) wait_vm<4 * LPL>();
  else if (n == 5) wait_vm<5 * LPL>();
  else wait_vm<6 * LPL>();
}

// A k-step's fragments of a wave: four channel tiles' and four row tiles'.
struct Fragments {
  i32x4 a[4], b[4];
};
__device__ __forceinline__ void read_weights(Fragments& f, const i32x4* w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) f.a[i] = w[i * 64];
}
__device__ __forceinline__ void read_rows(Fragments& f, const i32x4* x) {
#pragma unroll
  for (int j = 0; j < 4; ++j) f.b[j] = x[2 * j * 64];
}
// Row tiles J .. J + 3.
template <int J, int RT>
__device__ __forceinline__ void multiply(const Fragments& f, i32x4 (&acc)[4][RT]) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      acc[i][J + j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.a[i], f.b[j], acc[i][J + j], 0, 0, 0);
}

// The tiles of a workgroup: every n_slots-th of its XCD's range.
struct Walk {
  int u, end, stride;
  __device__ bool done() const { return u >= end; }
};

// GATED and T do not matter where SPLIT.
template <typename T, bool GATED, bool SPLIT, typename S>
__global__ __launch_bounds__(S::kThreads, S::kWavesPerSimd) void prompt_i8_kernel(const PromptI8 q) {
  constexpr int kRows = S::kRows, kChannels = S::kChannels, kBand = S::kBand, RT = S::RT, LPL = S::LPL, kBlocks = S::kRows / 16;  // of 8 rows, a chunk
  __shared__ __attribute__((aligned(16))) i32x4 lds[S::kLdsU4];
  auto scales_at = [](int t) -> uint32_t { return S::kScaleBase + (t & (S::kScaleSlots - 1)) * S::kScaleSlot; };
  const GemmI8& p = q.g;
  const int xcd = (int)(blockIdx.x & 7);
  Walk walk{xcd * q.per_xcd + (int)(blockIdx.x >> 3), min(q.total, (xcd + 1) * q.per_xcd), (int)(gridDim.x >> 3)};
  if (walk.done()) return;
  const int units = SPLIT ? 1 : (walk.end - walk.u + walk.stride - 1) / walk.stride;
  // (channel tile, row tile) of unit u, in the shape's tiles
  auto tile_of = [&](int u, int& nt, int& mt) {
    if (SPLIT) u %= q.tiles;
    const int band_tiles = kBand * q.m_tiles;
    const int band = u / band_tiles;
    const int in_band = u - band * band_tiles;
    const int gsz = min(kBand, q.n_tiles - band * kBand);
    mt = in_band / gsz;
    nt = band * kBand + (in_band - mt * gsz);
  };

  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int split = SPLIT ? walk.u / q.tiles : 0;
  const int k0 = split * q.split_steps;
  const int steps = min(q.split_steps, p.k_steps - k0);  // even
  const int all = units * steps;
  const uint32_t l0 = lds_addr(lds);

  // K-steps are counted through all of a workgroup's tiles.  Step i multiplies weight slot
  // i % WS and row slot (i / 2) % RS.  Before it each loader's loads of what it needs are done
  // and every wave has passed the barrier, a compute wave with its reads done (read_barrier), which
  // frees the slots read at step i - 1 for what the loaders issue next: while a tile's outputs are stored, the next tile's
  // first steps are on their way.  A tile's scales are loaded before its first step; the
  // waits count steps' loads alone, so that these only make them wait for more.
  if (wave >= S::kCompute + S::kWeightLoaders) {
    // Row loader a: chunk j = 2 v + r (128 bytes of half r of a tile's rows) into slot v % RS,
    // blocks kBlocks r + LPL a .. of 8 rows each.  Chunk j is issued after barrier j - kRowLead:
    // its slot last held pair v - RS, multiplied up to step 2 v - 2 RS + 1.
    const int a = wave - S::kCompute - S::kWeightLoaders;
    const int piece = (lane & 7) ^ (lane >> 3);
    const int last = (p.K - 1) >> 4;  // a row's last piece: the weight is 0 behind it
    uint32_t off[2][LPL];
    const uint8_t* xb;
    int tile = 0;
    auto begin = [&](int u) {
      int nt, mt;
      tile_of(u, nt, mt);
      const int m0 = mt * kRows;
#pragma unroll
      for (int h = 0; h < LPL / 4; ++h) {
        const int m = 16 * LPL * a + 64 * h;
        dma4(p.sx, 4 * (uint32_t)min(m0 + m + lane, p.M - 1), l0 + scales_at(tile) + 4 * (kChannels + m));
      }
      ++tile;
      xb = p.x + (int64_t)m0 * p.xs;
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int i = 0; i < LPL; ++i)
          off[r][i] = (uint32_t)((int64_t)(min(m0 + 8 * (kBlocks * r + LPL * a + i) + (lane >> 3), p.M - 1) - m0) * p.xs);
    };
    begin(walk.u);
    int j = 0, v8 = 4 * k0, slot = 0;  // the next chunk, the first piece and the slot of its pair
    int in_tile = 0;                   // its step in its tile
    auto chunk = [&]() {
      const uint32_t at = 16 * (uint32_t)min(v8 + piece, last);
      const uint32_t dst = l0 + S::kRowBase + slot * S::kRowSlot + (kBlocks * (j & 1) + LPL * a) * 1024;
      if (j & 1) {
#pragma unroll
        for (int i = 0; i < LPL; ++i) dma16(xb, off[1][i] + at, dst + i * 1024);
        slot = slot == S::RS - 1 ? 0 : slot + 1;
        v8 += 8;
      } else {
#pragma unroll
        for (int i = 0; i < LPL; ++i) dma16(xb, off[0][i] + at, dst + i * 1024);
      }
      ++j;
      if (++in_tile == steps && j < all) {
        in_tile = 0;
        v8 = 4 * k0;
        walk.u += walk.stride;
        begin(walk.u);
      }
    };
    while (j < S::kRowLead && j < all) chunk();
    for (int i = 0; i < all; ++i) {
      wait_groups<S::LPL>(min(i + S::kRowLead, all) - (2 * (i >> 1) + 2));  // pair i / 2 needs chunks < 2 (i / 2) + 2
      barrier();
      if (j < all) chunk();
    }
    return;
  }
  if (wave >= S::kCompute) {
    // Weight loader l: fragments LPL l .. of step i + kWeightLead after barrier i (tiles past
    // the last are clamped to it; their sums are never stored).
    const int l = wave - S::kCompute;
    const uint32_t voff = (uint32_t)(lane * 16);
    int t0 = 0, ks = 0, slot = 0, issued = 0, tile = 0;
    auto begin = [&](int u) {
      int nt, mt;
      tile_of(u, nt, mt);
      t0 = nt * (kChannels / 16);
      ks = k0;
#pragma unroll
      for (int h = 0; h < LPL / 4; ++h) {
        const int n = 16 * LPL * l + 64 * h;
        dma4(p.sw, 4 * (uint32_t)min(16 * t0 + n + lane, 16 * p.tiles - 1), l0 + scales_at(tile) + 4 * n);
      }
      ++tile;
    };
    begin(walk.u);
    auto stage = [&]() {
      const u32x4* w = p.w + (int64_t)ks * p.tiles * 64;
      const uint32_t dst = l0 + slot * S::kWeightSlot;
#pragma unroll
      for (int i = 0; i < LPL; ++i)
        dma16(w + (int64_t)min(t0 + LPL * l + i, p.tiles - 1) * 64, voff, dst + (LPL * l + i) * 1024);
      slot = slot == S::WS - 1 ? 0 : slot + 1;
      ++issued;
      if (++ks == k0 + steps && issued < all) {
        walk.u += walk.stride;
        begin(walk.u);
      }
    };
    while (issued < S::kWeightLead && issued < all) stage();
    for (int i = 0; i < all; ++i) {
      wait_groups<S::LPL>(min(i + S::kWeightLead, all) - (i + 1));
      barrier();
      if (issued < all) stage();
    }
    return;
  }

  const int wr = wave / S::WC, wc = wave % S::WC;
  const int r16 = lane & 15, g = lane >> 4, rr = r16 & 7;
  const int boff = 2 * RT * wc * 64 + (r16 >> 3) * 64 + 8 * rr;
  const int boff0 = boff + (g ^ rr), boff1 = boff + ((4 + g) ^ rr);
  const i32x4* wfrag = lds + 4 * wr * 64 + lane;
  int ws = 0, xs = 0, tile = 0;  // slots
  auto whole_step = [&](const i32x4* w, const i32x4* x, i32x4 (&acc)[4][RT]) __attribute__((always_inline)) {
    Fragments f;
    read_weights(f, w);
    read_rows(f, x);
    multiply<0>(f, acc);
    if constexpr (RT == 8) {
      read_rows(f, x + 8 * 64);
      multiply<4>(f, acc);
    }
  };
  for (; tile < units; walk.u += walk.stride) {
    int nt, mt;
    tile_of(walk.u, nt, mt);
    const int t0 = nt * (kChannels / 16) + 4 * wr, m0 = mt * kRows + 16 * RT * wc;
    i32x4 acc[4][RT];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < RT; ++j) acc[i][j] = i32x4{0, 0, 0, 0};
    if (t0 >= p.tiles) {  // the wave's sums would never be stored
      for (int i = 0; i < steps; ++i) read_barrier();
      ws = (ws + steps) % S::WS;
      xs = (xs + steps / 2) % S::RS;
      ++tile;
      continue;
    } else {
      for (int i = 0; i < steps; i += 2) {
        const i32x4* xst = lds + S::kRowBase / 16 + xs * (S::kRowSlot / 16);
        read_barrier();
        whole_step(wfrag + ws * (S::kWeightSlot / 16), xst + boff0, acc);
        ws = ws == S::WS - 1 ? 0 : ws + 1;
        read_barrier();
        whole_step(wfrag + ws * (S::kWeightSlot / 16), xst + boff1, acc);
        ws = ws == S::WS - 1 ? 0 : ws + 1;
        xs = xs == S::RS - 1 ? 0 : xs + 1;
      }
    }
    if (SPLIT) {
      int32_t* part = q.part + ((int64_t)split * p.M + m0) * 16 * p.tiles + 16 * t0 + 4 * g;
#pragma unroll
      for (int j = 0; j < RT; ++j) {
        if (m0 + 16 * j + r16 >= p.M) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (t0 + i < p.tiles) *reinterpret_cast<i32x4*>(part + (int64_t)(16 * j + r16) * 16 * p.tiles + 16 * i) = acc[i][j];
      }
      return;
    }
    // No load from memory here: one behind a store would wait for the store.
    const float* sw = reinterpret_cast<const float*>(lds) + scales_at(tile) / 4 + 64 * wr + 4 * g;
    const float* sx = reinterpret_cast<const float*>(lds) + scales_at(tile) / 4 + kChannels + 16 * RT * wc + r16;
    ++tile;
    // Where the wave's outputs are all there, an address is a uniform row block's and the
    // lane's offset in it, which no store changes.
    const uint32_t off = (uint32_t)r16 * (uint32_t)p.os + 4 * g;
    auto store = [&](auto WHOLE) {
#pragma unroll
      for (int j = 0; j < RT; ++j) {
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
    if (m0 + 16 * RT <= p.M && (GATED ? 8 : 16) * (t0 + 4) <= p.cols)
      store(std::true_type{});
    else
      store(std::false_type{});
  }
}

}  // namespace

// The splits' sums to outputs: a thread four channels of a tile (a gate's and its up's) of a row.
template <typename T, bool GATED>
__global__ __launch_bounds__(256) void join_i8_kernel(const GemmI8 p, const int32_t* part, int splits) {
  const int per_row = (GATED ? p.tiles / 2 : p.tiles) * 4;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (int64_t)per_row * p.M) return;
  const int m = (int)(i / per_row), c = (int)(i - (int64_t)m * per_row);
  const int t = GATED ? 2 * (c >> 2) : c >> 2, g = c & 3;
  const int64_t slab = (int64_t)p.M * 16 * p.tiles;
  const int32_t* at = part + (int64_t)m * 16 * p.tiles + 16 * t + 4 * g;
  i32x4 a{0, 0, 0, 0}, b{0, 0, 0, 0};
#pragma unroll 4
  for (int s = 0; s < splits; ++s) {
    a += *reinterpret_cast<const i32x4*>(at + s * slab);
    if (GATED) b += *reinterpret_cast<const i32x4*>(at + s * slab + 16);
  }
  const f32x4 sa = tile_scales(p, t, g), sb = tile_scales(p, t + 1, g);
  const float sx = p.sx[m];
  float v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    v[e] = (float)a[e] * sa[e] * sx;
    if (GATED) v[e] = silu(v[e]) * ((float)b[e] * sb[e] * sx);
  }
  store_cols<T, false>(p, static_cast<T*>(p.out) + (int64_t)m * p.os, 4 * g, GATED ? 8 * t : 16 * t, g, v);
}

template <typename S, typename T, bool GATED>
hipError_t launch_shape(const GemmI8& p, int splits, hipStream_t s) {
  PromptI8 q{};
  q.g = p;
  q.n_tiles = (int)ceil_div(p.tiles, S::kChannels / 16);
  q.m_tiles = (int)ceil_div(p.M, S::kRows);
  q.tiles = q.n_tiles * q.m_tiles;
  q.split_steps = 2 * (int)ceil_div(p.k_steps / 2, splits);
  splits = (int)ceil_div(p.k_steps, q.split_steps);
  q.total = q.tiles * splits;
  q.per_xcd = (int)ceil_div(q.total, 8);
  if constexpr (S::kSplits) {
    if (splits > 1) {
      q.part = static_cast<int32_t*>(p.workspace);
      hipLaunchKernelGGL((prompt_i8_kernel<float, false, true, S>), dim3((unsigned)(8 * q.per_xcd)), dim3(S::kThreads), 0,
                         s, q);
      const int64_t threads = (int64_t)p.M * (GATED ? p.tiles / 2 : p.tiles) * 4;
      hipLaunchKernelGGL((join_i8_kernel<T, GATED>), dim3((unsigned)ceil_div(threads, 256)), dim3(256), 0, s, p, q.part,
                         splits);
      return hipGetLastError();
    }
  }
  // as many workgroups as the compute units' LDS holds walk the tiles
  const int slots = std::max(device_cus() * (160 * 1024 / (16 * S::kLdsU4)) / 8, 1);
  hipLaunchKernelGGL((prompt_i8_kernel<T, GATED, false, S>), dim3((unsigned)(8 * std::min(q.per_xcd, slots))),
                     dim3(S::kThreads), 0, s, q);
  return hipGetLastError();
}

template <typename T, bool GATED>
hipError_t launch_prompt_i8(const GemmI8& p, hipStream_t s) {
  if (p.plan.kind == PlanI8::kWide) return launch_shape<Wide, T, GATED>(p, 1, s);
  return launch_shape<Narrow, T, GATED>(p, p.plan.splits, s);
}

template hipError_t launch_prompt_i8<float, false>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<float, true>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<uint16_t, false>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<uint16_t, true>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<_Float16, false>(const GemmI8&, hipStream_t);
template hipError_t launch_prompt_i8<_Float16, true>(const GemmI8&, hipStream_t);

}  // namespace dflash
