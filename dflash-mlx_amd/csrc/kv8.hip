// The 8-bit key/value cache: append (with the query / key norm and rotary in
// front of it), load and read back (include/dflash_kv8.h).
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>
#include <stdint.h>

#include "kv8_common.h"

namespace dflash {
namespace {

constexpr int kRow = kHD + 8;  // bf16 of a token's row in LDS (16 bytes of pad)

// Quantise block j of head bh from the tail: a thread holds 32 neighbouring
// values of the block in its stored order (keys [64][128], values [128][64]).
template <int TYPE>
__device__ __forceinline__ void quantise_tail_block(const Kv8& c, int64_t bh, int j, bool values, uint32_t* red) {
  const int t = threadIdx.x;
  const int at = (j & 1) * kBlk;
  const uint16_t* src = values ? c.tail_values(bh) + (t >> 1) * kSlots + at + (t & 1) * 32
                               : c.tail_keys(bh) + (at + (t >> 2)) * kHD + (t & 3) * 32;
  u32x4 w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = ld16(src + 8 * i);
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) a = max(a, abs_bits16(w[i]));
  const f32x2 sm = block_scale<TYPE>(group_max_u32(a, red));
  uint8_t* dst = (values ? c.values(bh, j) : c.keys(bh, j)) + 32 * t;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const u32x2 lo = quantise8<TYPE>(w[2 * i], sm.y), hi = quantise8<TYPE>(w[2 * i + 1], sm.y);
    *reinterpret_cast<u32x4*>(dst + 16 * i) = u32x4{lo.x, lo.y, hi.x, hi.y};
  }
  if (t == 0) (values ? c.vs : c.ks)[bh * c.nblk + j] = sm.x;
}

// Block L / 64 - 1 may have become complete since the last append: with L past the cache's
// end by a draft block's tokens, its last block.
__device__ __forceinline__ bool may_wait(int L, int Smax) {
  return L >= kBlk && L - kMaxDraft <= Smax && (L & 63) <= kMaxDraft;
}
__device__ __forceinline__ int waiting_block(int L, int Smax) { return (min(L, Smax) >> 6) - 1; }

// A block's 64 rows in registers: piece i of a thread is token tid / 16 + 16 i, features
// 8 (tid % 16) .. + 7.
struct Rows {
  u32x4 x[4];
};

// Four dwords as four rows of bytes, transposed.
__device__ __forceinline__ void transpose4(uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
  const uint32_t ab0 = __builtin_amdgcn_perm(b, a, 0x05010400u), ab2 = __builtin_amdgcn_perm(b, a, 0x07030602u);
  const uint32_t cd0 = __builtin_amdgcn_perm(d, c, 0x05010400u), cd2 = __builtin_amdgcn_perm(d, c, 0x07030602u);
  a = __builtin_amdgcn_perm(cd0, ab0, 0x05040100u);
  b = __builtin_amdgcn_perm(cd0, ab0, 0x07060302u);
  c = __builtin_amdgcn_perm(cd2, ab2, 0x05040100u);
  d = __builtin_amdgcn_perm(cd2, ab2, 0x07060302u);
}

// LDS of a block's values on their way from [position][feature] to [feature][position] or
// back: codes, rows of 33 dwords (a wave's dwords of 8 rows 8 apart, 8 side by side each,
// fall into 64 banks), or bf16.
struct Turn {
  union {
    uint32_t codes[kBlk][kHD / 4 + 1];
    uint16_t rows[kBlk][kRow];
  };
};

// The codes of a block whose rows are in registers.  Values are stored transposed: a
// thread turns 4 features x 8 positions, so that eight lanes store a feature's 64 bytes.
template <int TYPE>
__device__ __forceinline__ void store_codes(const Kv8& c, int64_t bh, int j, bool values, const Rows& r, Turn& lds,
                                            uint32_t* red) {
  const int t = threadIdx.x;
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) a = max(a, abs_bits16(r.x[i]));
  const f32x2 sm = block_scale<TYPE>(group_max_u32(a, red));
  if (t == 0) (values ? c.vs : c.ks)[bh * c.nblk + j] = sm.x;
  if (!values) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<u32x2*>(c.keys(bh, j) + 8 * (t + 256 * i)) = quantise8<TYPE>(r.x[i], sm.y);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32x2 q = quantise8<TYPE>(r.x[i], sm.y);
    uint32_t* dst = &lds.codes[(t >> 4) + 16 * i][2 * (t & 15)];
    dst[0] = q.x;
    dst[1] = q.y;
  }
  __syncthreads();
  const int p0 = 8 * (t & 7), quad = t >> 3;
  uint32_t w[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = lds.codes[p0 + i][quad];
  transpose4(w[0], w[1], w[2], w[3]);
  transpose4(w[4], w[5], w[6], w[7]);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    *reinterpret_cast<u32x2*>(c.values(bh, j) + (4 * quad + i) * kBlk + p0) = u32x2{w[i], w[4 + i]};
  __syncthreads();
}

// The rows of block j at positions [from, to) into the tail: values turned, 8 positions a
// store (one by one, a load of 4 sequences of 8192 took 42 us for 18: the last block's
// workgroup outlasted the rest).
__device__ __forceinline__ void store_tail(const Kv8& c, int64_t bh, int j, bool values, const Rows& r, int from, int to,
                                           Turn& lds) {
  const int t = threadIdx.x;
  if (!values) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int pos = kBlk * j + (t >> 4) + 16 * i;
      if (pos >= from && pos < to)
        *reinterpret_cast<u32x4*>(c.tail_keys(bh) + (pos & (kSlots - 1)) * kHD + 8 * (t & 15)) = r.x[i];
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) *reinterpret_cast<u32x4*>(&lds.rows[(t >> 4) + 16 * i][8 * (t & 15)]) = r.x[i];
  __syncthreads();
  uint16_t* dst = c.tail_values(bh) + (t >> 1) * kSlots + (j & 1) * kBlk;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const int tk = (t & 1) * 32 + 8 * g, pos = kBlk * j + tk;
    if (pos >= from && pos + 8 <= to) {
      u32x4 w;
#pragma unroll
      for (int u = 0; u < 4; ++u)
        w[u] = lds.rows[tk + 2 * u][t >> 1] | ((uint32_t)lds.rows[tk + 2 * u + 1][t >> 1] << 16);
      *reinterpret_cast<u32x4*>(dst + tk) = w;
    } else {
      for (int i = 0; i < 8; ++i)
        if (pos + i >= from && pos + i < to) dst[tk + i] = lds.rows[tk + i][t >> 1];
    }
  }
  __syncthreads();
}

struct AppendParams {
  Kv8 c;
  const uint16_t* proj;  // [B*T, row_stride]: Hq x (q | gate), Hkv x k, Hkv x v
  int64_t row_stride;
  const uint16_t* q_norm_w;
  const uint16_t* k_norm_w;
  const int32_t* lens;
  uint16_t* q_out;
  int32_t* overflow;
  int T, Hq, rot;
  int nb;      // prompt: block tasks of a head
  int qtiles;  // prompt: 16-token query tiles of a sequence
  float eps;
  double freq[kHD / 2];  // base^(-2i/rot), i < rot / 2
};

// A head's row is held by 16 lanes, lane f of them features 8 f .. 8 f + 7 (16 bytes):
// a wave normalizes and rotates four rows at a time, the sum of squares takes four DPP
// adds, and the square root and division serve four rows.
//
// Cosine and sine of position pos at one frequency: the angle less its multiple of pi / 2
// in fp64, then the Taylor series of both on [-pi / 4, pi / 4] in fp32 (the first terms left
// out are below 2e-9), with what the reduced angle's rounding to fp32 loses put back to first
// order.  Right to about an fp32 step at any position.
__device__ __forceinline__ f32x2 cos_sin(int pos, double freq) {
  const double half_pi = 1.5707963267948966192313216916398;
  const double a = (double)pos * freq;
  const double n = rint(a * (1.0 / half_pi));
  const double r = fma(-n, half_pi, a);
  const float x = (float)r, lo = (float)(r - (double)x), z = x * x;
  float s = fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  s = fmaf(z, s, 1.f / 120.f);
  s = fmaf(z, s, -1.f / 6.f);
  s = fmaf(z * x, s, x);
  float c = fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  c = fmaf(z, c, -1.f / 720.f);
  c = fmaf(z, c, 1.f / 24.f);
  c = fmaf(z, c, -0.5f);
  c = fmaf(z, c, 1.f);
  const float sn = fmaf(c, lo, s), cs = fmaf(-s, lo, c);
  const int q = (int)((int64_t)n & 3);  // quarter turns
  const float u = q & 1 ? sn : cs, v = q & 1 ? cs : sn;
  return f32x2{q == 1 || q == 2 ? -u : u, q >= 2 ? -v : v};
}

// The cosines and sines of N positions pos0 .. in LDS: [N][rot / 2] each, all
// cosines first.  A thread keeps one frequency (256 is a multiple of rot / 2).
template <int N>
__device__ __forceinline__ void rotation_table(float* table, int pos0, const AppendParams& p) {
  if (p.rot == 0) return;
  const int half = p.rot >> 1, shift = __builtin_ctz(half);
  const int i = threadIdx.x & (half - 1);
  const double freq = p.freq[i];
#pragma unroll 2
  for (int t = threadIdx.x >> shift; t < N; t += 256 >> shift) {
    const f32x2 cs = cos_sin(pos0 + t, freq);
    table[t * half + i] = cs.x;
    table[(N + t) * half + i] = cs.y;
  }
}

constexpr int kDppQuadReverse = 0x1B;  // quad_perm [3,2,1,0]

// RMSNorm and rotary of a row's eight features at lane f: cosines cs[rot / 2], sines
// sn[rot / 2].  fp32 throughout, rounded to bf16 once.
__device__ __forceinline__ u32x4 norm_rotate8(u32x4 xw, u32x4 ww, const float* cs, const float* sn, int f, int rot,
                                              float eps) {
  float x[8], w[8];
  unpack8(xw, x);
  unpack8(ww, w);
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
  const float inv = 1.f / sqrtf(row16_sum(ss) / (float)kHD + eps);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = x[i] * inv * w[i];
  if (rot > 0) {
    // the other half of the pair: lane f ^ (rot / 16) of the row
    float y[8];
    if (rot == 32) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = dpp_mov<kDppQuadSwap2>(x[i]);
    } else if (rot == 16) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = dpp_mov<kDppQuadSwap1>(x[i]);
    } else if (rot == 64) {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = dpp_mov<kDppQuadReverse>(dpp_mov<kDppRowHalfMirror>(x[i]));  // f ^ 7 ^ 3
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = dpp_mov<kDppRowHalfMirror>(dpp_mov<kDppRowMirror>(x[i]));  // f ^ 15 ^ 7
    }
    if (8 * f < rot) {
      const int half = rot >> 1;
      const bool low = 8 * f < half;
      const int i0 = low ? 8 * f : 8 * f - half;
      f32x4 c[2], s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        c[i] = *reinterpret_cast<const f32x4*>(cs + i0 + 4 * i);
        s[i] = *reinterpret_cast<const f32x4*>(sn + i0 + 4 * i);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = fmaf(x[i], c[i >> 2][i & 3], (low ? -y[i] : y[i]) * s[i >> 2][i & 3]);
    }
  }
  return cvt8_bf16(x);
}

// ------------------------------------------------------------ draft append
// Workgroups 0 .. 2 B Hkv - 1: the waiting block of one head, keys or values, if
// any (16 KB of the tail in, 8 KB of codes out).  The others: 16 heads of a token, keys
// and values to the tail.
// The tail's slots that a waiting block is read from are not written by the same
// call: it waits only where L % 64 <= 16, and the at most 16 new tokens then stay in
// block L / 64, the other half of the slots.
// A few KB a head, bound by latency: 32 sequences of one token, 16 heads on 4, 4.1 us.
template <int TYPE>
__global__ __launch_bounds__(256) void kv8_append_draft_kernel(const AppendParams p) {
  __shared__ uint32_t red[4];
  __shared__ __attribute__((aligned(16))) float table[kHD];
  const Kv8& c = p.c;
  const int nquant = 2 * c.B * c.Hkv;
  if ((int)blockIdx.x < nquant) {
    const int64_t bh = blockIdx.x >> 1;
    const int L = p.lens[bh / c.Hkv];
    if (may_wait(L, c.Smax)) quantise_tail_block<TYPE>(c, bh, waiting_block(L, c.Smax), blockIdx.x & 1, red);
    return;
  }
  const int slots = p.Hq + 2 * c.Hkv, groups = (slots + 15) >> 4;
  const int wg = blockIdx.x - nquant;
  const int bt = wg / groups;
  const int tid = threadIdx.x, f = tid & 15;
  const int slot = (wg - bt * groups) * 16 + (tid >> 4);
  const int b = bt / p.T;
  const int L = p.lens[b];
  const int pos = L + (bt - b * p.T);
  const bool in_cache = L >= 0 && L <= c.Smax && pos < c.Smax;
  if (!in_cache && slot == 0 && f == 0 && p.overflow != nullptr) p.overflow[b] = 1;
  const bool is_q = slot < p.Hq, is_k = !is_q && slot < p.Hq + c.Hkv;
  const int head = is_q ? 2 * slot : p.Hq + slot;  // in units of 128 of the row: q | gate, k, v
  u32x4 x = {0u, 0u, 0u, 0u}, w = x;
  if (slot < slots) {
    x = ld16(p.proj + (int64_t)bt * p.row_stride + head * kHD + 8 * f);
    const uint16_t* wsrc = (is_q ? p.q_norm_w : p.k_norm_w) + 8 * f;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(wsrc)[i];
  }
  if (tid < p.rot >> 1) {
    const f32x2 cs = cos_sin(pos, p.freq[tid]);
    table[tid] = cs.x;
    table[(p.rot >> 1) + tid] = cs.y;
  }
  __syncthreads();
  const u32x4 y = norm_rotate8(x, w, table, table + (p.rot >> 1), f, p.rot, p.eps);
  const int at = pos & (kSlots - 1);
  if (is_q) {
    *reinterpret_cast<u32x4*>(p.q_out + ((int64_t)bt * p.Hq + slot) * kHD + 8 * f) = y;
  } else if (is_k) {
    if (in_cache)
      *reinterpret_cast<u32x4*>(c.tail_keys((int64_t)b * c.Hkv + slot - p.Hq) + at * kHD + 8 * f) = y;
  } else if (slot < slots && in_cache) {
    uint16_t* col = c.tail_values((int64_t)b * c.Hkv + slot - p.Hq - c.Hkv) + 8 * f * kSlots + at;
#pragma unroll
    for (int i = 0; i < 8; ++i) col[i * kSlots] = (uint16_t)(x[i >> 1] >> (16 * (i & 1)));
  }
}

// ----------------------------------------------------------- prompt append
// Block j's 64 rows of head h: positions of this call from proj (keys normalized and
// rotated), earlier ones from the tail, others zero.
__device__ __forceinline__ Rows prompt_rows(const AppendParams& p, int b, int h, int L, int j, bool values, Turn& lds,
                                            float* table) {
  const Kv8& c = p.c;
  const int64_t bh = (int64_t)b * c.Hkv + h;
  const int tid = threadIdx.x, f = tid & 15;
  const int end = min(L + p.T, c.Smax);
  const uint16_t* proj = p.proj + (int64_t)b * p.T * p.row_stride + (2 * p.Hq + h + (values ? c.Hkv : 0)) * kHD + 8 * f;
  Rows r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int pos = kBlk * j + (tid >> 4) + 16 * i;
    r.x[i] = u32x4{0u, 0u, 0u, 0u};
    if (pos >= L && pos < end)
      r.x[i] = ld16(proj + (int64_t)(pos - L) * p.row_stride);
    else if (pos < L && !values)
      r.x[i] = ld16(c.tail_keys(bh) + (pos & (kSlots - 1)) * kHD + 8 * f);
  }
  if (values) {
    if (kBlk * j >= L) return r;
    // the tail's values are transposed: thread (feature, 32 slots)
    const uint16_t* src = c.tail_values(bh) + (tid >> 1) * kSlots + (j & 1) * kBlk + (tid & 1) * 32;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const u32x4 w = ld16(src + 8 * i);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        lds.rows[(tid & 1) * 32 + 8 * i + u][tid >> 1] = (uint16_t)(w[u >> 1] >> (16 * (u & 1)));
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int tk = (tid >> 4) + 16 * i;
      if (kBlk * j + tk < L) r.x[i] = *reinterpret_cast<const u32x4*>(&lds.rows[tk][8 * f]);
    }
    __syncthreads();
    return r;
  }
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p.k_norm_w + 8 * f)[i];
  rotation_table<kBlk>(table, kBlk * j, p);
  __syncthreads();
  const int half = p.rot >> 1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int tk = (tid >> 4) + 16 * i, pos = kBlk * j + tk;
    const u32x4 y = norm_rotate8(r.x[i], w, table + tk * half, table + (kBlk + tk) * half, f, p.rot, p.eps);
    if (pos >= L && pos < end) r.x[i] = y;
  }
  __syncthreads();  // the table may be written again
  return r;
}

// Workgroups: nb block tasks for the keys and nb for the values of every head, then
// 16 tokens x 4 query heads each.  Task i has block L / 64 + i: its codes if the prompt
// completes it, its rows to the tail if it is one of the last two.  Where something is
// read from the tail (a waiting block, the first block's earlier positions), task 0 alone
// touches it: it reads first and stores the last two blocks' rows, which take the same
// slots, afterwards.  Dynamic LDS: the rotation table, 64 rot floats.
// 4096 tokens of 16 heads on 4 move 46 MB in 13 us, 3.5 TB/s of the 5.2 that a large copy
// reaches: a workgroup's way from its loads through the block's maximum to its codes, and
// the query tiles' rotation tables, computed again for every four heads, are not hidden.
// (More waves a CU spill.)
template <int TYPE>
__global__ __launch_bounds__(256, 4) void kv8_append_prompt_kernel(const AppendParams p) {
  __shared__ __attribute__((aligned(16))) Turn lds;
  __shared__ uint32_t red[4];
  extern __shared__ __attribute__((aligned(16))) float table[];
  const Kv8& c = p.c;
  const int64_t ntask = (int64_t)c.B * c.Hkv * 2 * p.nb;
  int64_t id = blockIdx.x;
  if (id < ntask) {
    const int i = (int)(id % p.nb);
    id /= p.nb;
    const bool values = id & 1;
    const int64_t bh = id >> 1;
    const int b = (int)(bh / c.Hkv), h = (int)(bh % c.Hkv);
    const int L = p.lens[b];
    if (i == 0 && may_wait(L, c.Smax)) quantise_tail_block<TYPE>(c, bh, waiting_block(L, c.Smax), values, red);
    if (L < 0 || L > c.Smax) return;
    const int first = L >> 6, end = min(L + p.T, c.Smax), done = end >> 6, j = first + i;
    const bool reads_tail = (L & 63) != 0 || may_wait(L, c.Smax);
    const int tail0 = max(done - 1, first);  // the first block that the tail keeps
#pragma unroll 1
    for (int step = 0; step < (reads_tail && i == 0 ? 3 : 1); ++step) {
      const int jj = step == 0 ? j : tail0 + step - 1;
      const bool quantises = step == 0 && jj < done;
      const bool keeps = step == 0 ? !reads_tail && jj >= tail0 : jj <= done;
      if (kBlk * jj >= end || !(quantises || keeps)) continue;
      const Rows r = prompt_rows(p, b, h, L, jj, values, lds, table);
      if (quantises) store_codes<TYPE>(c, bh, jj, values, r, lds, red);
      if (keeps) store_tail(c, bh, jj, values, r, L, end, lds);
    }
    return;
  }
  id -= ntask;
  const int hgroups = (p.Hq + 3) >> 2;
  const int h0 = 4 * (int)(id % hgroups);
  id /= hgroups;
  const int tile = (int)(id % p.qtiles), b = (int)(id / p.qtiles);
  const int L = p.lens[b], t0 = 16 * tile;
  if (h0 == 0 && tile == 0 && threadIdx.x == 0 && (L < 0 || L > c.Smax - p.T) && p.overflow != nullptr)
    p.overflow[b] = 1;
  const int tk = threadIdx.x >> 4, f = threadIdx.x & 15, t = t0 + tk;  // a token a 16 lanes
  const int64_t row = (int64_t)b * p.T + min(t, p.T - 1);
  u32x4 x[4], w;
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = ld16(p.proj + row * p.row_stride + 2 * min(h0 + i, p.Hq - 1) * kHD + 8 * f);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(p.q_norm_w + 8 * f)[i];
  rotation_table<16>(table, L + t0, p);
  __syncthreads();
  const int half = p.rot >> 1;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const u32x4 y = norm_rotate8(x[i], w, table + tk * half, table + (16 + tk) * half, f, p.rot, p.eps);
    if (t < p.T && h0 + i < p.Hq) *reinterpret_cast<u32x4*>(p.q_out + (row * p.Hq + h0 + i) * kHD + 8 * f) = y;
  }
}

// -------------------------------------------------------------------- load
struct LoadParams {
  Kv8 c;
  const uint16_t* k;
  const uint16_t* v;
  int64_t ks[3], vs[3];  // strides: b, h, position
  const int32_t* lens;
  int S, nb;
};

// Workgroup (block j, keys or values, head): codes if the block is complete, the tail
// if it is one of the last two.  Bound by memory: 4 sequences of 8192 positions, 101 MB
// in 18 us, 5.5 TB/s.
template <int TYPE>
__global__ __launch_bounds__(256) void kv8_load_kernel(const LoadParams p) {
  __shared__ __attribute__((aligned(16))) Turn lds;
  __shared__ uint32_t red[4];
  const Kv8& c = p.c;
  const int j = (int)(blockIdx.x % p.nb);
  const int64_t id = blockIdx.x / p.nb;
  const bool values = id & 1;
  const int64_t bh = id >> 1;
  const int b = (int)(bh / c.Hkv), h = (int)(bh % c.Hkv);
  const int n = min(p.lens[b], min(p.S, c.Smax));
  if (kBlk * j >= n) return;
  const int64_t* st = values ? p.vs : p.ks;
  const uint16_t* src = (values ? p.v : p.k) + b * st[0] + h * st[1];
  Rows r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r.x[i] = ld16(src + min(kBlk * j + (int)(threadIdx.x >> 4) + 16 * i, n - 1) * st[2] + 8 * (threadIdx.x & 15));
  if (j < n >> 6) store_codes<TYPE>(c, bh, j, values, r, lds, red);
  if (j >= (n >> 6) - 1) store_tail(c, bh, j, values, r, 0, n, lds);
}

// -------------------------------------------------------------------- read
struct ReadParams {
  Kv8 c;
  const int32_t* lens;
  const int32_t* starts;
  int start, count, nb;
  uint16_t* k;
  uint16_t* v;
};

// Workgroup (block of positions, keys or values, head).  A block's rows come from its
// codes (values turned by 4 features x 8 positions a thread) or from the tail, and go
// out as whole rows, 16 bytes a lane.  Bound by memory: 4 sequences of 8190 positions, 101
// MB (two thirds of it written) in 15 us, 6.6 TB/s.
template <int TYPE>
__global__ __launch_bounds__(256) void kv8_read_kernel(const ReadParams p) {
  __shared__ __attribute__((aligned(16))) Turn lds;
  __shared__ uint32_t red[4];
  const Kv8& c = p.c;
  const int i = (int)(blockIdx.x % p.nb);
  const int64_t id = blockIdx.x / p.nb;
  const bool values = id & 1;
  const int64_t bh = id >> 1;
  uint16_t* out = values ? p.v : p.k;
  if (out == nullptr) return;
  const int b = (int)(bh / c.Hkv), t = threadIdx.x;
  const int L = p.lens[b];
  const int held = min(max(L, 0), c.Smax);
  const int64_t start = (int64_t)p.start + (p.starts ? p.starts[b] : 0);
  // block floor(start / 64) + i covers the outputs 64 block - start ..
  const int64_t block = (start >> 6) + i;
  if (kBlk * block >= start + p.count) return;
  Rows r;
#pragma unroll
  for (int u = 0; u < 4; ++u) r.x[u] = u32x4{0u, 0u, 0u, 0u};
  if (block >= 0 && kBlk * block < held) {
    const int j = (int)block;
    const bool waits = j == waiting_block(L, c.Smax) && may_wait(L, c.Smax);
    if (j < held >> 6 && !waits) {
      const float s = (values ? c.vs : c.ks)[bh * c.nblk + j];
      u32x2 q[4];
      if (!values) {
#pragma unroll
        for (int u = 0; u < 4; ++u) q[u] = *reinterpret_cast<const u32x2*>(c.keys(bh, j) + 8 * (t + 256 * u));
      } else {
        const int p0 = 8 * (t & 7), quad = t >> 3;
        uint32_t w[8];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const u32x2 x = *reinterpret_cast<const u32x2*>(c.values(bh, j) + (4 * quad + u) * kBlk + p0);
          w[u] = x.x;
          w[4 + u] = x.y;
        }
        transpose4(w[0], w[1], w[2], w[3]);
        transpose4(w[4], w[5], w[6], w[7]);
#pragma unroll
        for (int u = 0; u < 8; ++u) lds.codes[p0 + u][quad] = w[u];
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const uint32_t* src = &lds.codes[(t >> 4) + 16 * u][2 * (t & 15)];
          q[u] = u32x2{src[0], src[1]};
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) r.x[u] = values_bf16<TYPE>(q[u], s);
    } else {
      const int at = (j & 1) * kBlk;
      if (!values) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          r.x[u] = ld16(c.tail_keys(bh) + (at + (t >> 4) + 16 * u) * kHD + 8 * (t & 15));
      } else {
        const uint16_t* src = c.tail_values(bh) + (t >> 1) * kSlots + at + (t & 1) * 32;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const u32x4 w = ld16(src + 8 * u);
#pragma unroll
          for (int x = 0; x < 8; ++x)
            lds.rows[(t & 1) * 32 + 8 * u + x][t >> 1] = (uint16_t)(w[x >> 1] >> (16 * (x & 1)));
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u) r.x[u] = *reinterpret_cast<const u32x4*>(&lds.rows[(t >> 4) + 16 * u][8 * (t & 15)]);
      }
      if (waits) {  // as it will read once it has its codes
        uint32_t a = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) a = max(a, abs_bits16(r.x[u]));
        const f32x2 sm = block_scale<TYPE>(group_max_u32(a, red));
#pragma unroll
        for (int u = 0; u < 4; ++u) r.x[u] = values_bf16<TYPE>(quantise8<TYPE>(r.x[u], sm.y), sm.x);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int64_t pos = kBlk * block + (t >> 4) + 16 * u, o = pos - start;
    if (o < 0 || o >= p.count) continue;
    *reinterpret_cast<u32x4*>(out + (bh * p.count + o) * kHD + 8 * (t & 15)) =
        pos < held ? r.x[u] : u32x4{0u, 0u, 0u, 0u};
  }
}

bool fits_grid(int64_t wgs) { return wgs <= INT32_MAX; }

}  // namespace
}  // namespace dflash

using namespace dflash;

#define DFLASH_KV8_LAUNCH(kernel, type, grid, lds, stream, p)                                    \
  do {                                                                                           \
    if ((type) == DFLASH_KV_INT8)                                                                \
      hipLaunchKernelGGL((kernel<DFLASH_KV_INT8>), dim3((unsigned)(grid)), dim3(256), lds,       \
                         static_cast<hipStream_t>(stream), p);                                   \
    else                                                                                         \
      hipLaunchKernelGGL((kernel<DFLASH_KV_E4M3>), dim3((unsigned)(grid)), dim3(256), lds,       \
                         static_cast<hipStream_t>(stream), p);                                   \
  } while (0)

extern "C" int dflash_kv8_append(const dflash_kv8_cache* cache, const void* proj, int64_t proj_row_stride,
                                 const void* q_norm_w, const void* k_norm_w, const int32_t* lens,
                                 void* q_out, int32_t* overflow, int T, int Hq, int rot_dims,
                                 float rope_base, float eps, int prompt, void* stream) {
  AppendParams p{};
  if (const int rc = check_cache(cache, &p.c)) return rc;
  const int B = p.c.B, Hkv = p.c.Hkv;
  if (T < 0 || Hq <= 0 || Hq % Hkv != 0 || (!prompt && T > kMaxDraft)) return DFLASH_ERR_SHAPE;
  if (!(rot_dims == 0 || rot_dims == 16 || rot_dims == 32 || rot_dims == 64 || rot_dims == 128))
    return DFLASH_ERR_UNSUPPORTED;
  if (proj_row_stride < (int64_t)(2 * (int64_t)Hq + 2 * Hkv) * kHD) return DFLASH_ERR_SHAPE;
  if (T > INT32_MAX - p.c.Smax) return DFLASH_ERR_SHAPE;  // positions are 32-bit
  if (B == 0 || T == 0) return DFLASH_OK;
  if (proj == nullptr || q_norm_w == nullptr || k_norm_w == nullptr || lens == nullptr || q_out == nullptr)
    return DFLASH_ERR_NULL;
  if (((uintptr_t)proj & 15) || proj_row_stride % 8 || ((uintptr_t)q_norm_w & 3) || ((uintptr_t)k_norm_w & 3) ||
      ((uintptr_t)q_out & 15))
    return DFLASH_ERR_ALIGN;
  p.proj = static_cast<const uint16_t*>(proj);
  p.row_stride = proj_row_stride;
  p.q_norm_w = static_cast<const uint16_t*>(q_norm_w);
  p.k_norm_w = static_cast<const uint16_t*>(k_norm_w);
  p.lens = lens;
  p.q_out = static_cast<uint16_t*>(q_out);
  p.overflow = overflow;
  p.T = T; p.Hq = Hq; p.rot = rot_dims;
  for (int i = 0; i < rot_dims / 2; ++i) p.freq[i] = exp2(-2.0 * i / rot_dims * log2((double)rope_base));
  p.eps = eps;
  if (!prompt) {
    const int64_t grid = (int64_t)2 * B * Hkv + (int64_t)B * T * ceil_div(Hq + 2 * Hkv, 16);
    if (!fits_grid(grid)) return DFLASH_ERR_SHAPE;
    DFLASH_KV8_LAUNCH(kv8_append_draft_kernel, cache->type, grid, 0, stream, p);
  } else {
    p.nb = (int)std::min<int64_t>(T / kBlk + 2, p.c.nblk);
    p.qtiles = (int)ceil_div(T, 16);
    const int64_t grid = (int64_t)2 * B * Hkv * p.nb + (int64_t)B * p.qtiles * ceil_div(Hq, 4);
    if (!fits_grid(grid)) return DFLASH_ERR_SHAPE;
    DFLASH_KV8_LAUNCH(kv8_append_prompt_kernel, cache->type, grid, (unsigned)(kBlk * rot_dims * sizeof(float)), stream, p);
  }
  return to_status(hipGetLastError());
}

extern "C" int dflash_kv8_load(const dflash_kv8_cache* cache, const void* k, const int64_t* k_strides,
                               const void* v, const int64_t* v_strides, const int32_t* lens, int S,
                               void* stream) {
  LoadParams p{};
  if (const int rc = check_cache(cache, &p.c)) return rc;
  if (S < 0) return DFLASH_ERR_SHAPE;
  if (p.c.B == 0 || S == 0) return DFLASH_OK;
  if (k == nullptr || v == nullptr || lens == nullptr || k_strides == nullptr || v_strides == nullptr)
    return DFLASH_ERR_NULL;
  if (((uintptr_t)k & 15) || ((uintptr_t)v & 15)) return DFLASH_ERR_ALIGN;
  for (int i = 0; i < 3; ++i) {
    if (k_strides[i] < 0 || v_strides[i] < 0) return DFLASH_ERR_SHAPE;
    if (k_strides[i] % 8 || v_strides[i] % 8) return DFLASH_ERR_ALIGN;
    p.ks[i] = k_strides[i];
    p.vs[i] = v_strides[i];
  }
  p.k = static_cast<const uint16_t*>(k);
  p.v = static_cast<const uint16_t*>(v);
  p.lens = lens;
  p.S = S;
  p.nb = (int)ceil_div(std::min(S, p.c.Smax), kBlk);
  const int64_t grid = (int64_t)2 * p.c.B * p.c.Hkv * p.nb;
  if (!fits_grid(grid)) return DFLASH_ERR_SHAPE;
  DFLASH_KV8_LAUNCH(kv8_load_kernel, cache->type, grid, 0, stream, p);
  return to_status(hipGetLastError());
}

extern "C" int dflash_kv8_read(const dflash_kv8_cache* cache, const int32_t* lens, const int32_t* starts,
                               int start, int count, void* k_out, void* v_out, void* stream) {
  ReadParams p{};
  if (const int rc = check_cache(cache, &p.c)) return rc;
  if (count < 0) return DFLASH_ERR_SHAPE;
  if (p.c.B == 0 || count == 0) return DFLASH_OK;
  if (lens == nullptr || (k_out == nullptr && v_out == nullptr)) return DFLASH_ERR_NULL;
  if (((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15)) return DFLASH_ERR_ALIGN;
  p.lens = lens;
  p.starts = starts;
  p.start = start;
  p.count = count;
  p.nb = (int)(((int64_t)count + 62) / kBlk + 1);  // blocks that count positions can touch
  p.k = static_cast<uint16_t*>(k_out);
  p.v = static_cast<uint16_t*>(v_out);
  const int64_t grid = (int64_t)2 * p.c.B * p.c.Hkv * p.nb;
  if (!fits_grid(grid)) return DFLASH_ERR_SHAPE;
  DFLASH_KV8_LAUNCH(kv8_read_kernel, cache->type, grid, 0, stream, p);
  return to_status(hipGetLastError());
}
