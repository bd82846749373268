// Gated attention over the 8-bit key/value cache (include/dflash_kv8.h): a few
// new tokens a sequence (verify blocks, single-token decode) and prompt rows.
#include <hip/hip_runtime.h>
#include <math.h>

#include <algorithm>
#include <stdint.h>

#include "kv8_common.h"

namespace dflash {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;

// ------------------------------------------------------------------ verify
// The T * Hq / Hkv query rows of a (sequence, key/value head) are packed into RT
// tiles of 16 (row t * rep + r is query head r of the group, token t).  Work is
// counted in blocks of 64 positions over all heads and sequences; every workgroup
// takes an equal run of them, whatever the sequences' lengths, its four waves
// block by block in turn.  A wave keeps running maximum, sum and output of all rows
// in registers:
//   - S^T = K Q^T and O^T = V^T P^T on v_mfma_f32_16x16x32_bf16.  A lane (r = lane
//     % 16, g = lane / 16) holds row r's scores of 16 positions: result row 4 g + e
//     of tile n is position 16 g + 8 (n / 2) + 4 (n % 2) + e (the tile's operand row
//     i is loaded from position 16 (i / 4) + ..), so tiles 2 s and 2 s + 1 are
//     the operand of P V's step s as they stand, with the 8 values 16 g + 8 s .. of
//     V^T, and P never leaves the lane.
//   - a block's key scale is one factor of its scores; its value scale goes into
//     the exponent (weights 2^(x + log2 scale - m), m the running maximum of that),
//     and the sum takes the weights times 1 / scale.
// The runs' ends cut heads into parts: those go to the workspace and a second
// launch merges them; a head that one workgroup has to itself is finished there.
constexpr int kMinRun = 4;  // blocks of a run: one for each wave

struct VerifyParams {
  Kv8 c;
  const uint16_t* q;  // [B, T, Hq, D]
  const int32_t* lens;
  const uint16_t* gate;
  int64_t gate_stride;
  uint16_t* out;    // [B, T, Hq * D]
  float* part_o;    // [2 * runs][16 RT][D]
  float* part_ml;   // [2 * runs][16 RT][2]
  int T, Hq, rep, runs, rows;  // rows: 16 RT
  float scale;
};

__device__ __forceinline__ int wave_sum_i32(int x) {
#pragma unroll
  for (int off = 32; off >= 1; off >>= 1) x += __shfl_xor(x, off, 64);
  return x;
}

// Positions that sequence b's rows attend to, and their blocks (0: takes no part).
__device__ __forceinline__ int seen_positions(int L, int T, int Smax) {
  return L < 0 ? 0 : min(min(L, Smax) + T, Smax);
}
__device__ __forceinline__ int seen_blocks(int L, int T, int Smax) {
  return (seen_positions(L, T, Smax) + kBlk - 1) >> 6;
}

// Blocks of one head of all sequences; *before: of the sequences before b.
__device__ __forceinline__ int all_blocks(const VerifyParams& p, int b, int* before) {
  const int lane = threadIdx.x & 63;
  int n = 0, pre = 0;
  for (int b0 = 0; b0 < p.c.B; b0 += 64) {
    const int i = b0 + lane;
    const int v = i < p.c.B ? seen_blocks(p.lens[i], p.T, p.c.Smax) : 0;
    n += v;
    pre += i < b ? v : 0;
  }
  if (before != nullptr) *before = wave_sum_i32(pre);
  return wave_sum_i32(n);
}

// The sequence that unit u falls in, and the units before it.
__device__ __forceinline__ int sequence_of(const VerifyParams& p, int u, int* before) {
  const int lane = threadIdx.x & 63;
  int carry = 0;
  for (int b0 = 0; b0 < p.c.B; b0 += 64) {
    const int i = b0 + lane;
    const int v = i < p.c.B ? p.c.Hkv * seen_blocks(p.lens[i], p.T, p.c.Smax) : 0;
    int incl = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const int x = __shfl_up(incl, off, 64);
      if (lane >= off) incl += x;
    }
    const uint64_t past = __ballot(carry + incl > u);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      *before = carry + __shfl(incl - v, l, 64);
      return b0 + l;
    }
    carry += __shfl(incl, 63, 64);
  }
  *before = carry;
  return p.c.B;
}

__device__ __forceinline__ int run_length(const VerifyParams& p, int units) {
  return max(kMinRun, (units + p.runs - 1) / p.runs);
}

__device__ __forceinline__ float max_over_groups(float x) {  // lanes r, r + 16, r + 32, r + 48
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const f32x2 b = both_halves(x);
  return fmaxf(b.x, b.y);
}

__device__ __forceinline__ bool has_nonfinite(uint32_t w) {
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
__device__ __forceinline__ uint32_t drop_nonfinite(uint32_t w) {
  if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
  if ((w & 0x7f800000u) == 0x7f800000u) w &= 0x0000ffffu;
  return w;
}

// Eight bf16 with those from n on zero.
__device__ __forceinline__ u32x4 keep_first(u32x4 w, int n) {
#pragma unroll
  for (int i = 0; i < 4; ++i)
    w[i] &= n >= 2 * i + 2 ? 0xffffffffu : n == 2 * i + 1 ? 0x0000ffffu : 0u;
  return w;
}

template <int RT>
struct Rows {  // a wave's running state: lane (r, g) has row 16 rt + r, features 16 dt + 4 g + e
  float m[RT], l[RT];
  f32x4 o[RT][8];
};

// One block's scores to weights: s[rt][n] in, the operand of P V out.
template <int RT>
__device__ __forceinline__ void softmax_block(Rows<RT>& a, f32x4 (&s)[RT][4], float sl, float lv, float iv,
                                              u32x4 (&pb)[RT][2]) {
#pragma unroll
  for (int rt = 0; rt < RT; ++rt) {
    float mx = -INFINITY;
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[rt][n][e]);
    mx = fmaf(max_over_groups(mx), sl, lv);
    if (__any(mx > a.m[rt])) {
      const float mn = fmaxf(a.m[rt], mx);
      const float alpha = a.m[rt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(a.m[rt] - mn);
      a.l[rt] *= alpha;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) a.o[rt][dt] *= alpha;
      a.m[rt] = mn;
    }
    const float off = lv - (a.m[rt] == -INFINITY ? 0.f : a.m[rt]);
    float sum = 0.f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      float pe[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        pe[i] = __builtin_amdgcn_exp2f(fmaf(s[rt][2 * k + (i >> 2)][i & 3], sl, off));
        sum += pe[i];
      }
      pb[rt][k] = cvt8_bf16(pe);
    }
    a.l[rt] = fmaf(sum, iv, a.l[rt]);
  }
}

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}

template <int TYPE, int RT>
__global__ __launch_bounds__(256, RT <= 2 ? 2 : 1) void attn_verify_q8_kernel(const VerifyParams p) {
  __shared__ __attribute__((aligned(16))) float so[4][16 * RT][kHD + 4];
  __shared__ float sml[4][16 * RT][2];
  const Kv8& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int units = c.Hkv * all_blocks(p, 0, nullptr);
  const int per = run_length(p, units);
  const int run0 = blockIdx.x * per;
  int left = min(per, units - run0);
  if (left <= 0) return;
  int before;
  int b = __builtin_amdgcn_readfirstlane(sequence_of(p, run0, &before));
  int rem = __builtin_amdgcn_readfirstlane(run0 - before);
  const float sl0 = (p.scale == 0.f ? 1.f : fabsf(p.scale)) * kLog2e;
  bool first_part = true;
  int h = -1, blk = 0;
  while (left > 0) {
    const int L = __builtin_amdgcn_readfirstlane(p.lens[b]);
    const int seen = seen_positions(L, p.T, c.Smax);
    const int nb = (seen + kBlk - 1) >> 6;
    if (nb == 0) {
      ++b;
      continue;
    }
    if (h < 0) {
      h = rem / nb;
      blk = rem - h * nb;
    }
    const int b1 = min(nb, blk + left);
    const int base = min(L, c.Smax), done = base >> 6;
    const int64_t bh = (int64_t)b * c.Hkv + h;
    // the rows' queries: operand (c2, hh) holds features 64 c2 + 16 g + 8 hh ..
    u32x4 qf[RT][4];
    int last[RT];  // the last position the lane's row sees
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      const int row = 16 * rt + r, t = min(row / p.rep, p.T - 1), rr = row % p.rep;
      last[rt] = min(base + t, seen - 1);
      const uint16_t* src = p.q + (((int64_t)b * p.T + t) * p.Hq + h * p.rep + rr) * kHD + 16 * g;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        qf[rt][k] = ld16(src + 64 * (k >> 1) + 8 * (k & 1));
        // scores are scaled by a positive factor: the sign goes to q, a zero to q itself
        if (!(p.scale > 0.f))
          qf[rt][k] = p.scale < 0.f ? qf[rt][k] ^ 0x80008000u : p.scale == 0.f ? u32x4{0u, 0u, 0u, 0u} : qf[rt][k];
      }
    }
    Rows<RT> a;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      a.m[rt] = -INFINITY;
      a.l[rt] = 0.f;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) a.o[rt][dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    for (int j = blk + wave; j < b1; j += 4) {
      f32x4 s[RT][4];
      u32x4 pb[RT][2];
#pragma unroll
      for (int rt = 0; rt < RT; ++rt)
#pragma unroll
        for (int n = 0; n < 4; ++n) s[rt][n] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (j < done) {  // codes; every row sees the whole block
        const uint8_t* kb = c.keys(bh, j) + 16 * g;
        const uint8_t* vb = c.values(bh, j) + r * kBlk + 16 * g;
        u32x4 kc[4][2], vc[8];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            kc[n][k] = ld16(kb + (16 * (r >> 2) + 8 * (n >> 1) + 4 * (n & 1) + (r & 3)) * kHD + 64 * k);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) vc[dt] = ld16(vb + 16 * dt * kBlk);
        const float ks = c.ks[bh * c.nblk + j], vs = c.vs[bh * c.nblk + j];
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const u32x2 lo = codes_bf16<TYPE>(kc[n][k >> 1][2 * (k & 1)]);
            const u32x2 hi = codes_bf16<TYPE>(kc[n][k >> 1][2 * (k & 1) + 1]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][n] = mfma_bf16(u32x4{lo.x, lo.y, hi.x, hi.y}, qf[rt][k], s[rt][n]);
          }
        softmax_block<RT>(a, s, sl0 * ks, __log2f(vs), 1.f / vs, pb);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const u32x2 lo = codes_bf16<TYPE>(vc[dt][2 * k]), hi = codes_bf16<TYPE>(vc[dt][2 * k + 1]);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
              a.o[rt][dt] = mfma_bf16(u32x4{lo.x, lo.y, hi.x, hi.y}, pb[rt][k], a.o[rt][dt]);
          }
      } else {  // the tail, in bf16
        const int at = (j & 1) * kBlk, p0 = kBlk * j;
        const uint16_t* kb = c.tail_keys(bh) + at * kHD + 16 * g;
        const uint16_t* vb = c.tail_values(bh) + r * kSlots + at + 16 * g;
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const u32x4 kf = ld16(kb + (16 * (r >> 2) + 8 * (n >> 1) + 4 * (n & 1) + (r & 3)) * kHD + 64 * (k >> 1) +
                                  8 * (k & 1));
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) s[rt][n] = mfma_bf16(kf, qf[rt][k], s[rt][n]);
          }
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              if (p0 + 16 * g + 8 * (n >> 1) + 4 * (n & 1) + e > last[rt]) s[rt][n][e] = -INFINITY;
        softmax_block<RT>(a, s, sl0, 0.f, 1.f, pb);
        // slots past the held positions hold anything; a row's weight for a
        // token it does not see is 0, which a NaN or an infinity would not leave 0
        bool bad = false;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            u32x4 vf = keep_first(ld16(vb + 16 * dt * kSlots + 8 * k), seen - (p0 + 16 * g + 8 * k));
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              bad |= has_nonfinite(vf[i]);
              vf[i] = drop_nonfinite(vf[i]);
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) a.o[rt][dt] = mfma_bf16(vf, pb[rt][k], a.o[rt][dt]);
          }
        if (__any(bad)) {  // what was dropped, for the rows that see it
          const int n = min(kBlk, seen - p0);
          for (int i = 0; i < n; ++i)
#pragma unroll
            for (int dt = 0; dt < 8; ++dt)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t x = c.tail_values(bh)[(16 * dt + 4 * g + e) * kSlots + at + i];
                if ((x & 0x7f80u) != 0x7f80u) continue;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
                  if (p0 + i <= last[rt]) a.o[rt][dt][e] += bf16_bits_to_f32(x);
              }
        }
      }
    }
    // the four waves' states through LDS
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
      float l = a.l[rt];
      l += __shfl_xor(l, 16, 64);
      l += __shfl_xor(l, 32, 64);
      const int row = 16 * rt + r;
      if (g == 0) {
        sml[wave][row][0] = a.m[rt];
        sml[wave][row][1] = l;
      }
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(&so[wave][row][16 * dt + 4 * g]) = a.o[rt][dt];
    }
    __syncthreads();
    const bool whole = blk == 0 && b1 == nb;
    const int64_t part = 2 * (int64_t)blockIdx.x + (first_part ? 0 : 1);
    for (int i = tid; i < 16 * RT * 32; i += 256) {
      const int row = i >> 5, d = (i & 31) * 4;
      if (row >= p.T * p.rep) break;
      float m = -INFINITY, l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) m = fmaxf(m, sml[w][row][0]);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float mw = sml[w][row][0];
        const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - m);
        l = fmaf(sml[w][row][1], f, l);
        o += *reinterpret_cast<const f32x4*>(&so[w][row][d]) * f;
      }
      if (whole) {
        const int t = row / p.rep, qh = h * p.rep + row % p.rep;
        const int64_t bt = (int64_t)b * p.T + t;
        const u32x2 gv = *reinterpret_cast<const u32x2*>(p.gate + bt * p.gate_stride + qh * 2 * kHD + kHD + d);
        const float inv = 1.f / l;
        const float ga[4] = {bf16_lo(gv.x), bf16_hi(gv.x), bf16_lo(gv.y), bf16_hi(gv.y)};
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[e] * inv * (1.f / (1.f + __expf(-ga[e])));
        *reinterpret_cast<u32x2*>(p.out + (bt * p.Hq + qh) * kHD + d) = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
      } else {
        *reinterpret_cast<f32x4*>(p.part_o + (part * p.rows + row) * kHD + d) = o;
        if (d == 0) *reinterpret_cast<f32x2*>(p.part_ml + (part * p.rows + row) * 2) = f32x2{m, l};
      }
    }
    __syncthreads();
    first_part = false;
    left -= b1 - blk;
    blk = 0;
    if (b1 == nb && ++h == c.Hkv) {
      h = 0;
      ++b;
    }
  }
}

// One workgroup per (token, query head): merges the parts of a head that several
// runs share, wave w the parts w, w + 4, ..; lane l has features 2 l, 2 l + 1.
__global__ __launch_bounds__(256) void attn_verify_q8_merge_kernel(const VerifyParams p) {
  __shared__ float sm[4], sl[4];
  __shared__ f32x2 so[4][64];
  const int bt = blockIdx.x, qh = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int b = bt / p.T, t = bt - b * p.T, h = qh / p.rep, row = t * p.rep + qh % p.rep;
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + ((int64_t)bt * p.Hq + qh) * kHD + 2 * lane);
  const int nb = seen_blocks(p.lens[b], p.T, p.c.Smax);
  if (nb == 0) {  // takes no part
    if (wave == 0) *dst = 0u;
    return;
  }
  int before;
  const int per = run_length(p, p.c.Hkv * all_blocks(p, b, &before));
  const int u0 = p.c.Hkv * before + h * nb;
  const int w0 = u0 / per, w1 = (u0 + nb - 1) / per;
  if (w0 == w1) return;  // finished by its one run
  const int head = 2 * w0 + (u0 > w0 * per ? 1 : 0);  // part of the first run; 2 w of the others
  float m = -INFINITY, l = 0.f, a0 = 0.f, a1 = 0.f;
  for (int s0 = w0 + wave; s0 <= w1; s0 += 16) {
    f32x2 ml[4], os[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int s = min(s0 + 4 * u, w1);
      const int64_t i = (int64_t)(s == w0 ? head : 2 * s) * p.rows + row;
      ml[u] = *reinterpret_cast<const f32x2*>(p.part_ml + 2 * i);
      os[u] = *reinterpret_cast<const f32x2*>(p.part_o + i * kHD + 2 * lane);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (s0 + 4 * u > w1) continue;
      const float mn = fmaxf(m, ml[u].x);
      const float ca = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      const float cb = ml[u].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[u].x - mn);
      l = l * ca + ml[u].y * cb;
      a0 = a0 * ca + os[u].x * cb;
      a1 = a1 * ca + os[u].y * cb;
      m = mn;
    }
  }
  if (lane == 0) {
    sm[wave] = m;
    sl[wave] = l;
  }
  so[wave][lane] = f32x2{a0, a1};
  __syncthreads();
  if (wave != 0) return;
  float mm = -INFINITY;
#pragma unroll
  for (int k = 0; k < 4; ++k) mm = fmaxf(mm, sm[k]);
  float lsum = 0.f, o0 = 0.f, o1 = 0.f;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float f = sm[k] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(sm[k] - mm);
    lsum = fmaf(sl[k], f, lsum);
    o0 = fmaf(so[k][lane].x, f, o0);
    o1 = fmaf(so[k][lane].y, f, o1);
  }
  const float inv = 1.f / lsum;
  const uint32_t gv =
      *reinterpret_cast<const uint32_t*>(p.gate + (int64_t)bt * p.gate_stride + qh * 2 * kHD + kHD + 2 * lane);
  const float g0 = 1.f / (1.f + __expf(-bf16_lo(gv))), g1 = 1.f / (1.f + __expf(-bf16_hi(gv)));
  *dst = pack2(o0 * inv * g0, o1 * inv * g1);
}

int verify_runs(int64_t B, int Hkv, int Smax, int rt) {
  const int cus = device_cus() > 0 ? device_cus() : 256;
  const int64_t most = (int64_t)cus * (rt <= 2 ? 2 : 1);  // workgroups that fit at a time
  return (int)std::max<int64_t>(1, std::min(most, ceil_div(B * Hkv * (Smax / kBlk), kMinRun)));
}

template <int TYPE>
void launch_verify(const VerifyParams& p, int rt, hipStream_t s) {
  const dim3 grid((unsigned)p.runs);
  switch (rt) {
    case 1: hipLaunchKernelGGL((attn_verify_q8_kernel<TYPE, 1>), grid, dim3(256), 0, s, p); break;
    case 2: hipLaunchKernelGGL((attn_verify_q8_kernel<TYPE, 2>), grid, dim3(256), 0, s, p); break;
    case 3: hipLaunchKernelGGL((attn_verify_q8_kernel<TYPE, 3>), grid, dim3(256), 0, s, p); break;
    default: hipLaunchKernelGGL((attn_verify_q8_kernel<TYPE, 4>), grid, dim3(256), 0, s, p); break;
  }
}

// ------------------------------------------------------------------ prompt
// The prompt rows' attention: the bf16 cache's kernel (model_ops.hip) with the turns'
// keys and values coming from codes.  A workgroup owns RB blocks of 32 query rows of
// REP query heads of one key/value head, two waves per head and block, which walk the
// keys 128 at a time, wave half hf the 64 keys from 64 hf of each turn: one block of
// the cache, so its scales are two factors of the wave's turn (the key scale in the
// scores', the value scale in the weights' exponent, as in the verify kernel).
//   - Products on v_mfma_f32_32x32x16_bf16 in transposed form, S^T = K Q^T and
//     O^T = V^T P^T: a lane holds one query's column, its maximum is in-lane but for
//     lane ^ 32, P^T never leaves registers.
//   - A turn's codes are loaded once per workgroup, a turn ahead, and become bf16 on
//     their way to the other of two LDS buffers: 16-byte piece c of row r at slot
//     c ^ (r % 8).
struct PrefillParams {
  Kv8 c;
  const uint16_t* q;  // [B, P, Hq, D]
  const int32_t* lens;
  const uint16_t* gate;
  int64_t gate_stride;
  uint16_t* out;  // [B, P, Hq * D]
  int P, Hq;
  int heads, groups;  // launched head groups (Hkv * groups) and groups of a key/value head
  int nblk;           // row blocks
  int xcds;           // XCDs that a launched head group owns (0: groups in order)
  float scale;
};

constexpr int kPRows = 32;                     // query rows of a wave
constexpr int kPKeys = 2 * kBlk;               // keys of a turn
constexpr int kPBuf = 2 * kPKeys * kHD * 2;    // bytes of one turn's K and V^T in bf16
constexpr int kPMerge = 66 * 64;               // floats of a wave's O, m and l
constexpr int kPPitch = kHD + 4;               // floats of a normalized row in LDS

constexpr int prefill_lds(int pairs) {
  const int merge = 4 * pairs * (kPMerge + kPRows * kPPitch);
  return merge > 2 * kPBuf ? merge : 2 * kPBuf;
}

template <int TYPE, int REP, int RB>
__global__ __launch_bounds__(128 * REP * RB, 2) void attn_prefill_q8_kernel(const PrefillParams p) {
  constexpr int PAIRS = REP * RB;
  constexpr int NT = 128 * PAIRS;
  constexpr int UNITS = kPKeys * kHD / 16;  // 16 values of K (and of V^T) each
  constexpr int PER = (UNITS + NT - 1) / NT;
  __shared__ __attribute__((aligned(16))) unsigned char lds[prefill_lds(PAIRS)];
  __shared__ int dropped;  // the tail's values hold a NaN or an infinity
  const Kv8& c = p.c;
  const int b = blockIdx.y;
  const int xcd = blockIdx.x & 7;
  const int hg = p.xcds ? xcd / p.xcds : (int)blockIdx.x / p.nblk;
  const int rank = p.xcds ? (int)(blockIdx.x >> 3) * p.xcds + xcd % p.xcds : (int)blockIdx.x % p.nblk;
  if (rank >= p.nblk) return;
  const int blk = p.nblk - 1 - rank;  // later rows see more keys: first
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int r32 = lane & 31, hl = lane >> 5;
  const int hf = wave / PAIRS, pair = wave % PAIRS;
  const int len = p.lens[b];
  const int base = min(max(len, 0), c.Smax);
  const int64_t bh = (int64_t)b * c.Hkv + hg / p.groups;
  const int t0 = blk * RB * kPRows;
  const int tw = RB == 1 ? t0 : t0 + pair / REP * kPRows;
  const int qh = hg * REP + (RB == 1 ? pair : pair % REP);
  const int seen = len < 0 ? 0 : min(base + p.P, c.Smax);  // positions of the cache
  const int done = seen >> 6;
  const int turns = len < 0 ? 0 : (min(base + min(t0 + RB * kPRows, p.P), c.Smax) + kPKeys - 1) / kPKeys;
  const int Lw = len >= 0 && (RB == 1 || tw < p.P) ? min(base + min(tw + kPRows, p.P), c.Smax) : 0;
  if (tid == 0) dropped = 0;
  u32x4 kv[PER][2], vv[PER][2];
  // K unit e: key e / 8, features 16 (e % 8) ..; V^T unit e: block e / 512, feature
  // (e / 4) % 128, keys 16 (e % 4) ..  Blocks past the cache's last are clamped.
  auto load_turn = [&](int turn) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = min(tid + NT * i, UNITS - 1);
      const int j = min(2 * turn + (e >> 9), c.nblk - 1);
      const int key = (e >> 3) & 63, d = (e >> 2) & 127;
      if (j < done) {
        kv[i][0] = ld16(c.keys(bh, j) + key * kHD + (e & 7) * 16);
        vv[i][0] = ld16(c.values(bh, j) + d * kBlk + (e & 3) * 16);
      } else {
        const int at = (j & 1) * kBlk;
        const uint16_t* ks = c.tail_keys(bh) + (at + key) * kHD + (e & 7) * 16;
        const uint16_t* vs = c.tail_values(bh) + d * kSlots + at + (e & 3) * 16;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          kv[i][u] = ld16(ks + 8 * u);
          vv[i][u] = ld16(vs + 8 * u);
        }
      }
    }
  };
  auto store_turn = [&](unsigned char* buf, int turn) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = tid + NT * i;
      if (UNITS % NT != 0 && e >= UNITS) continue;
      const int j = min(2 * turn + (e >> 9), c.nblk - 1);
      const int key = e >> 3, d = (e >> 2) & 127;
      u32x4 kw[2], vw[2];
      if (j < done) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const u32x2 x = codes_bf16<TYPE>(kv[i][0][u]), y = codes_bf16<TYPE>(vv[i][0][u]);
          kw[u >> 1][2 * (u & 1)] = x.x;
          kw[u >> 1][2 * (u & 1) + 1] = x.y;
          vw[u >> 1][2 * (u & 1)] = y.x;
          vw[u >> 1][2 * (u & 1) + 1] = y.y;
        }
      } else {
        bool bad = false;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          kw[u] = kv[i][u];
          vw[u] = keep_first(vv[i][u], seen - (kBlk * j + 16 * (e & 3) + 8 * u));
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            bad |= has_nonfinite(vw[u][x]);
            vw[u][x] = drop_nonfinite(vw[u][x]);
          }
        }
        if (bad) dropped = 1;
      }
      unsigned char* krow = buf + key * 256;
      const int c0 = 2 * (e & 7), sk = key & 7;
      *reinterpret_cast<u32x4*>(krow + ((c0 ^ sk) << 4)) = kw[0];
      *reinterpret_cast<u32x4*>(krow + (((c0 + 1) ^ sk) << 4)) = kw[1];
      // 16 keys: the first piece keeps 0-3 and 8-11 (hl = 0), the second 4-7 and 12-15
      unsigned char* vrow = buf + kPBuf / 2 + (e >> 9) * (kHD * 128) + d * 128;
      const int c1 = 2 * (e & 3), sv = d & 7;
      *reinterpret_cast<u32x4*>(vrow + ((c1 ^ sv) << 4)) = u32x4{vw[0].x, vw[0].y, vw[1].x, vw[1].y};
      *reinterpret_cast<u32x4*>(vrow + (((c1 + 1) ^ sv) << 4)) = u32x4{vw[0].z, vw[0].w, vw[1].z, vw[1].w};
    }
  };
  load_turn(0);
  const uint16_t* qr = p.q + (((int64_t)b * p.P + min(tw + r32, p.P - 1)) * p.Hq + qh) * kHD + hl * 8;
  u32x4 qb[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) qb[k] = ld16(qr + 16 * k);
  if (!(p.scale > 0.f)) {  // as in the verify kernel
#pragma unroll
    for (int k = 0; k < 8; ++k)
      qb[k] = p.scale < 0.f ? qb[k] ^ 0x80008000u : p.scale == 0.f ? u32x4{0u, 0u, 0u, 0u} : qb[k];
  }
  __syncthreads();  // dropped is 0
  store_turn(lds, 0);
  if (turns > 1) load_turn(1);
  float m = -INFINITY, l = 0.f;
  f32x16 o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) o[dt] = f32x16{};
  const float sl0 = (p.scale == 0.f ? 1.f : fabsf(p.scale)) * kLog2e;
  const int last = min(base + tw + r32, Lw - 1);  // the last key this lane's row sees
  __syncthreads();
  for (int j = 0; j < turns; ++j) {
    const unsigned char* buf = lds + (j & 1) * kPBuf;
    const int kb = 2 * j + hf, k0 = kBlk * kb;
    float ks = 1.f, vs = 1.f;
    if (kb < done) {
      ks = c.ks[bh * c.nblk + kb];
      vs = c.vs[bh * c.nblk + kb];
    }
    if (j + 1 < turns) {
      store_turn(lds + ((j + 1) & 1) * kPBuf, j + 1);
      if (j + 2 < turns) load_turn(j + 2);
    }
    if (k0 < Lw) {
      const unsigned char* sk = buf + 64 * hf * 256;
      const unsigned char* sv = buf + kPBuf / 2 + hf * (kHD * 128);
      const float sl = sl0 * ks, lv = __log2f(vs), iv = 1.f / vs;
      f32x16 st[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) {
        st[kt] = f32x16{};
#pragma unroll
        for (int k = 0; k < 8; ++k)
          st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(
                                             sk + (32 * kt + r32) * 256 + (((2 * k + hl) ^ (r32 & 7)) << 4))),
              __builtin_bit_cast(bf16x8, qb[k]), st[kt], 0, 0, 0);
      }
      const bool masked = k0 + 63 > base + tw;  // some row does not see the whole block
      if (masked) {
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int key = k0 + 32 * kt + 8 * (i >> 2) + 4 * hl + (i & 3);
            if (key > last) st[kt][i] = -INFINITY;
          }
      }
      float mx = st[0][0];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[kt][i]);
      const f32x2 mb = both_halves(mx);
      mx = fmaf(fmaxf(mb.x, mb.y), sl, lv);
      if (__any(mx > m)) {
        const float mn = fmaxf(m, mx);
        const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
        m = mn;
      }
      const float off = lv - (m == -INFINITY ? 0.f : m);
      float sum = 0.f;
      u32x4 pb[4];
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        float pe[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          pe[i] = __builtin_amdgcn_exp2f(fmaf(st[s >> 1][8 * (s & 1) + i], sl, off));
          sum += pe[i];
        }
        pb[s] = cvt8_bf16(pe);
      }
      if (masked && !(sl + off == sl + off)) {
        // a block that reads as NaN, past some rows' last key: nothing of it for a row
        // that does not see it (its whole weight is NaN here, not 0)
        if (k0 > last) {
          sum = 0.f;
#pragma unroll
          for (int s = 0; s < 4; ++s) pb[s] = u32x4{0u, 0u, 0u, 0u};
        }
      }
      l = fmaf(sum, iv, l);
#pragma unroll
      for (int s = 0; s < 4; ++s)
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(
                                             sv + (32 * dt + r32) * 128 + (((2 * s + hl) ^ (r32 & 7)) << 4))),
              __builtin_bit_cast(bf16x8, pb[s]), o[dt], 0, 0, 0);
    }
    __syncthreads();
  }
  if (dropped && hf == 0) {  // the tail's dropped values, for the rows that see them
    for (int pos = kBlk * done; pos < seen; ++pos)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const uint32_t x = c.tail_values(bh)[(32 * dt + 8 * (i >> 2) + 4 * hl + (i & 3)) * kSlots + (pos & (kSlots - 1))];
          if ((x & 0x7f80u) == 0x7f80u && pos <= last) o[dt][i] += bf16_bits_to_f32(x);
        }
  }
  // The second key half's sums go to the first through LDS, which leaves the
  // normalized rows there; every wave then gates and stores whole rows.
  float* red = reinterpret_cast<float*>(lds) + pair * kPMerge + lane;
  float* rows = reinterpret_cast<float*>(lds) + PAIRS * kPMerge;  // [PAIRS][32][kPPitch]
  if (hf == 1) {
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) red[(16 * dt + i) * 64] = o[dt][i];
    red[64 * 64] = m;
    red[65 * 64] = l;
  }
  constexpr int OUT = PAIRS * kPRows * 16 / NT;  // pieces of 8 features a thread stores
  auto row_of = [&](int e) { return t0 + (RB == 1 ? 0 : (e >> 9) / REP * kPRows) + ((e >> 4) & 31); };
  auto head_of = [&](int e) { return hg * REP + (RB == 1 ? e >> 9 : (e >> 9) % REP); };
  u32x4 gt[OUT];
#pragma unroll
  for (int i = 0; i < OUT; ++i) {
    const int e = tid + NT * i;
    gt[i] = ld16(p.gate + ((int64_t)b * p.P + min(row_of(e), p.P - 1)) * p.gate_stride + head_of(e) * 2 * kHD + kHD +
                 (e & 15) * 8);
  }
  __syncthreads();
  if (hf == 0) {
    const float m1 = red[64 * 64], l1 = red[65 * 64];
    const float mn = fmaxf(m, m1);
    float c0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    float c1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - mn);
    const f32x2 lb = both_halves(l * c0 + l1 * c1);
    const float ls = lb.x + lb.y;
    const float inv = ls == 0.f ? 0.f : 1.f / ls;  // 0: the sequence takes no part
    c0 *= inv;
    c1 *= inv;
    float* row = rows + (pair * kPRows + r32) * kPPitch;
#pragma unroll
    for (int dt = 0; dt < 4; ++dt)
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = o[dt][4 * i4 + e] * c0 + red[(16 * dt + 4 * i4 + e) * 64] * c1;
        *reinterpret_cast<f32x4*>(row + 32 * dt + 8 * i4 + 4 * hl) = v;
      }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OUT; ++i) {
    const int e = tid + NT * i, t = row_of(e);
    if (t >= p.P) continue;
    const float* row = rows + (e >> 4) * kPPitch + (e & 15) * 8;
    float g[8], v[8];
    unpack8(gt[i], g);
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = row[u] * (1.f / (1.f + __expf(-g[u])));
    *reinterpret_cast<u32x4*>(p.out + (((int64_t)b * p.P + t) * p.Hq + head_of(e)) * kHD + (e & 15) * 8) = pack8(v);
  }
}

// Row blocks of a workgroup: as many as make eight waves, two a SIMD (six with three
// heads), as in the bf16 cache's kernel.
constexpr int prefill_row_blocks(int rep) { return rep == 1 ? 4 : rep == 2 ? 2 : 1; }

template <int TYPE, int REP>
void launch_prefill(const PrefillParams& p, dim3 grid, hipStream_t s) {
  constexpr int RB = prefill_row_blocks(REP);
  hipLaunchKernelGGL((attn_prefill_q8_kernel<TYPE, REP, RB>), grid, dim3(128 * REP * RB), 0, s, p);
}

template <int TYPE>
void launch_prefill(const PrefillParams& p, int rep, dim3 grid, hipStream_t s) {
  switch (rep) {
    case 1: launch_prefill<TYPE, 1>(p, grid, s); break;
    case 2: launch_prefill<TYPE, 2>(p, grid, s); break;
    case 3: launch_prefill<TYPE, 3>(p, grid, s); break;
    default: launch_prefill<TYPE, 4>(p, grid, s); break;
  }
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" size_t dflash_attn_verify_q8_workspace_bytes(int B, int T, int Hq, int Hkv, int Smax) {
  if (B <= 0 || T <= 0 || T > kMaxDraft || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || (int64_t)T * (Hq / Hkv) > 64 ||
      Smax <= 0 || Smax % kBlk != 0)
    return 0;
  const int rt = (int)ceil_div((int64_t)T * (Hq / Hkv), 16);
  return (size_t)2 * verify_runs(B, Hkv, Smax, rt) * 16 * rt * (kHD + 2) * sizeof(float);
}

extern "C" int dflash_attn_verify_q8(const dflash_kv8_cache* cache, const void* q, const int32_t* lens,
                                     const void* gate_src, int64_t gate_row_stride, void* out, int T, int Hq,
                                     float scale, void* workspace, size_t workspace_bytes, void* stream) {
  VerifyParams p{};
  if (const int rc = check_cache(cache, &p.c)) return rc;
  const int B = p.c.B, Hkv = p.c.Hkv;
  if (T < 0 || T > kMaxDraft || Hq <= 0 || Hq % Hkv != 0 || (int64_t)T * (Hq / Hkv) > 64) return DFLASH_ERR_SHAPE;
  if (gate_row_stride < (int64_t)2 * Hq * kHD) return DFLASH_ERR_SHAPE;
  if ((int64_t)B * T > INT32_MAX || Hq > 65535 || (int64_t)B * Hkv * p.c.nblk > INT32_MAX / 2) return DFLASH_ERR_SHAPE;
  if (B == 0 || T == 0) return DFLASH_OK;
  if (q == nullptr || lens == nullptr || gate_src == nullptr || out == nullptr || workspace == nullptr)
    return DFLASH_ERR_NULL;
  if (((uintptr_t)q & 15) || ((uintptr_t)gate_src & 7) || gate_row_stride % 4 || ((uintptr_t)out & 7) ||
      ((uintptr_t)workspace & 15))
    return DFLASH_ERR_ALIGN;
  if (workspace_bytes < dflash_attn_verify_q8_workspace_bytes(B, T, Hq, Hkv, p.c.Smax)) return DFLASH_ERR_WORKSPACE;
  p.q = static_cast<const uint16_t*>(q);
  p.lens = lens;
  p.gate = static_cast<const uint16_t*>(gate_src);
  p.gate_stride = gate_row_stride;
  p.out = static_cast<uint16_t*>(out);
  p.T = T; p.Hq = Hq; p.rep = Hq / Hkv;
  p.scale = scale;
  const int rt = (int)ceil_div((int64_t)T * p.rep, 16);
  p.rows = 16 * rt;
  p.runs = verify_runs(B, Hkv, p.c.Smax, rt);
  p.part_o = static_cast<float*>(workspace);
  p.part_ml = p.part_o + (int64_t)2 * p.runs * p.rows * kHD;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->type == DFLASH_KV_INT8) launch_verify<DFLASH_KV_INT8>(p, rt, s);
  else launch_verify<DFLASH_KV_E4M3>(p, rt, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return (int)e;
  hipLaunchKernelGGL(attn_verify_q8_merge_kernel, dim3((unsigned)(B * T), (unsigned)Hq), dim3(256), 0, s, p);
  return to_status(hipGetLastError());
}

extern "C" int dflash_attn_prefill_q8(const dflash_kv8_cache* cache, const void* q, const int32_t* lens,
                                      const void* gate_src, int64_t gate_row_stride, void* out, int P, int Hq,
                                      float scale, void* stream) {
  PrefillParams p{};
  if (const int rc = check_cache(cache, &p.c)) return rc;
  const int B = p.c.B, Hkv = p.c.Hkv;
  if (P < 0 || Hq <= 0 || Hq % Hkv != 0 || Hq / Hkv > 16 || B > 65535) return DFLASH_ERR_SHAPE;
  if (gate_row_stride < (int64_t)2 * Hq * kHD || P > INT32_MAX - p.c.Smax) return DFLASH_ERR_SHAPE;
  if (B == 0 || P == 0) return DFLASH_OK;
  if (q == nullptr || lens == nullptr || gate_src == nullptr || out == nullptr) return DFLASH_ERR_NULL;
  if (((uintptr_t)q & 15) || ((uintptr_t)gate_src & 15) || gate_row_stride % 8 || ((uintptr_t)out & 15))
    return DFLASH_ERR_ALIGN;
  // the launched heads: up to four query heads of a key/value head together
  int rep = 4;
  while (Hq / Hkv % rep != 0) --rep;
  p.q = static_cast<const uint16_t*>(q);
  p.lens = lens;
  p.gate = static_cast<const uint16_t*>(gate_src);
  p.gate_stride = gate_row_stride;
  p.out = static_cast<uint16_t*>(out);
  p.P = P; p.Hq = Hq;
  p.heads = Hq / rep;
  p.groups = p.heads / Hkv;
  p.nblk = (int)ceil_div(P, kPRows * prefill_row_blocks(rep));
  p.xcds = 8 % p.heads == 0 ? 8 / p.heads : 0;
  p.scale = scale;
  const int64_t wgs = p.xcds ? 8 * ceil_div(p.nblk, p.xcds) : (int64_t)p.nblk * p.heads;
  if (wgs > INT32_MAX) return DFLASH_ERR_SHAPE;
  const dim3 grid((unsigned)wgs, (unsigned)B);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->type == DFLASH_KV_INT8) launch_prefill<DFLASH_KV_INT8>(p, rep, grid, s);
  else launch_prefill<DFLASH_KV_E4M3>(p, rep, grid, s);
  return to_status(hipGetLastError());
}
