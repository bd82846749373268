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
// The T * Hq / Hkv query rows of a (sequence, key/value head), row t * rep + r being
// query head r of the group at token t, against the positions that they see.  Work is
// counted in blocks of 64 positions over all heads and sequences and shared by the
// launch's workgroups whatever the sequences' lengths (Batch).  That cuts heads into
// parts, which go to the workspace and are merged by the workgroup that brings a head's
// last one (up to 16 rows: 8 KB a part at most) or by a second launch (a part of 64 rows is
// 32 KB: one workgroup would take longer over a head's than the launch does); a head that
// one workgroup has to itself is finished there.
//   - Products on MFMA in transposed form, S^T = K Q^T and O^T = V^T P^T: a lane
//     holds one row's scores and outputs, and P stays in its registers.
//   - A block's key scale is one factor of its scores; its value scale goes into
//     the exponent (weights 2^(x + log2 scale - m), m the running maximum of that),
//     and the sum takes the weights times 1 / scale.
//   - Weights are rounded to bf16 for P V (the codes are exact in it): off by at most
//     2^-8 of themselves, where the codes are by 2^-8 of the block's largest value (int8)
//     or 2^-4 of their own (e4m3).  Sums, maxima and outputs stay in fp32.
// Every position's 256 bytes of codes are read once, which bounds the kernel where rows
// are few: 32 sequences of up to 8191 positions (16 heads on 4, one token, int8), 204 MB
// in 45 us, 4.5 TB/s of the 5.2 that a large copy reaches.
struct VerifyParams {
  Kv8 c;
  const uint16_t* q;  // [B, T, Hq, D]
  const int32_t* lens;
  const uint16_t* gate;
  int64_t gate_stride;
  uint16_t* out;    // [B, T, Hq * D]
  float* part_o;    // [2 * runs][part_rows][D], in the order that the kernel's lanes hold them
  float* part_ml;   // [2 * runs][part_rows][2]
  int32_t* count;   // [B, Hkv] parts that have arrived (up to 16 rows); zero between calls
  int T, Hq, rep, runs, min_cut;
  int waves;      // of a workgroup (up to 16 rows)
  int part_rows;  // rows of a part in the workspace
  int sliced;     // the merge of more than 16 rows: a workgroup per sixteenth of a head's outputs
  uint32_t rep_inv;
  float scale;

  __device__ int token_of(int row) const { return (int)((uint32_t)row * rep_inv >> 16); }  // row / rep, row < 64
};

// Positions that sequence b's rows attend to, and their blocks (0: takes no part).
__device__ __forceinline__ int seen_positions(int L, int T, int Smax) {
  return L < 0 ? 0 : min(min(L, Smax) + T, Smax);
}
__device__ __forceinline__ int seen_blocks(int L, int T, int Smax) {
  return (seen_positions(L, T, Smax) + kBlk - 1) >> 6;
}

// Inclusive sum over the wave's lanes.
__device__ __forceinline__ int wave_scan(int x) {
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false);  // row_shr:1, 2, 4, 8
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false);
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 to rows 1, 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 to rows 2, 3
  return x;
}

// Largest of the wave's values, 0 or more.
__device__ __forceinline__ int wave_most(int x) {
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false));
  x = max(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false));
  return __builtin_amdgcn_readlane(x, 63);
}

// How the launch's workgroups share the blocks, from the lengths: `cut` blocks are a
// workgroup's even share, at least min_cut.  Where every head cut into pieces of at most
// that gives no more pieces than workgroups, a workgroup takes one piece of one head
// (`pieces`); otherwise all blocks, in order of sequence and head, are cut into runs of
// the even share, which cross from head to head.  Pieces have a part each and are merged
// in even numbers (16 tokens after 4096: 14.7 us, as runs 16.5); runs fill the device
// where there are more heads than pieces can be had of (12 sequences of 8 heads).  Units: pieces, or
// blocks.  Lane i of chunk c has sequence 64 c + i; up to 64 sequences are loaded once and
// stay in the lanes.
// A head of up to 16 rows is merged by one workgroup, which takes about a 32nd of a row for
// each part of what a block takes: its parts are at most so many that the merge is no longer
// than the part before it, sqrt(blocks rows / 32) blocks each (1 key/value head, 16 rows
// after 32768: 20 us, else 40; 4 heads 21.4, else 24.6).
struct Batch {
  const VerifyParams& p;
  int len, incl;  // of the first chunk: lengths, and units of one head up to and with the lane's
  bool pieces;
  int cut;
  int per;        // units of a workgroup
  int units;      // of the launch

  __device__ __forceinline__ explicit Batch(const VerifyParams& params) : p(params) {
    int nblk = 0, n = 0, longest = 0;
    for (int c = chunks() - 1; c >= 0; --c) {
      load(c);
      const int nb = seen_blocks(len, p.T, p.c.Smax);
      nblk += __builtin_amdgcn_readlane(wave_scan(nb), 63);
      if (p.part_rows == 16) longest = max(longest, wave_most(nb));
    }
    nblk *= p.c.Hkv;
    cut = max(p.min_cut, (nblk + p.runs - 1) / p.runs);
    if (p.part_rows == 16) cut = max(cut, (int)sqrtf((float)longest * (float)(p.T * p.rep) * (1.f / 32.f)));
    pieces = true;
    for (int c = chunks() - 1; c >= 0; --c) {
      if (p.c.B > 64) load(c);
      scan();
      n += __builtin_amdgcn_readlane(incl, 63);
    }
    pieces = n * p.c.Hkv <= p.runs;
    units = pieces ? n * p.c.Hkv : nblk;
    per = pieces ? 1 : cut;
    if (!pieces) scan();
  }
  __device__ __forceinline__ int chunks() const { return (p.c.B + 63) >> 6; }
  __device__ __forceinline__ void load(int c) {
    const int i = 64 * c + (int)(threadIdx.x & 63);
    len = i < p.c.B ? p.lens[i] : -1;
  }
  __device__ __forceinline__ void scan() { incl = wave_scan(units_of(seen_blocks(len, p.T, p.c.Smax))); }
  __device__ __forceinline__ int units_of(int nb) const { return pieces ? (nb + cut - 1) / cut : nb; }
  __device__ __forceinline__ int length(int b) const {
    return p.c.B <= 64 ? __builtin_amdgcn_readlane(len, b) : __builtin_amdgcn_readfirstlane(p.lens[b]);
  }
  // Units of one head of the sequences before b.
  __device__ __forceinline__ int before(int b) {
    int carry = 0;
    if (p.c.B > 64)
      for (int c = 0; c <= b >> 6; ++c) {
        load(c);
        scan();
        if (c < b >> 6) carry += __builtin_amdgcn_readlane(incl, 63);
      }
    const int i = b & 63;
    return carry + (i == 0 ? 0 : __builtin_amdgcn_readlane(incl, i - 1));
  }
  // The sequence that unit u falls in; *rest: u's place in it.
  __device__ __forceinline__ int sequence_of(int u, int* rest) {
    int carry = 0;
    for (int c = 0; c < chunks(); ++c) {
      if (p.c.B > 64) {
        load(c);
        scan();
      }
      const uint64_t past = __ballot(p.c.Hkv * (carry + incl) > u);
      if (past != 0) {
        const int i = __builtin_ctzll(past);
        *rest = u - p.c.Hkv * (carry + (i == 0 ? 0 : __builtin_amdgcn_readlane(incl, i - 1)));
        return 64 * c + i;
      }
      carry += __builtin_amdgcn_readlane(incl, 63);
    }
    *rest = 0;
    return p.c.B;  // (u past the last unit: no caller asks)
  }
};

// A workgroup's share: from block blk of (b, h) on, `left` blocks.
struct Share {
  int b, h, blk, left;
};
__device__ __forceinline__ Share share_of(const VerifyParams& p, Batch& batch, int wg) {
  const int u = wg * batch.per;
  Share s{0, 0, 0, min(batch.per, batch.units - u)};
  if (s.left <= 0) return s;
  int rest;
  s.b = batch.sequence_of(u, &rest);
  const int nb = seen_blocks(batch.length(s.b), p.T, p.c.Smax), n = batch.units_of(nb);
  s.h = rest / n;
  s.blk = rest - s.h * n;
  if (batch.pieces) {
    const int size = (nb + n - 1) / n;
    s.blk *= size;
    s.left = min(size, nb - s.blk);  // (0 where even pieces leave the last one nothing)
  }
  return s;
}

__device__ __forceinline__ float max_over_groups(float x) {  // lanes r, r + 16, r + 32, r + 48
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
  const f32x2 b = both_halves(x);
  return fmaxf(b.x, b.y);
}

// Values that are not finite are dropped before P V, where the weight 0 of a row that
// does not see their token would not leave 0, and added to the rows that do see it
// afterwards (dropped_values).  That takes care of the tail's slots past the held
// positions too, which hold anything.  In packed bf16 an exponent of all ones carries
// into bits 15 and 31.
__device__ __forceinline__ uint32_t nonfinite_bits(uint32_t w) { return (w & 0x7f807f80u) + 0x00800080u; }
__device__ __forceinline__ uint32_t nonfinite_bits(u32x4 w) {
  return nonfinite_bits(w.x) | nonfinite_bits(w.y) | nonfinite_bits(w.z) | nonfinite_bits(w.w);
}
__device__ __forceinline__ bool any_nonfinite(uint32_t bits) { return (bits & 0x80008000u) != 0; }
__device__ __forceinline__ u32x4 drop_nonfinite(u32x4 w) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t y = nonfinite_bits(w[i]) & 0x80008000u;
    w[i] &= ~(y | (y - (y >> 15)));
  }
  return w;
}

__device__ __forceinline__ f32x4 mfma_bf16(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                 0, 0);
}

// The reciprocal is off by one unit in the last place of 32 bits, under a 2^16th of the
// rounding of the bf16 result.
__device__ __forceinline__ float sigmoid(float g) { return __builtin_amdgcn_rcpf(1.f + __expf(-g)); }

// Four normalized features of a row, times the sigmoid of their gates.
__device__ __forceinline__ u32x2 load_gate(const VerifyParams& p, int64_t bt, int qh, int d) {
  return *reinterpret_cast<const u32x2*>(p.gate + bt * p.gate_stride + qh * 2 * kHD + kHD + d);
}
__device__ __forceinline__ void store_gated(const VerifyParams& p, int64_t bt, int qh, int d, f32x4 v, u32x2 g) {
  const float ga[4] = {bf16_lo(g.x), bf16_hi(g.x), bf16_lo(g.y), bf16_hi(g.y)};
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] *= sigmoid(ga[e]);
  *reinterpret_cast<u32x2*>(p.out + (bt * p.Hq + qh) * kHD + d) = u32x2{pack2(v[0], v[1]), pack2(v[2], v[3])};
}

// The sum of feature d's values at tail positions from .. to that are not finite: what a
// row that sees them gets instead, a NaN or an infinity as in the plain sum.
__device__ __forceinline__ float dropped_values(const Kv8& c, int64_t bh, int d, int from, int to) {
  const uint16_t* row = c.tail_values(bh) + d * kSlots;
  float sum = 0.f;
#pragma unroll 1
  for (int pos = from; pos <= to; ++pos) {
    const uint32_t x = row[pos & (kSlots - 1)];
    if ((x & 0x7f80u) == 0x7f80u) sum += bf16_bits_to_f32(x);
  }
  return sum;
}

// Scores are scaled by a positive factor: the scale's sign goes to q, a zero to q itself.
struct QuerySign {
  uint32_t keep, flip;
  __device__ explicit QuerySign(float scale)
      : keep(scale == 0.f ? 0u : 0xffffffffu), flip(scale < 0.f ? 0x80008000u : 0u) {}
  __device__ u32x4 operator()(u32x4 q) const { return (q & keep) ^ flip; }
};
__device__ __forceinline__ float positive_scale(float scale) { return (scale == 0.f ? 1.f : fabsf(scale)) * kLog2e; }

// A block's value scale as the weights take it: lv, its logarithm, goes into the weights'
// exponent; lc, the same no further out than 2^-40 and 2^40, into the running maximum's; iv =
// 2^-lc is what the sum takes its weights times.  Past 2^-40 or 2^40 (`apart`) the sum's are
// of their own, 2^(lc - lv) of those for P V: or weights that count in it would be lost
// beside a block of 2^100 times their scale (values that are all zero have 2^-107).  NaN
// stays NaN.
constexpr int kMostScale = 40;
struct ValueScale {
  float lv, lc, iv;
  bool apart;
  __device__ __forceinline__ explicit ValueScale(float vs) {
    lc = lv = __log2f(vs);
    iv = __builtin_amdgcn_rcpf(vs);
    const uint32_t least = (127u - kMostScale) << 23, bits = __builtin_amdgcn_readfirstlane(__float_as_uint(vs));
    apart = bits - least > (2u * kMostScale) << 23;
    if (apart) {
      lc = lv > kMostScale ? kMostScale : lv < 0.f ? -(float)kMostScale : lv;
      iv = __builtin_amdgcn_exp2f(-lc);
    }
  }
};

// N scores of one row and block to weights w[], the running maximum m, sum l and the
// outputs' factor (1 if the maximum stays).
template <int N>
__device__ __forceinline__ float weights(const float (&s)[N], float mx, float sl, const ValueScale& vs, float& m,
                                         float& l, float (&w)[N]) {
  mx = fmaf(mx, sl, vs.lc);
  float alpha = 1.f;
  if (__any(mx > m)) {
    const float mn = fmaxf(m, mx);
    alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    l *= alpha;
    m = mn;
  }
  const float top = m == -INFINITY ? 0.f : m;
  const float off = vs.lv - top;
  float sum = 0.f, own = 0.f;
  if (vs.apart) {
#pragma unroll
    for (int i = 0; i < N; ++i) own += __builtin_amdgcn_exp2f(fmaf(s[i], sl, vs.lc - top));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    w[i] = __builtin_amdgcn_exp2f(fmaf(s[i], sl, off));
    sum += w[i];
  }
  l = fmaf(vs.apart ? own : sum, vs.iv, l);
  return alpha;
}

// The parts of a head, in slots of the workspace (two a workgroup: one for the head that
// its share starts in, one for a later one): `head` of workgroup w0, 2 w of the others up
// to w1.
struct Parts {
  int w0, w1, head;
  __device__ int at(int w) const { return w == w0 ? head : 2 * w; }
};
__device__ __forceinline__ Parts parts_of(const VerifyParams& p, Batch& batch, int b, int h, int nb) {
  const int n = batch.units_of(nb);
  const int u0 = p.c.Hkv * batch.before(b) + h * n;
  if (batch.pieces) {
    const int size = (nb + n - 1) / n;
    return Parts{u0, u0 + (nb + size - 1) / size - 1, 2 * u0};
  }
  const int w0 = u0 / batch.per;
  return Parts{w0, (u0 + nb - 1) / batch.per, 2 * w0 + (u0 > w0 * batch.per ? 1 : 0)};
}

// Running merge of the parts that one lane walks, N at a time (a maximum of -infinity: no
// part); V is the vector of outputs that it holds.
template <class V>
struct Merged {
  float m = -INFINITY, l = 0.f;
  V o = V{};
  template <int N>
  __device__ __forceinline__ void add(const f32x2 (&ml)[N], const V (&po)[N]) {
    float mn = m;
#pragma unroll
    for (int u = 0; u < N; ++u) mn = fmaxf(mn, ml[u].x);
    const float ca = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    l *= ca;
    o *= ca;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const float f = ml[u].x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[u].x - mn);
      l = fmaf(ml[u].y, f, l);
      o += po[u] * f;
    }
    m = mn;
  }
};

// ------------------------------------------------- up to 16 rows (single tokens)
// W waves, block by block in turn, straight from memory to registers: nothing is
// shared.  v_mfma_f32_16x16x32_bf16; lane (r, g) = (lane % 16, lane / 16) has row r.
// Operand row i of K's tile n is position 16 (i / 4) + 8 (n / 2) + 4 (n % 2) + i % 4,
// so that result rows 4 g + e of tiles 2 s and 2 s + 1 are positions 16 g + 8 s .. + 7,
// the ones whose values lie side by side in a row of V^T.  The next block's keys
// are loaded once these are consumed, its values likewise: 16 KB a wave in flight, and no
// barrier before the merge.  Few rows leave the matrix unit idle anyway; what counts is
// bytes in flight.
constexpr int kPartsAhead = 8;

// Parts of up to 16 rows are merged by the workgroup that brings the last one: stored and
// loaded at agent scope, counted after the stores are acknowledged (the protocol and the
// hardware ordering that it rests on are in device_common.h).  In order of their runs,
// whichever comes last.  A second launch instead: 17.9 us against 11.2 (1 token after 500).
__device__ __forceinline__ void store_part(float* base, int64_t i, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(base) + i,
                     (uint64_t)__float_as_uint(x) | ((uint64_t)__float_as_uint(y) << 32), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ f32x2 load_part(const float* base, int64_t i) {
  const uint64_t x = __hip_atomic_load(reinterpret_cast<const uint64_t*>(base) + i, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  return f32x2{__uint_as_float((uint32_t)x), __uint_as_float((uint32_t)(x >> 32))};
}

template <int TYPE, int W>
__global__ __launch_bounds__(64 * W, 2) void attn_verify_q8_rows16_kernel(const VerifyParams p) {
  __shared__ __attribute__((aligned(16))) float so[W][16][kHD + 4];
  __shared__ float sml[W][16][2];
  __shared__ int dropped[2];  // a head's tail values hold a NaN or an infinity
  __shared__ int arrived;
  const Kv8& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 15, g = lane >> 4;
  if (tid == 0) dropped[0] = 0;
  __syncthreads();
  Batch batch(p);
  // sequences that take no part: their rows are zero
  for (int b = blockIdx.x; b < c.B; b += gridDim.x) {
    if (batch.length(b) >= 0) continue;
    const int n = p.T * p.Hq * kHD / 2;
    uint32_t* dst = reinterpret_cast<uint32_t*>(p.out) + (int64_t)b * n;
    for (int i = tid; i < n; i += 64 * W) dst[i] = 0u;
  }
  Share at = share_of(p, batch, blockIdx.x);
  const float sl0 = positive_scale(p.scale);
  const QuerySign sign(p.scale);
  const int nrows = p.T * p.rep;
  const int t = min(p.token_of(r), p.T - 1), rr = r - p.token_of(r) * p.rep;
  const int key0 = 16 * (r >> 2) + (r & 3);  // operand row r of tile n: + 8 (n / 2) + 4 (n % 2)
  bool first_part = true;
  int flag = 0;  // the head's of dropped[]
  while (at.left > 0) {
    const int L = batch.length(at.b);
    const int seen = seen_positions(L, p.T, c.Smax);
    const int nb = (seen + kBlk - 1) >> 6;
    if (nb == 0) {
      ++at.b;
      continue;
    }
    // The next head's flag, last read before the barrier that ended the head before this
    // one, is cleared ahead of this head's barriers: behind them a wave may set it.
    if (tid == 0) dropped[flag ^ 1] = 0;
    const int b1 = min(nb, at.blk + at.left);
    const int base = min(L, c.Smax), done = base >> 6;
    const int64_t bh = (int64_t)at.b * c.Hkv + at.h;
    const int last = min(base + t, seen - 1);  // the last position the lane's row sees
    u32x4 qf[4];  // operand (k / 2, k % 2): features 64 (k / 2) + 16 g + 8 (k % 2) ..
    const uint16_t* qsrc = p.q + (((int64_t)at.b * p.T + t) * p.Hq + at.h * p.rep + rr) * kHD + 16 * g;
    const int coded = min(b1, done);
    int j = at.blk + wave;
#pragma unroll
    for (int k = 0; k < 4; ++k) qf[k] = sign(ld16(qsrc + 64 * (k >> 1) + 8 * (k & 1)));
    float m = -INFINITY, l = 0.f;
    f32x4 o[8];
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float s[16], w[16];
    u32x4 pb[2];
    auto softmax = [&](float sl, const ValueScale& scale) {
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      const float alpha = weights<16>(s, max_over_groups(mx), sl, scale, m, l, w);
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[dt] *= alpha;
      }
      pb[0] = cvt8_bf16(w);
      pb[1] = cvt8_bf16(w + 8);
    };
    if (j < coded) {  // codes: every row sees the whole block
      u32x4 kc[4][2], vc[8];
      float ks = 0.f, vs = 0.f;
      const uint8_t* kb = c.keys(bh, 0) + key0 * kHD + 16 * g;
      const uint8_t* vb = c.values(bh, 0) + r * kBlk + 16 * g;
      const float* ksp = c.ks + bh * c.nblk;
      const float* vsp = c.vs + bh * c.nblk;
      auto load_keys = [&](int j) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int k = 0; k < 2; ++k)
            kc[n][k] = ld16(kb + (int64_t)j * kBlkBytes + (8 * (n >> 1) + 4 * (n & 1)) * kHD + 64 * k);
      };
      auto load_values = [&](int j) {
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) vc[dt] = ld16(vb + (int64_t)j * kBlkBytes + 16 * dt * kBlk);
      };
      load_keys(j);
      load_values(j);
      ks = ksp[j];
      vs = vsp[j];
      do {
        const int next = min(j + W, coded - 1);  // (past the last: loaded again, not used)
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const u32x2 lo = codes_bf16<TYPE>(kc[n][k >> 1][2 * (k & 1)]);
            const u32x2 hi = codes_bf16<TYPE>(kc[n][k >> 1][2 * (k & 1) + 1]);
            acc = mfma_bf16(u32x4{lo.x, lo.y, hi.x, hi.y}, qf[k], acc);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) s[4 * n + e] = acc[e];
        }
        const float sl = sl0 * ks;
        const ValueScale scale(vs);
        load_keys(next);
        ks = ksp[next];
        vs = vsp[next];
        softmax(sl, scale);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const u32x2 lo = codes_bf16<TYPE>(vc[dt][2 * k]), hi = codes_bf16<TYPE>(vc[dt][2 * k + 1]);
            o[dt] = mfma_bf16(u32x4{lo.x, lo.y, hi.x, hi.y}, pb[k], o[dt]);
          }
        load_values(next);
        j += W;
      } while (j < coded);
    }
    for (; j < b1; j += W) {  // the tail, in bf16
      const int slot = (j & 1) * kBlk, p0 = kBlk * j;
      const uint16_t* tk = c.tail_keys(bh) + (slot + key0) * kHD + 16 * g;
      const uint16_t* tv = c.tail_values(bh) + r * kSlots + slot + 16 * g;
      u32x4 kt[4][4], vt[8][2];
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          kt[n][k] = ld16(tk + (8 * (n >> 1) + 4 * (n & 1)) * kHD + 64 * (k >> 1) + 8 * (k & 1));
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) vt[dt][0] = ld16(tv + 16 * dt * kSlots);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < 4; ++k) acc = mfma_bf16(kt[n][k], qf[k], acc);
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[4 * n + e] = p0 + 16 * g + 8 * (n >> 1) + 4 * (n & 1) + e > last ? -INFINITY : acc[e];
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) vt[dt][1] = ld16(tv + 16 * dt * kSlots + 8);
      softmax(sl0, ValueScale(1.f));
      uint32_t bits = 0;
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) bits |= nonfinite_bits(vt[dt][0]) | nonfinite_bits(vt[dt][1]);
      if (__any(any_nonfinite(bits))) {
        if (any_nonfinite(bits)) dropped[flag] = 1;
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
          vt[dt][0] = drop_nonfinite(vt[dt][0]);
          vt[dt][1] = drop_nonfinite(vt[dt][1]);
        }
      }
#pragma unroll
      for (int dt = 0; dt < 8; ++dt)
#pragma unroll
        for (int k = 0; k < 2; ++k) o[dt] = mfma_bf16(vt[dt][k], pb[k], o[dt]);
    }
    // the waves' states through LDS
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    if (g == 0) {
      sml[wave][r][0] = m;
      sml[wave][r][1] = l;
    }
#pragma unroll
    for (int dt = 0; dt < 8; ++dt) *reinterpret_cast<f32x4*>(&so[wave][r][16 * dt + 4 * g]) = o[dt];
    __syncthreads();
    const bool whole = at.blk == 0 && b1 == nb;
    const int64_t part = 2 * (int64_t)blockIdx.x + (first_part ? 0 : 1);
    for (int i = tid; i < nrows * 32; i += 64 * W) {
      const int row = i >> 5, d = (i & 31) * 4;
      const int tt = p.token_of(row), qh = at.h * p.rep + row - tt * p.rep;
      u32x2 gate = {0u, 0u};
      if (whole) gate = load_gate(p, (int64_t)at.b * p.T + tt, qh, d);
      float mm = -INFINITY, ll = 0.f;
#pragma unroll
      for (int x = 0; x < W; ++x) mm = fmaxf(mm, sml[x][row][0]);
      f32x4 oo = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int x = 0; x < W; ++x) {
        const float mw = sml[x][row][0];
        const float f = mw == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(mw - mm);
        ll = fmaf(sml[x][row][1], f, ll);
        oo += *reinterpret_cast<const f32x4*>(&so[x][row][d]) * f;
      }
      if (dropped[flag])
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          const float x = dropped_values(c, bh, d + e, kBlk * max(done, at.blk), min(min(base + tt, seen - 1), kBlk * b1 - 1));
          oo.x += e == 0 ? x : 0.f;
          oo.y += e == 1 ? x : 0.f;
          oo.z += e == 2 ? x : 0.f;
          oo.w += e == 3 ? x : 0.f;
        }
      if (whole) {
        store_gated(p, (int64_t)at.b * p.T + tt, qh, d, oo * (1.f / ll), gate);
      } else {
        const int64_t at2 = ((part * p.part_rows + row) * kHD + d) / 2;
        store_part(p.part_o, at2, oo.x, oo.y);
        store_part(p.part_o, at2 + 1, oo.z, oo.w);
        if (d == 0) store_part(p.part_ml, part * p.part_rows + row, mm, ll);
      }
    }
    if (!whole) {
      const Parts parts = parts_of(p, batch, at.b, at.h, nb);
      __builtin_amdgcn_s_waitcnt(0);  // this thread's part is where every XCD sees it
      __syncthreads();
      if (tid == 0)
        arrived = __hip_atomic_fetch_add(p.count + bh, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (arrived == parts.w1 - parts.w0) {  // the last: merge them, in their order
        if (tid == 0) __hip_atomic_store(p.count + bh, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        const int items = min(nrows * 32, 64 * W), groups = min(64 * W / items, W), group = tid / items;
        for (int i0 = 0; i0 < nrows * 32; i0 += items) {
          const int i = i0 + tid - group * items, row = min(i >> 5, nrows - 1), d = (i & 31) * 4;
          const int tt = p.token_of(row), qh = at.h * p.rep + row - tt * p.rep;
          Merged<f32x4> a;
          u32x2 gate = {0u, 0u};
          if (group == 0) gate = load_gate(p, (int64_t)at.b * p.T + tt, qh, d);
          if (group < groups) {
            for (int w0 = parts.w0; w0 <= parts.w1; w0 += groups * kPartsAhead) {
              f32x2 ml[kPartsAhead];
              f32x4 os[kPartsAhead];
#pragma unroll
              for (int u = 0; u < kPartsAhead; ++u) {
                ml[u] = f32x2{-INFINITY, 0.f};
                os[u] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (w0 + groups * u > parts.w1) continue;  // (no group has a part left)
                const int w = w0 + groups * u + group;
                const int64_t x = (int64_t)parts.at(min(w, parts.w1)) * p.part_rows + row;
                const f32x2 o0 = load_part(p.part_o, (x * kHD + d) / 2), o1 = load_part(p.part_o, (x * kHD + d) / 2 + 1);
                ml[u] = load_part(p.part_ml, x);
                os[u] = f32x4{o0.x, o0.y, o1.x, o1.y};
              }
#pragma unroll
              for (int u = 0; u < kPartsAhead; ++u)
                if (w0 + groups * u + group > parts.w1) {  // (the last again, not to be added: it may be infinite)
                  ml[u].x = -INFINITY;
                  os[u] = f32x4{0.f, 0.f, 0.f, 0.f};
                }
              a.add(ml, os);
            }
            if (d == 0) {
              sml[group][row][0] = a.m;
              sml[group][row][1] = a.l;
            }
            *reinterpret_cast<f32x4*>(&so[group][row][d]) = a.o;
          }
          __syncthreads();
          if (group == 0) {
            const int n = min(groups, parts.w1 - parts.w0 + 1);
            for (int x = 1; x < n; x += 4) {
              f32x2 ml[4];
              f32x4 os[4];
#pragma unroll
              for (int u = 0; u < 4; ++u) {
                const int y = min(x + u, n - 1);
                ml[u] = f32x2{x + u < n ? sml[y][row][0] : -INFINITY, sml[y][row][1]};
                os[u] = *reinterpret_cast<const f32x4*>(&so[y][row][d]);
                if (x + u >= n) os[u] = f32x4{0.f, 0.f, 0.f, 0.f};
              }
              a.add(ml, os);
            }
            if (i < nrows * 32) store_gated(p, (int64_t)at.b * p.T + tt, qh, d, a.o * (1.f / a.l), gate);
          }
          if (64 * W >= 16 * 32) break;  // (one round)
        }
      }
    }
    __syncthreads();
    flag ^= 1;
    first_part = false;
    at.left -= b1 - at.blk;
    at.blk = 0;
    if (b1 == nb && ++at.h == c.Hkv) {
      at.h = 0;
      ++at.b;
    }
  }
}

// ------------------------------------------------- up to 64 rows (draft blocks)
// RT tiles of 32 rows, two waves each: wave half hf takes 32 of a block's 64
// positions, on v_mfma_f32_32x32x16_bf16 (lane: row lane % 32, positions 8 (i / 4) + 4
// (lane / 32) + i % 4 of its half in result element i).  All waves read the same
// block: its codes are loaded once, a block ahead, and become bf16 on their way
// to the other of two LDS buffers, as the prompt kernel's.
// 16 tokens after 131000 (16 heads on 4, int8): 40 us and 6.5 us of merge for 134 MB and
// 17.2 GFLOP.  Two waves a SIMD go through conversion, barrier, scores, softmax and
// products block by block, 1.9 us each (4.4 TB/s), and that chain bounds it beside 10 us of
// start and end: two blocks ahead (46.6 us a call against 45.9), four LDS reads ahead of
// the products and the scales in lanes (no change) left it alone; codes straight to every
// wave's registers took 50.2.
template <int TYPE, int RT>
__global__ __launch_bounds__(128 * RT, 2) void attn_verify_q8_rows64_kernel(const VerifyParams p) {
  constexpr int NT = 128 * RT, PER = kBlk * kHD / 16 / NT;
  constexpr int BUF = 2 * kBlk * kHD * 2;  // bytes of a block's K and V^T in bf16
  __shared__ __attribute__((aligned(16))) unsigned char lds[2 * BUF];
  __shared__ f32x2 sml[RT][2][32];
  __shared__ int dropped[2];  // a head's tail values hold a NaN or an infinity
  const Kv8& c = p.c;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r32 = lane & 31, hl = lane >> 5;
  const int hf = wave / RT, rt = wave % RT;
  if (tid == 0) dropped[0] = 0;
  __syncthreads();
  Batch batch(p);
  Share at = share_of(p, batch, blockIdx.x);
  const float sl0 = positive_scale(p.scale);
  const QuerySign sign(p.scale);
  const int nrows = p.T * p.rep;
  const int row = 32 * rt + r32;
  const int t = min(p.token_of(row), p.T - 1), rr = row - p.token_of(row) * p.rep;
  bool first_part = true;
  int flag = 0;  // the head's of dropped[]
  while (at.left > 0) {
    const int L = batch.length(at.b);
    const int seen = seen_positions(L, p.T, c.Smax);
    const int nb = (seen + kBlk - 1) >> 6;
    if (nb == 0) {
      ++at.b;
      continue;
    }
    // The next head's flag, last read before the barrier that ended the head before this
    // one, is cleared ahead of this head's barriers: behind them a wave may set it.
    if (tid == 0) dropped[flag ^ 1] = 0;
    const int b1 = min(nb, at.blk + at.left);
    const int base = min(L, c.Smax), done = base >> 6;
    const int64_t bh = (int64_t)at.b * c.Hkv + at.h;
    const int last = min(base + t, seen - 1);
    u32x4 kv[PER], vv[PER];
    // Unit i of a thread: K's key kkey + NT / 8 i, features 16 (tid % 8) ..; V^T's feature
    // vrow + NT / 4 i, keys 16 (tid % 4) ..  (both steps multiples of 8: one swizzle).
    const int kkey = tid >> 3, vrow = tid >> 2;
    float ks = 1.f, vs = 1.f;  // of the loaded block
    const float* ksp = c.ks + bh * c.nblk;
    const float* vsp = c.vs + bh * c.nblk;
    auto load_block = [&](int j) {
      if (j >= min(done, b1)) {
        ks = vs = 1.f;
        return;
      }
      ks = ksp[j];
      vs = vsp[j];
      const uint8_t* ksrc = c.keys(bh, j) + 16 * tid;
      const uint8_t* vsrc = c.values(bh, j) + 16 * tid;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        kv[i] = ld16(ksrc + 16 * NT * i);
        vv[i] = ld16(vsrc + 16 * NT * i);
      }
    };
    auto store_pair = [&](unsigned char* row, int piece, int swizzle, u32x4 x, u32x4 y) {
      *reinterpret_cast<u32x4*>(row + ((piece ^ swizzle) << 4)) = x;
      *reinterpret_cast<u32x4*>(row + (((piece + 1) ^ swizzle) << 4)) = y;
    };
    auto store_block = [&](unsigned char* buf, int j) {
      unsigned char* kdst = buf + kkey * 256;
      unsigned char* vdst = buf + BUF / 2 + vrow * 128;
      if (j < done) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          u32x2 x[4];
#pragma unroll
          for (int u = 0; u < 4; ++u) x[u] = codes_bf16<TYPE>(kv[i][u]);
          store_pair(kdst + 32 * NT * i, 2 * (tid & 7), kkey & 7, u32x4{x[0].x, x[0].y, x[1].x, x[1].y},
                     u32x4{x[2].x, x[2].y, x[3].x, x[3].y});
          __builtin_amdgcn_sched_barrier(0);
          // 16 keys: the first piece keeps 0-3 and 8-11 (lane / 32 = 0), the second 4-7 and 12-15
#pragma unroll
          for (int u = 0; u < 4; ++u) x[u] = codes_bf16<TYPE>(vv[i][u]);
          store_pair(vdst + 32 * NT * i, 2 * (tid & 3), vrow & 7, u32x4{x[0].x, x[0].y, x[2].x, x[2].y},
                     u32x4{x[1].x, x[1].y, x[3].x, x[3].y});
          __builtin_amdgcn_sched_barrier(0);
        }
      } else {
        const int slot = (j & 1) * kBlk;
        const uint16_t* ksrc = c.tail_keys(bh) + (slot + kkey) * kHD + (tid & 7) * 16;
        const uint16_t* vsrc = c.tail_values(bh) + vrow * kSlots + slot + (tid & 3) * 16;
        u32x4 kt[PER][2], vt[PER][2];
#pragma unroll
        for (int i = 0; i < PER; ++i)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            kt[i][u] = ld16(ksrc + 16 * NT * i + 8 * u);
            vt[i][u] = ld16(vsrc + 32 * NT * i + 8 * u);
          }
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          store_pair(kdst + 32 * NT * i, 2 * (tid & 7), kkey & 7, kt[i][0], kt[i][1]);
          bits |= nonfinite_bits(vt[i][0]) | nonfinite_bits(vt[i][1]);
          const u32x4 x = drop_nonfinite(vt[i][0]), y = drop_nonfinite(vt[i][1]);
          store_pair(vdst + 32 * NT * i, 2 * (tid & 3), vrow & 7, u32x4{x.x, x.y, y.x, y.y}, u32x4{x.z, x.w, y.z, y.w});
        }
        if (any_nonfinite(bits)) dropped[flag] = 1;
      }
    };
    load_block(at.blk);
    const uint16_t* qsrc = p.q + (((int64_t)at.b * p.T + t) * p.Hq + at.h * p.rep + rr) * kHD + 8 * hl;
    u32x4 qb[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) qb[k] = sign(ld16(qsrc + 16 * k));
    float m = -INFINITY, l = 0.f;
    f32x16 o[4];
#pragma unroll
    for (int dt = 0; dt < 4; ++dt) o[dt] = f32x16{};
#pragma unroll 1
    for (int j = at.blk; j < b1; ++j) {
      // one barrier a block: the buffer that block j + 1 goes to was read before this one
      unsigned char* buf = lds + (j & 1) * BUF;
      store_block(buf, j);
      const float sl = sl0 * ks;
      const ValueScale scale(vs);
      load_block(j + 1);
      __syncthreads();
      const unsigned char* sk = buf + (32 * hf + r32) * 256;
      const unsigned char* sv = buf + BUF / 2 + r32 * 128;
      f32x16 st = {};
#pragma unroll
      for (int k = 0; k < 8; ++k)
        st = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(sk + (((2 * k + hl) ^ (r32 & 7)) << 4))),
            __builtin_bit_cast(bf16x8, qb[k]), st, 0, 0, 0);
      const int k0 = kBlk * j + 32 * hf;
      if (j >= done) {
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + 8 * (i >> 2) + 4 * hl + (i & 3) > last) st[i] = -INFINITY;
      }
      float s[16], w[16];
      float mx = st[0];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = st[i];
        mx = fmaxf(mx, st[i]);
      }
      const f32x2 mb = both_halves(mx);
      const float alpha = weights<16>(s, fmaxf(mb.x, mb.y), sl, scale, m, l, w);
      if (__any(alpha != 1.f)) {
#pragma unroll
        for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
      }
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const u32x4 pb = cvt8_bf16(w + 8 * x);
#pragma unroll
        for (int dt = 0; dt < 4; ++dt)
          o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
              __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(
                                             sv + 32 * dt * 128 + (((2 * (2 * hf + x) + hl) ^ (r32 & 7)) << 4))),
              __builtin_bit_cast(bf16x8, pb), o[dt], 0, 0, 0);
      }
    }
    __syncthreads();
    // Both halves' states through LDS: the waves of a tile finish eight sixteenths of its
    // outputs each, sixteenth q (features 32 (q / 4) + 8 (q % 4) + 4 hl ..) as the lanes
    // hold it.
    f32x4* so = reinterpret_cast<f32x4*>(lds) + rt * (2 * 16 * 64) + lane;
#pragma unroll
    for (int q = 0; q < 16; ++q)
      so[(hf * 16 + q) * 64] = f32x4{o[q >> 2][4 * (q & 3)], o[q >> 2][4 * (q & 3) + 1], o[q >> 2][4 * (q & 3) + 2],
                                     o[q >> 2][4 * (q & 3) + 3]};
    const f32x2 lb = both_halves(l);
    sml[rt][hf][r32] = f32x2{m, lb.x + lb.y};
    __syncthreads();
    const f32x2 ml0 = sml[rt][0][r32], ml1 = sml[rt][1][r32];
    const float mn = fmaxf(ml0.x, ml1.x);
    float c0 = ml0.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml0.x - mn);
    float c1 = ml1.x == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml1.x - mn);
    const float ls = ml0.y * c0 + ml1.y * c1;
    const bool whole = at.blk == 0 && b1 == nb;
    const int64_t part = (2 * (int64_t)blockIdx.x + (first_part ? 0 : 1)) * RT + rt;
    const float inv = whole ? 1.f / ls : 1.f;
    c0 *= inv;
    c1 *= inv;
#pragma unroll 2
    for (int q = 8 * hf; q < 8 * hf + 8; ++q) {
      f32x4 v = so[q * 64] * c0 + so[(16 + q) * 64] * c1;
      const int d = 32 * (q >> 2) + 8 * (q & 3) + 4 * hl;
      if (dropped[flag])
#pragma unroll 1
        for (int e = 0; e < 4; ++e) {
          const float x = dropped_values(c, bh, d + e, kBlk * max(done, at.blk), min(last, kBlk * b1 - 1));
          v.x += e == 0 ? x : 0.f;
          v.y += e == 1 ? x : 0.f;
          v.z += e == 2 ? x : 0.f;
          v.w += e == 3 ? x : 0.f;
        }
      if (!whole) {
        *reinterpret_cast<f32x4*>(p.part_o + part * (32 * kHD) + 256 * q + 4 * lane) = v;
      } else if (row < nrows) {
        const int64_t bt = (int64_t)at.b * p.T + t;
        const int qh = at.h * p.rep + rr;
        store_gated(p, bt, qh, d, v, load_gate(p, bt, qh, d));
      }
    }
    if (!whole && hf == 0 && hl == 0) *reinterpret_cast<f32x2*>(p.part_ml + (part * 32 + r32) * 2) = f32x2{mn, ls};
    __syncthreads();
    flag ^= 1;
    first_part = false;
    at.left -= b1 - at.blk;
    at.blk = 0;
    if (b1 == nb && ++at.h == c.Hkv) {
      at.h = 0;
      ++at.b;
    }
  }
}

// ------------------------------------------------------------------- merge
// The waves take the parts in turn, kMergeAhead loads in flight: up to 128 parts cost one
// trip to memory.
constexpr int kMergeWaves = 16, kMergeAhead = 8;

// Up to 64 rows, a part's outputs as the lanes stored them.  With few heads (p.sliced), a
// workgroup per (sequence, key/value head, tile, sixteenth q of its outputs), whose waves
// take the parts in turn; with many, which have few parts each if any, a workgroup per
// (sequence, head, tile) and a wave per sixteenth.  Slices for all: 128 sequences of 16
// tokens after 200 150 us for 31, 16 after 4096 42 for 29, nearly all workgroups without a
// part; for none: 16 tokens after 131000 75.9 for 46.4, after 4096 22.4 for 15.2.
__global__ __launch_bounds__(64 * kMergeWaves) void attn_verify_q8_merge64_kernel(const VerifyParams p) {
  __shared__ float sm[kMergeWaves][32], sl[kMergeWaves][32];
  __shared__ f32x4 so[kMergeWaves][64];
  const int tiles = p.part_rows >> 5;
  const int hx = p.sliced ? blockIdx.x >> 4 : blockIdx.x;
  const int rt = hx % tiles, h = hx / tiles, b = blockIdx.y;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int q = p.sliced ? blockIdx.x & 15 : wave;
  const int first = p.sliced ? wave : 0, stride = p.sliced ? kMergeWaves : 1;  // of the wave's parts
  const int r32 = lane & 31, hl = lane >> 5, row = 32 * rt + r32;
  const int t = p.token_of(row), qh = h * p.rep + row - t * p.rep, d = 32 * (q >> 2) + 8 * (q & 3) + 4 * hl;
  const bool live = row < p.T * p.rep;
  Batch batch(p);
  const int nb = seen_blocks(__builtin_amdgcn_readfirstlane(p.lens[b]), p.T, p.c.Smax);
  if (nb == 0) {  // takes no part
    if (first == 0 && live)
      *reinterpret_cast<u32x2*>(p.out + (((int64_t)b * p.T + t) * p.Hq + qh) * kHD + d) = u32x2{0u, 0u};
    return;
  }
  const Parts parts = parts_of(p, batch, b, h, nb);
  if (parts.w0 == parts.w1) return;  // finished by its one run
  u32x2 gate = {0u, 0u};
  if (first == 0 && live) gate = load_gate(p, (int64_t)b * p.T + t, qh, d);
  Merged<f32x4> a;
  for (int w = parts.w0 + first; w <= parts.w1; w += stride * kMergeAhead) {
    f32x2 ml[kMergeAhead];
    f32x4 os[kMergeAhead];
#pragma unroll
    for (int u = 0; u < kMergeAhead; ++u) {
      ml[u] = f32x2{-INFINITY, 0.f};
      os[u] = f32x4{0.f, 0.f, 0.f, 0.f};
      if (w + stride * u > parts.w1) continue;
      const int64_t i = (int64_t)parts.at(w + stride * u) * tiles + rt;
      ml[u] = *reinterpret_cast<const f32x2*>(p.part_ml + (i * 32 + r32) * 2);
      os[u] = *reinterpret_cast<const f32x4*>(p.part_o + i * (32 * kHD) + 256 * q + 4 * lane);
    }
    a.add(ml, os);
  }
  if (p.sliced) {
    if (hl == 0) {
      sm[wave][r32] = a.m;
      sl[wave][r32] = a.l;
    }
    so[wave][lane] = a.o;
    __syncthreads();
    if (wave != 0) return;
    f32x2 ml[kMergeWaves - 1];
    f32x4 os[kMergeWaves - 1];
#pragma unroll
    for (int k = 1; k < kMergeWaves; ++k) {  // (a wave without a part left -infinity)
      ml[k - 1] = f32x2{sm[k][r32], sl[k][r32]};
      os[k - 1] = so[k][lane];
    }
    a.add(ml, os);
  }
  if (live) store_gated(p, (int64_t)b * p.T + t, qh, d, a.o * (1.f / a.l), gate);
}

// Rows of a part: the least tile that holds them.  One tile larger, us a call: up to 16
// rows 13.3 for 10.8 (1 token after 500), 77.8 for 45.3 (32 sequences after 8191); up to
// 32 rows 46.5 for 42.6 (8 sequences of 8 tokens after 16000, 16 heads on 4).
// Blocks of a piece where there are few: 2 (16 tokens after 4096: 14.7 us; 1: 15.7, 4: 15.4).
// Workgroups: what the device holds at a time, or fewer for a small cache.  sliced: where
// that makes the merge two rounds of the device at most.  waves (up to 16 rows): eight; two,
// in four times the workgroups, where there are at least as many heads as those, which then
// go side by side instead of one after another: one token of 256 sequences of 4 heads after
// 60 13.9 us for 21.9, after 500 40 for 48, after 4000 159 for 154, 512 of 2 after 100 18.8
// for 36.9; more than 8 rows lose more at length than they gain (4 tokens after 500 55 for 52).
struct VerifyShape {
  int part_rows, min_cut, runs, sliced, waves;
};
VerifyShape verify_shape(int64_t B, int rows, int Hkv, int Smax) {
  const int cus = device_cus() > 0 ? device_cus() : 256;
  VerifyShape v;
  v.part_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
  v.min_cut = 2;
  v.waves = rows <= 8 && B * Hkv >= 4 * cus ? 2 : 8;
  v.sliced = B * Hkv * v.part_rows / 2 <= 2 * cus;
  v.runs = (int)std::max<int64_t>(1, std::min<int64_t>(rows > 16 ? 2 * cus : cus * 8 / v.waves, B * Hkv * ceil_div(Smax / kBlk, v.min_cut)));
  return v;
}

size_t count_bytes(int64_t B, int Hkv) { return (size_t)ceil_div(B * Hkv * 4, 256) * 256; }

template <int TYPE>
void launch_verify(const VerifyParams& p, hipStream_t s) {
  const dim3 grid((unsigned)p.runs);
  if (p.part_rows == 16 && p.waves == 2)
    hipLaunchKernelGGL((attn_verify_q8_rows16_kernel<TYPE, 2>), grid, dim3(64 * 2), 0, s, p);
  else if (p.part_rows == 16)
    hipLaunchKernelGGL((attn_verify_q8_rows16_kernel<TYPE, 8>), grid, dim3(64 * 8), 0, s, p);
  else if (p.part_rows == 32)
    hipLaunchKernelGGL((attn_verify_q8_rows64_kernel<TYPE, 1>), grid, dim3(128), 0, s, p);
  else
    hipLaunchKernelGGL((attn_verify_q8_rows64_kernel<TYPE, 2>), grid, dim3(256), 0, s, p);
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
//   - Weights are rounded to bf16 for P V, as in the verify kernel.
// 4 D operations a pair of positions bound it.  16 heads on 4, e4m3: 4096 rows 87 us, 790
// TFLOP/s; 2048 rows after 14336 280 us, 920 TFLOP/s; a large library product of bf16
// reaches 1300.  int8 takes 92 us for 4096 rows (its bytes take more instructions to
// become bf16).  A turn takes 5000 cycles, of which the matrix unit works 2048; one wave's
// softmax (1400) and staging (1100) run beside the other's products, and what is left over
// is the wait for LDS and for the slower wave at the barrier.
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
  int splits;         // most workgroups that share a row block's turns
  float* part_o;      // [splits, B, P, Hq, D] of a split: softmax . v over its keys alone
  float* part_w;      // [splits, B, P, Hq]: log2 of the sum of its exponentials
  float scale;
};

constexpr int kPRows = 32;                     // query rows of a wave
constexpr int kPKeys = 2 * kBlk;               // keys of a turn
constexpr int kPHalf = kPKeys * kHD * 2;       // bytes of one turn's K (or V^T) in bf16
constexpr int kPMerge = 68 * 64;               // floats that the two waves of a row tile exchange
constexpr int kPPitch = kHD + 4;               // floats of a normalized row in LDS

// Least turns of a split: 2 (600 rows after 1000 29.2 us, 64 after 500 17.0, 300 alone
// 14.6; 1: 29.2, 15.4, 15.4; 4: 29.9, 18.6, 14.6).
constexpr int kSplitTurns = 2;

// Turns of the row block that ends before row `end`, and the splits that share them.
__device__ __forceinline__ int prefill_turns(const PrefillParams& p, int len, int end) {
  return len < 0 ? 0 : (min(min(len, p.c.Smax) + min(end, p.P), p.c.Smax) + kPKeys - 1) / kPKeys;
}
__device__ __forceinline__ int prefill_splits(const PrefillParams& p, int turns) {
  return max(1, min(p.splits, turns / kSplitTurns));
}

constexpr int prefill_lds(int pairs) {
  const int merge = 4 * pairs * (kPMerge + kPRows * kPPitch);
  return merge > 4 * kPHalf ? merge : 4 * kPHalf;
}

// Orders a run of N products with one LDS read each so that READS reads stay ahead of them
// (2048 rows after 14336: 289 us as the compiler orders them, 276 with four; two are the
// same, six 1 % slower).
template <int N, int READS>
__device__ __forceinline__ void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, READS, 0);
#pragma unroll
  for (int i = 0; i < N - READS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
  }
  __builtin_amdgcn_sched_group_barrier(0x008, READS, 0);
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
  const int all = prefill_turns(p, len, t0 + RB * kPRows);
  const int splits = prefill_splits(p, all), split = blockIdx.z;
  if (split >= splits) return;
  const int first = all * split / splits, turns = all * (split + 1) / splits;  // this split's: first .. turns - 1
  const int Lw = len >= 0 && (RB == 1 || tw < p.P) ? min(base + min(tw + kPRows, p.P), c.Smax) : 0;
  if (tid == 0) dropped = 0;
  constexpr int OUT = PAIRS * kPRows * 16 / NT;  // pieces of 8 features of the rows a thread loads and stores
  auto row_of = [&](int e) { return t0 + (RB == 1 ? 0 : (e >> 9) / REP * kPRows) + ((e >> 4) & 31); };
  auto head_of = [&](int e) { return hg * REP + (RB == 1 ? e >> 9 : (e >> 9) % REP); };
  u32x4 kv[PER], vv[PER];
  // K unit e: key e / 8, features 16 (e % 8) ..; V^T unit e: block e / 512, feature
  // (e / 4) % 128, keys 16 (e % 4) ..  A wave's 64 units lie in one block of the turn,
  // half_of: the block's address and the choice between codes and tail are the wave's.
  // Blocks past the cache's last are clamped.
  auto half_of = [&](int i) { return NT == 512 ? i : min(64 * wave + NT * i, UNITS - 1) >> 9; };
  auto block_of = [&](int turn, int i) { return min(2 * turn + half_of(i), c.nblk - 1); };
  auto unit_of = [&](int i) { return NT == 512 ? tid : (tid + NT * i) & 511; };
  auto beyond = [&](int i) { return UNITS % NT != 0 && 64 * wave + NT * i >= UNITS; };
  auto load_keys = [&](int turn, u32x4 (&kv)[PER]) {
    if (turn >= turns) return;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = block_of(turn, i);
      if (j < done) kv[i] = ld16(c.keys(bh, j) + 16 * unit_of(i));
    }
  };
  auto load_values = [&](int turn) {
    if (turn >= turns) return;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int j = block_of(turn, i);
      if (j < done) vv[i] = ld16(c.values(bh, j) + 16 * unit_of(i));
    }
  };
  auto store_pair = [&](unsigned char* row, int piece, int swizzle, u32x4 x, u32x4 y) {
    *reinterpret_cast<u32x4*>(row + ((piece ^ swizzle) << 4)) = x;
    *reinterpret_cast<u32x4*>(row + (((piece + 1) ^ swizzle) << 4)) = y;
  };
  auto store_keys = [&](int turn, const u32x4 (&kv)[PER]) {
    if (turn >= turns) return;
    unsigned char* buf = lds + (turn & 1) * kPHalf;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (beyond(i)) continue;
      const int e = unit_of(i), j = block_of(turn, i), key = e >> 3;
      unsigned char* row = buf + half_of(i) * (kBlk * 256) + key * 256;
      if (j < done) {
        u32x2 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = codes_bf16<TYPE>(kv[i][u]);
        store_pair(row, 2 * (e & 7), key & 7, u32x4{x[0].x, x[0].y, x[1].x, x[1].y}, u32x4{x[2].x, x[2].y, x[3].x, x[3].y});
      } else {
        const uint16_t* src = c.tail_keys(bh) + ((j & 1) * kBlk + key) * kHD + (e & 7) * 16;
        store_pair(row, 2 * (e & 7), key & 7, ld16(src), ld16(src + 8));
      }
    }
  };
  auto store_values = [&](int turn) {
    if (turn >= turns) return;
    unsigned char* buf = lds + 2 * kPHalf + (turn & 1) * kPHalf;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (beyond(i)) continue;
      const int e = unit_of(i), j = block_of(turn, i), d = e >> 2;
      unsigned char* row = buf + half_of(i) * (kHD * 128) + d * 128;
      // 16 keys: the first piece keeps 0-3 and 8-11 (hl = 0), the second 4-7 and 12-15
      if (j < done) {
        u32x2 x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = codes_bf16<TYPE>(vv[i][u]);
        store_pair(row, 2 * (e & 3), d & 7, u32x4{x[0].x, x[0].y, x[2].x, x[2].y}, u32x4{x[1].x, x[1].y, x[3].x, x[3].y});
      } else {
        const uint16_t* src = c.tail_values(bh) + d * kSlots + (j & 1) * kBlk + (e & 3) * 16;
        const u32x4 v0 = ld16(src), v1 = ld16(src + 8);
        if (any_nonfinite(nonfinite_bits(v0) | nonfinite_bits(v1))) dropped = 1;
        const u32x4 x = drop_nonfinite(v0), y = drop_nonfinite(v1);
        store_pair(row, 2 * (e & 3), d & 7, u32x4{x.x, x.y, y.x, y.y}, u32x4{x.z, x.w, y.z, y.w});
      }
    }
  };
  // The queries' rows come whole, 16 lanes a row, and are read back from LDS as the
  // products take them; they stand in the buffer of V first + 1.
  unsigned char* sq = lds + 2 * kPHalf + ((first + 1) & 1) * kPHalf;
  const QuerySign sign(p.scale);
  u32x4 qv[OUT], kv1[PER];
#pragma unroll
  for (int i = 0; i < OUT; ++i) {
    const int e = tid + NT * i;
    qv[i] = ld16(p.q + (((int64_t)b * p.P + min(row_of(e), p.P - 1)) * p.Hq + head_of(e)) * kHD + (e & 15) * 8);
  }
  load_keys(first, kv);
  load_values(first);
  load_keys(first + 1, kv1);
#pragma unroll
  for (int i = 0; i < OUT; ++i) {
    const int e = tid + NT * i;
    *reinterpret_cast<u32x4*>(sq + (e >> 4) * 256 + (((e & 15) ^ ((e >> 4) & 7)) << 4)) = sign(qv[i]);
  }
  __syncthreads();  // the queries are there, and dropped is 0
  u32x4 qb[8];
#pragma unroll
  for (int k = 0; k < 8; ++k)
    qb[k] = *reinterpret_cast<const u32x4*>(sq + (pair * kPRows + r32) * 256 + (((2 * k + hl) ^ (r32 & 7)) << 4));
  store_keys(first, kv);
  store_values(first);
  store_keys(first + 1, kv1);
  load_keys(first + 2, kv);
  load_values(first + 1);
  float m = -INFINITY, l = 0.f;
  f32x16 o[4];
#pragma unroll
  for (int dt = 0; dt < 4; ++dt) o[dt] = f32x16{};
  const float sl0 = positive_scale(p.scale);
  const int last = min(base + tw + r32, Lw - 1);  // the last key this lane's row sees
  f32x16 st[2];
  u32x4 pb[4];
  float ks = 1.f, vs = 1.f;  // of the block whose scores are in st
  auto sees = [&](int turn) { return kBlk * (2 * turn + hf) < Lw; };
  auto scores = [&](int turn) {
    const int kb = 2 * turn + hf;
    ks = vs = 1.f;
    if (kb < done) {
      ks = c.ks[bh * c.nblk + kb];
      vs = c.vs[bh * c.nblk + kb];
    }
    const unsigned char* sk = lds + (turn & 1) * kPHalf + 64 * hf * 256;
    st[0] = st[1] = f32x16{};
#pragma unroll
    for (int k = 0; k < 8; ++k)
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
        st[kt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(
                                           sk + (32 * kt + r32) * 256 + (((2 * k + hl) ^ (r32 & 7)) << 4))),
            __builtin_bit_cast(bf16x8, qb[k]), st[kt], 0, 0, 0);
    reads_ahead<16, 4>();
  };
  auto softmax = [&](int turn) {
    const int k0 = kBlk * (2 * turn + hf);
    const float sl = sl0 * ks;
    const ValueScale scale(vs);
    const bool masked = k0 + 63 > base + tw;  // some row does not see the whole block
    if (masked) {
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (k0 + 32 * kt + 8 * (i >> 2) + 4 * hl + (i & 3) > last) st[kt][i] = -INFINITY;
    }
    float mx = st[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, st[kt][i]);
    const f32x2 mb = both_halves(mx);
    mx = fmaf(fmaxf(mb.x, mb.y), sl, scale.lc);
    if (__any(mx > m)) {
      const float mn = fmaxf(m, mx);
      const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
      l *= alpha;
#pragma unroll
      for (int dt = 0; dt < 4; ++dt) o[dt] *= alpha;
      m = mn;
    }
    const float top = m == -INFINITY ? 0.f : m;
    const float off = scale.lv - top;
    float sum = 0.f, own = 0.f, iv = scale.iv;
    if (scale.apart) {
#pragma unroll
      for (int i = 0; i < 32; ++i) own += __builtin_amdgcn_exp2f(fmaf(st[i >> 4][i & 15], sl, scale.lc - top));
    }
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
    if (masked && !(sl + off == sl + off) && k0 > last) {
      // a block that reads as NaN, past the row's last key: its weights are NaN here, not 0
      sum = own = iv = 0.f;
#pragma unroll
      for (int s = 0; s < 4; ++s) pb[s] = u32x4{0u, 0u, 0u, 0u};
    }
    l = fmaf(scale.apart ? own : sum, iv, l);
  };
  auto outputs = [&](int turn) {
    const unsigned char* sv = lds + 2 * kPHalf + (turn & 1) * kPHalf + hf * (kHD * 128);
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int dt = 0; dt < 4; ++dt)
        o[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
            __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(
                                           sv + (32 * dt + r32) * 128 + (((2 * s + hl) ^ (r32 & 7)) << 4))),
            __builtin_bit_cast(bf16x8, pb[s]), o[dt], 0, 0, 0);
    reads_ahead<16, 4>();
  };
  // K j + 2 and V j + 1 to LDS: the buffers of K j and V j - 1, both read in turn j - 1
  auto stage = [&](int j) {
    store_keys(j + 2, kv);
    store_values(j + 1);
    load_keys(j + 3, kv);
    load_values(j + 2);
  };
  __syncthreads();
  if (sees(first)) {
    scores(first);
    if (hf == 1) softmax(first);
  }
  __syncthreads();  // the first K is read: its buffer takes the third
  // Turn j: the products of K j + 1 and V j.  The first half's waves do their softmax and
  // staging before them, the second half's after: a SIMD holds one wave of each, and the
  // matrix unit has one's products beside the other's arithmetic.
  for (int j = first; j < turns; ++j) {
    if (hf == 0) {
      if (sees(j)) softmax(j);
      stage(j);
    }
    if (sees(j)) outputs(j);
    if (j + 1 < turns && sees(j + 1)) scores(j + 1);
    if (hf == 1) {
      if (j + 1 < turns && sees(j + 1)) softmax(j + 1);
      stage(j);
    }
    __syncthreads();
  }
  int te = tid;  // its rows' addresses are computed again rather than kept through the turns
  asm volatile("" : "+v"(te));
  // The two waves of a row tile exchange halves of their sums through LDS, which each
  // merges and leaves there as normalized rows; every wave then gates and stores whole rows.
  float* red = reinterpret_cast<float*>(lds) + pair * kPMerge + lane;
  float* rows = reinterpret_cast<float*>(lds) + PAIRS * kPMerge;  // [PAIRS][32][kPPitch]
  auto give = [&](const f32x16& x, const f32x16& y) {
    float* to = red + hf * (34 * 64);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      to[i * 64] = x[i];
      to[(16 + i) * 64] = y[i];
    }
    to[32 * 64] = m;
    to[33 * 64] = l;
  };
  if (hf == 0) give(o[2], o[3]);
  else give(o[0], o[1]);
  u32x4 gt[OUT];
  if (splits == 1) {
#pragma unroll
    for (int i = 0; i < OUT; ++i) {
      const int e = te + NT * i;
      gt[i] = ld16(p.gate + ((int64_t)b * p.P + min(row_of(e), p.P - 1)) * p.gate_stride + head_of(e) * 2 * kHD + kHD +
                   (e & 15) * 8);
    }
  }
  __syncthreads();
  {
    const float* from = red + (1 - hf) * (34 * 64);
    const float m1 = from[32 * 64], l1 = from[33 * 64];
    const float mn = fmaxf(m, m1);
    float c0 = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
    float c1 = m1 == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m1 - mn);
    const f32x2 lb = both_halves(l * c0 + l1 * c1);
    const float ls = lb.x + lb.y;
    const float inv = ls == 0.f ? 0.f : 1.f / ls;  // 0: the sequence takes no part
    c0 *= inv;
    c1 *= inv;
    const int64_t part = ((int64_t)split * c.B + b) * p.P;
    if (splits > 1 && hf == 0 && hl == 0 && tw + r32 < p.P) p.part_w[(part + tw + r32) * p.Hq + qh] = mn + __log2f(ls);
    float* row = rows + (pair * kPRows + r32) * kPPitch + 64 * hf + 4 * hl;
    auto merge = [&](const f32x16& x, int dt) {
#pragma unroll
      for (int i4 = 0; i4 < 4; ++i4) {
        f32x4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = x[4 * i4 + e] * c0 + from[(16 * dt + 4 * i4 + e) * 64] * c1;
        *reinterpret_cast<f32x4*>(row + 32 * dt + 8 * i4) = v;
      }
    };
    if (hf == 0) {
      merge(o[0], 0);
      merge(o[1], 1);
    } else {
      merge(o[2], 0);
      merge(o[3], 1);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < OUT; ++i) {
    const int e = te + NT * i, t = row_of(e);
    if (t >= p.P) continue;
    float* row = rows + (e >> 4) * kPPitch + (e & 15) * 8;
    float g[8], v[8];
    if (dropped) {
#pragma unroll 1
      for (int u = 0; u < 8; ++u)
        row[u] += dropped_values(c, bh, (e & 15) * 8 + u, kBlk * done, min(base + t, seen - 1));
    }
    if (splits > 1) {
      float* dst = p.part_o + ((((int64_t)split * c.B + b) * p.P + t) * p.Hq + head_of(e)) * kHD + (e & 15) * 8;
      *reinterpret_cast<f32x4*>(dst) = *reinterpret_cast<const f32x4*>(row);
      *reinterpret_cast<f32x4*>(dst + 4) = *reinterpret_cast<const f32x4*>(row + 4);
      continue;
    }
    unpack8(gt[i], g);
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = row[u] * sigmoid(g[u]);
    *reinterpret_cast<u32x4*>(p.out + (((int64_t)b * p.P + t) * p.Hq + head_of(e)) * kHD + (e & 15) * 8) =
        len < 0 ? u32x4{0u, 0u, 0u, 0u} : pack8(v);  // (whatever the gate holds)
  }
}

// The splits of a row joined, gated and stored: 16 lanes a row of a head, 8 features each.
// A feature that is not finite in a split is so in the row, whatever the split's weight.
// The fp32 rows are read once: 600 rows of 16 heads in three splits, 14.7 MB, 5.2 us.
__global__ __launch_bounds__(256) void attn_prefill_q8_merge_kernel(const PrefillParams p, int block_rows) {
  const int b = blockIdx.y;
  const int64_t e = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (e >= (int64_t)p.P * p.Hq) return;
  const int t = (int)(e / p.Hq), h = (int)(e % p.Hq), f = (threadIdx.x & 15) * 8;
  const int splits = prefill_splits(p, prefill_turns(p, p.lens[b], (t / block_rows + 1) * block_rows));
  if (splits == 1) return;  // the row is stored
  const int64_t row = (int64_t)b * p.P * p.Hq + e, step = (int64_t)p.c.B * p.P * p.Hq;
  const u32x4 gt = ld16(p.gate + ((int64_t)b * p.P + t) * p.gate_stride + h * 2 * kHD + kHD + f);
  typedef float f32x8 __attribute__((ext_vector_type(8)));
  constexpr int AHEAD = 4;
  Merged<f32x8> a;
  f32x8 bad = {};
  for (int k0 = 0; k0 < splits; k0 += AHEAD) {
    f32x2 ml[AHEAD];
    f32x8 os[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      ml[u] = f32x2{-INFINITY, 1.f};
      os[u] = f32x8{};
      if (k0 + u >= splits) continue;
      const int64_t at = (k0 + u) * step + row;
      ml[u].x = p.part_w[at];
      const f32x4 x = *reinterpret_cast<const f32x4*>(p.part_o + at * kHD + f);
      const f32x4 y = *reinterpret_cast<const f32x4*>(p.part_o + at * kHD + f + 4);
      os[u] = __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float y = os[u][i];
        const bool finite = fabsf(y) < INFINITY;
        os[u][i] = finite ? y : 0.f;
        bad[i] += finite ? 0.f : y;
      }
    a.add(ml, os);
  }
  const float inv = a.l == 0.f ? 0.f : 1.f / a.l;
  float g[8], v[8];
  unpack8(gt, g);
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = (a.o[i] * inv + bad[i]) * sigmoid(g[i]);
  *reinterpret_cast<u32x4*>(p.out + row * kHD + f) = pack8(v);
}

// Row blocks of a workgroup: as many as make eight waves, two a SIMD (six with three
// heads), as in the bf16 cache's kernel.  600 rows after 1000 on two heads a workgroup, four
// waves: 46.5 us for 39.5 (before keys were split).
constexpr int prefill_row_blocks(int rep) { return rep == 1 ? 4 : rep == 2 ? 2 : 1; }

template <int TYPE, int REP>
void launch_prefill(const PrefillParams& p, dim3 grid, hipStream_t s) {
  constexpr int RB = prefill_row_blocks(REP);
  hipLaunchKernelGGL((attn_prefill_q8_kernel<TYPE, REP, RB>), grid, dim3(128 * REP * RB), 0, s, p);
}

// The launched heads: up to four query heads of a key/value head together.
int prefill_rep(int per_kv) {
  int rep = 4;
  while (per_kv % rep != 0) --rep;
  return rep;
}

// Splits of a row block's keys: a workgroup fills a CU and takes its time for a turn
// whatever the others do, so as many as the rows' workgroups leave CUs for.  Unsplit, 512
// rows after 32256 took 488 us for 154, 100 after 8000 132 for 28; more splits than one
// round of the device holds are slower where rows see few keys (1500 rows: 51 us for 33).
int most_prefill_splits(int64_t wgs, int Smax) {
  const int64_t cus = device_cus() > 0 ? device_cus() : 256;
  return (int)std::max<int64_t>(1, std::min<int64_t>({cus / wgs, Smax / kPKeys / kSplitTurns, 64}));
}

int prefill_splits_of(int64_t B, int64_t P, int Hq, int Hkv, int Smax) {
  const int rep = prefill_rep(Hq / Hkv);
  return most_prefill_splits(B * ceil_div(P, kPRows * prefill_row_blocks(rep)) * (Hq / rep), Smax);
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
  const int rows = T * (Hq / Hkv);
  const VerifyShape v = verify_shape(B, rows, Hkv, Smax);
  int runs = v.runs;
  if (v.part_rows == 16) runs = std::max(runs, verify_shape(B, 1, Hkv, Smax).runs);  // (fewer rows may have more)
  return count_bytes(B, Hkv) + (size_t)2 * runs * v.part_rows * (kHD + 2) * sizeof(float);
}

extern "C" int dflash_attn_verify_q8(const dflash_kv8_cache* cache, const void* q, const int32_t* lens,
                                     const void* gate_src, int64_t gate_row_stride, void* out, int T, int Hq,
                                     float scale, void* workspace, size_t workspace_bytes, void* stream) {
  VerifyParams p{};
  if (const int rc = check_cache(cache, &p.c)) return rc;
  const int B = p.c.B, Hkv = p.c.Hkv;
  if (T < 0 || T > kMaxDraft || Hq <= 0 || Hq % Hkv != 0 || (int64_t)T * (Hq / Hkv) > 64) return DFLASH_ERR_SHAPE;
  if (gate_row_stride < (int64_t)2 * Hq * kHD) return DFLASH_ERR_SHAPE;
  if ((int64_t)B * T > INT32_MAX || B > 65535 || Hq > 65535 || (int64_t)B * Hkv * p.c.nblk > INT32_MAX / 2) return DFLASH_ERR_SHAPE;
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
  p.rep_inv = 65536u / p.rep + 1;
  const VerifyShape v = verify_shape(B, T * p.rep, Hkv, p.c.Smax);
  p.part_rows = v.part_rows;
  p.min_cut = v.min_cut;
  p.runs = v.runs;
  p.sliced = v.sliced;
  p.waves = v.waves;
  p.count = static_cast<int32_t*>(workspace);
  p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + count_bytes(B, Hkv));
  p.part_ml = p.part_o + (int64_t)2 * p.runs * p.part_rows * kHD;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->type == DFLASH_KV_INT8) launch_verify<DFLASH_KV_INT8>(p, s);
  else launch_verify<DFLASH_KV_E4M3>(p, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.part_rows == 16) return to_status(e);
  hipLaunchKernelGGL(attn_verify_q8_merge64_kernel, dim3((unsigned)(Hkv * p.part_rows / 32 * (p.sliced ? 16 : 1)), (unsigned)B),
                     dim3(64 * kMergeWaves), 0, s, p);
  return to_status(hipGetLastError());
}

extern "C" size_t dflash_attn_prefill_q8_workspace_bytes(int B, int P, int Hq, int Hkv, int Smax) {
  if (B <= 0 || P <= 0 || Hkv <= 0 || Hq <= 0 || Hq % Hkv != 0 || Hq / Hkv > 16 || Smax <= 0 || Smax % kBlk != 0) return 0;
  const int splits = prefill_splits_of(B, P, Hq, Hkv, Smax);
  return splits == 1 ? 0 : (size_t)splits * B * P * Hq * (kHD + 1) * sizeof(float);
}

extern "C" int dflash_attn_prefill_q8(const dflash_kv8_cache* cache, const void* q, const int32_t* lens,
                                      const void* gate_src, int64_t gate_row_stride, void* out, int P, int Hq,
                                      float scale, void* workspace, size_t workspace_bytes, void* stream) {
  PrefillParams p{};
  if (const int rc = check_cache(cache, &p.c)) return rc;
  const int B = p.c.B, Hkv = p.c.Hkv;
  if (P < 0 || Hq <= 0 || Hq % Hkv != 0 || Hq / Hkv > 16 || B > 65535) return DFLASH_ERR_SHAPE;
  if (gate_row_stride < (int64_t)2 * Hq * kHD || P > INT32_MAX - p.c.Smax) return DFLASH_ERR_SHAPE;
  if (B == 0 || P == 0) return DFLASH_OK;
  if (q == nullptr || lens == nullptr || gate_src == nullptr || out == nullptr) return DFLASH_ERR_NULL;
  if (((uintptr_t)q & 15) || ((uintptr_t)gate_src & 15) || gate_row_stride % 8 || ((uintptr_t)out & 15))
    return DFLASH_ERR_ALIGN;
  if (workspace != nullptr) {
    if ((uintptr_t)workspace & 15) return DFLASH_ERR_ALIGN;
    if (workspace_bytes < dflash_attn_prefill_q8_workspace_bytes(B, P, Hq, Hkv, p.c.Smax)) return DFLASH_ERR_WORKSPACE;
  }
  const int rep = prefill_rep(Hq / Hkv);
  p.q = static_cast<const uint16_t*>(q);
  p.lens = lens;
  p.gate = static_cast<const uint16_t*>(gate_src);
  p.gate_stride = gate_row_stride;
  p.out = static_cast<uint16_t*>(out);
  p.P = P; p.Hq = Hq;
  p.heads = Hq / rep;
  p.groups = p.heads / Hkv;
  p.nblk = (int)ceil_div(P, kPRows * prefill_row_blocks(rep));
  // an XCD keeps to one head group, whose codes stay in its L2: 4096 rows 89 us, groups in order 124
  p.xcds = 8 % p.heads == 0 ? 8 / p.heads : 0;
  p.scale = scale;
  const int64_t wgs = p.xcds ? 8 * ceil_div(p.nblk, p.xcds) : (int64_t)p.nblk * p.heads;
  if (wgs > INT32_MAX) return DFLASH_ERR_SHAPE;
  p.splits = workspace == nullptr ? 1 : prefill_splits_of(B, P, Hq, Hkv, p.c.Smax);
  p.part_o = static_cast<float*>(workspace);
  p.part_w = p.part_o + (int64_t)p.splits * B * P * Hq * kHD;
  const dim3 grid((unsigned)wgs, (unsigned)B, (unsigned)p.splits);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->type == DFLASH_KV_INT8) launch_prefill<DFLASH_KV_INT8>(p, rep, grid, s);
  else launch_prefill<DFLASH_KV_E4M3>(p, rep, grid, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || p.splits == 1) return to_status(e);
  hipLaunchKernelGGL(attn_prefill_q8_merge_kernel, dim3((unsigned)ceil_div((int64_t)P * Hq, 16), (unsigned)B), dim3(256),
                     0, s, p, kPRows * prefill_row_blocks(rep));
  return to_status(hipGetLastError());
}
