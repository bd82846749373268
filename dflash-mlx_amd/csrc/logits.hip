// What a request asks of the logits: penalties for repeated tokens, biases and
// grammar masks, applied on the way to the greedy accept or written out for a
// sampler (include/dflash_logits.h has the formulas).
//
// All of it is bound by the logits' bytes (600 KB a row of 151 936 in fp32), so the state is
// kept such that a pass reads little else: a bit a token says whether the token has a count
// or a bias at all, and only those few are looked up.  Draft tokens before a row are counted
// from a list in LDS of those that fall into the workgroup's slice, mostly none.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "accept_common.h"
#include "argmax_common.h"
#include "device_common.h"
#include "dflash_logits.h"
#include "host_common.h"

namespace dflash {
namespace {

constexpr int kLThreads = 256;
constexpr int kMaxAcceptRows = 16384;
constexpr uint32_t kCountMask = 0x7fffffffu;

// Rows of odd length begin at any element, so the 8 entries a lane works on are
// loaded and stored as vectors of their element's alignment.
typedef u32x4 u32x4_e2 __attribute__((aligned(2)));
typedef u32x4 u32x4_e4 __attribute__((aligned(4)));
typedef f32x4 f32x4_e4 __attribute__((aligned(4)));

struct ProcessParams {
  const void* logits;
  int64_t bs, rs;
  const int32_t* counts;  // null: no state
  const uint32_t* known;
  const float* bias;
  const float* penalties;
  const int32_t* draft;
  int64_t dstride;
  int n_draft;
  const uint32_t* mask;
  int64_t mask_bs, mask_rs;
  void* out;
  int64_t obs, ors;
  uint64_t* keys;
  int N, V, chunk, splits;
  unsigned rows;
};

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]);
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&x)[8]) {
  const f32x4 a = *reinterpret_cast<const f32x4_e4*>(p), b = *reinterpret_cast<const f32x4_e4*>(p + 4);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = a[i], x[4 + i] = b[i];
}
template <>
__device__ __forceinline__ void load8<uint16_t>(const uint16_t* p, float (&x)[8]) {
  const u32x4 a = *reinterpret_cast<const u32x4_e2*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i) x[2 * i] = bf16_lo(a[i]), x[2 * i + 1] = bf16_hi(a[i]);
}
template <>
__device__ __forceinline__ void load8<F16Tag>(const F16Tag* p, float (&x)[8]) {
  const u32x4 a = *reinterpret_cast<const u32x4_e2*>(p);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    x[2 * i] = f16_bits_to_f32((uint16_t)(a[i] & 0xffffu)), x[2 * i + 1] = f16_bits_to_f32((uint16_t)(a[i] >> 16));
}

template <typename T>
__device__ __forceinline__ T to_bits(float x);
template <>
__device__ __forceinline__ float to_bits<float>(float x) { return x; }
template <>
__device__ __forceinline__ uint16_t to_bits<uint16_t>(float x) { return f32_to_bf16_rne(x); }
template <>
__device__ __forceinline__ F16Tag to_bits<F16Tag>(float x) {
  return F16Tag{__builtin_bit_cast(uint16_t, (_Float16)x)};
}

template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&x)[8]) {
  u32x4 a;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    a[i] = (uint32_t)__builtin_bit_cast(uint16_t, to_bits<T>(x[2 * i])) |
           ((uint32_t)__builtin_bit_cast(uint16_t, to_bits<T>(x[2 * i + 1])) << 16);
  *reinterpret_cast<u32x4_e2*>(p) = a;
}
template <>
__device__ __forceinline__ void store8<float>(float* p, const float (&x)[8]) {
  *reinterpret_cast<f32x4_e4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f32x4_e4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
}

// One entry's penalties and bias: every step rounded, none fused, as the header
// writes them.
__device__ __forceinline__ float penalised(float l, uint32_t count, float bias, float rep, float pres, float freq,
                                           int extra) {
#pragma clang fp contract(off)
  const uint32_t made = (count & kCountMask) + (uint32_t)extra;
  if (made > 0 || (count >> 31)) l = l > 0.f ? __fdiv_rn(l, rep) : l * rep;
  if (made > 0) {
    const float f = freq * (float)made;
    l = l - f;
    l = l - pres;
  }
  return l + bias;
}

// The row's part of the state, and the draft tokens before the row that fall into
// the workgroup's slice (in LDS; nd of them).
struct RowState {
  const int32_t* counts;
  const float* bias;
  float rep, pres, freq;
  const int32_t* drafts;
  int nd;
};

__device__ __forceinline__ int times_drafted(const RowState& s, int v) {
  int n = 0;
  for (int k = 0; k < s.nd; ++k) n += s.drafts[k] == v;
  return n;
}

// The entries whose bit of `keep` is 0 as -inf.
__device__ __forceinline__ void keep_bits(float (&x)[8], uint32_t keep) {
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = keep >> e & 1 ? x[e] : -__builtin_inff();
}

// The largest of eight, a NaN above all.
__device__ __forceinline__ float largest(const float (&x)[8]) {
  float m = x[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) m = __builtin_elementwise_maximum(m, x[e]);
  return m;
}

// A slice of a row: a lane has up to kTurns eights of it, 256 apart, whose loads are all in
// flight at once.
constexpr int kListed = 2048;  // known tokens of a slice that are shared out evenly
template <typename T>
constexpr int kTurns = sizeof(T) == 2 ? 4 : 2;
template <typename T>
constexpr int kSlice = 8 * kLThreads * kTurns<T>;

// grid (rows, slices): one workgroup processes one slice of one row, and either writes it
// (WRITE; INPLACE: only the eights in which something changes, whole where a token of one is
// masked: storing the masked entries alone took 185 us where this takes 113, 32 x 16 rows of
// 151936 in fp32 of which 3 % are allowed) or reduces it to an argmax key.
//
// The slice streams by and is only masked: for the argmax a lane keeps the largest value and
// where its eight lie (their order among each other is looked up once, at the end).  The
// known tokens are few and lie unevenly; a lane that worked on one as it met it would have
// its whole wave wait for two trips to memory, and nearly every wave meets one.  So a lane
// leaves an eight with known tokens in LDS and their bits in a register, and then they are
// listed and shared out over all lanes.  32 x 16 rows of 151936 in bf16 under masks after
// 4000 tokens (167 MB), us, with the join of the keys: 112 as met; 67 listed from the bits
// after the stream, whose logits then come a second time; 64 listed turn by turn, 100
// instructions a turn of any wave that meets one; 61 so (masks alone 39).
template <typename T, bool WRITE, bool INPLACE>
__global__ __launch_bounds__(kLThreads) void process_kernel(const ProcessParams p) {
  constexpr int U = kTurns<T>;
  __shared__ int32_t drafts[DFLASH_LOGITS_MAX_DRAFT];
  __shared__ int nd_s, listed;
  __shared__ __attribute__((aligned(16))) T held[kSlice<T>];
  __shared__ uint16_t list[kListed];
  __shared__ uint64_t wbest[kLThreads / 64];
  const int row = blockIdx.x, split = blockIdx.y, tid = threadIdx.x;
  const int b = row / p.N, i = row - b * p.N;
  const int start = split * p.chunk, end = min(p.V, start + p.chunk);  // chunk % 16 == 0, <= kSlice
  const T* base = static_cast<const T*>(p.logits) + b * p.bs + i * p.rs;
  T* out = WRITE ? static_cast<T*>(p.out) + b * p.obs + i * p.ors : nullptr;

  // Where there is no mask or state the row's own bytes stand for theirs: a branch here would
  // have every load wait for the one before.
  const uint8_t* known_row = p.counts == nullptr ? nullptr : reinterpret_cast<const uint8_t*>(p.known + (int64_t)b * ((p.V + 31) >> 5));
  const uint8_t* mask_row = p.mask == nullptr ? nullptr : reinterpret_cast<const uint8_t*>(p.mask + b * p.mask_bs + i * p.mask_rs);
  const uint8_t* mask_at = mask_row != nullptr ? mask_row : reinterpret_cast<const uint8_t*>(base);
  const uint8_t* known_at = known_row != nullptr ? known_row : reinterpret_cast<const uint8_t*>(base);
  const uint32_t mask_or = mask_row != nullptr ? 0 : 0xffu, known_and = known_row != nullptr ? 0xffu : 0;

  // Eights tid, tid + 256, ... of the slice (the last one again where there is none).
  const int c0 = start >> 3, eights = (end - start) >> 3;
  float x[U][8];
  uint32_t allowed[U], known[U];
  if (eights > 0) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int c = c0 + min(tid + k * kLThreads, eights - 1);
      allowed[k] = mask_at[c] | mask_or;
      known[k] = known_at[c] & known_and;
      if (!INPLACE) load8<T>(base + 8 * c, x[k]);
    }
  }

  RowState s{};
  const int n_before = p.counts != nullptr ? min(p.n_draft, i) : 0;
  if (p.counts != nullptr) {
    s.counts = p.counts + (int64_t)b * p.V;
    s.bias = p.bias + (int64_t)b * p.V;
    s.rep = p.penalties[3 * b], s.pres = p.penalties[3 * b + 1], s.freq = p.penalties[3 * b + 2];
  }
  if (tid == 0) listed = 0;
  if (n_before > 0 && tid < 64) {  // wave 0 keeps the slice's drafts, in any order
    const int d = tid < n_before ? p.draft[b * p.dstride + tid] : -1;
    const bool in = d >= start && d < end;
    const unsigned long long hit = __ballot(in);
    if (in) drafts[__popcll(hit & ((1ull << tid) - 1))] = d;
    if (tid == 0) nd_s = __popcll(hit);
  }
  __syncthreads();
  s.drafts = drafts;
  s.nd = n_before > 0 ? nd_s : 0;

  uint64_t key = 0;
  // A known and allowed token v of logit l, with its count and bias.
  auto token = [&](int v, float l, int32_t count, float bias) {
    l = penalised(l, (uint32_t)count, bias, s.rep, s.pres, s.freq, s.nd ? times_drafted(s, v) : 0);
    if (WRITE)
      out[v] = to_bits<T>(l);
    else
      key = u64_max(key, argmax_key(l, v));
  };

  uint32_t due = 0;  // 8 bits a turn: known and allowed
  if (eights > 0) {
    for (int k = 0; k < s.nd; ++k) {  // a draft is known to its lane
      const int e = s.drafts[k] - start;
      if ((e >> 3) % kLThreads == tid)
#pragma unroll
        for (int j = 0; j < U; ++j)
          if ((e >> 3) / kLThreads == j) known[j] |= 1u << (e & 7);
    }
    float best = -__builtin_inff();
    int best_k = -1;
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int at = tid + k * kLThreads, c = c0 + at;
      if (at >= eights) continue;
      const uint32_t mine = known[k] & allowed[k];
      if (INPLACE) {
        if (mine == 0 && allowed[k] == 0xffu) continue;
        load8<T>(base + 8 * c, x[k]);
      }
      due |= mine << (8 * k);
      if (mine) store8<T>(held + 8 * at, x[k]);
      float y[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = x[k][e];
      keep_bits(y, WRITE ? allowed[k] : allowed[k] & ~known[k]);
      if (WRITE) {
        if (!INPLACE || allowed[k] != 0xffu) store8<T>(out + 8 * c, y);
      } else {
        const float m = largest(y);
        if (!(m <= best) && best == best) best = m, best_k = k;  // (the first NaN stays)
      }
    }
    if (!WRITE) {
      key = argmax_key(-__builtin_inff(), start);  // no value of the slice is below it
#pragma unroll
      for (int k = 0; k < U; ++k) {
        if (k != best_k) continue;
        keep_bits(x[k], allowed[k] & ~known[k]);
        int e = 7;
#pragma unroll
        for (int j = 6; j >= 0; --j) e = x[k][j] == best || (x[k][j] != x[k][j] && best != best) ? j : e;
        key = u64_max(key, argmax_key(best, 8 * (c0 + tid + k * kLThreads) + e));
      }
    }
  }
  // the row's last V % 8 entries, a lane each
  if (const int v = 8 * (c0 + eights) + tid; v < end) {
    const bool ok = mask_row == nullptr || (mask_row[v >> 3] >> (v & 7) & 1);
    const bool special = known_row != nullptr && ((known_row[v >> 3] >> (v & 7) & 1) || times_drafted(s, v));
    const float l = load_logit<T>(base + v);
    if (WRITE && !ok) out[v] = to_bits<T>(-__builtin_inff());
    if (WRITE && !INPLACE && ok && !special) out[v] = base[v];
    if (ok && special)
      token(v, l, s.counts[v], s.bias[v]);
    else
      key = u64_max(key, argmax_key(ok ? l : -__builtin_inff(), v));
  }

  if (due) {
    int at = atomicAdd(&listed, __popc(due));
    while (due) {
      const int bit = __builtin_ctz(due), e = 8 * (tid + (bit >> 3) * kLThreads) + (bit & 7);
      due &= due - 1;
      if (at < kListed)
        list[at++] = (uint16_t)e;
      else  // more than there is room for: at once (a lane's store of its own eight is behind it)
        token(start + e, load_logit<T>(held + e), s.counts[start + e], s.bias[start + e]);
    }
  }
  __syncthreads();  // (also: the stores of the listed tokens' eights are done)
  const int n = min(listed, kListed);
  for (int k = tid; k < n; k += 4 * kLThreads) {  // four trips to memory at a time
    int e[4];
    int32_t count[4];
    float bias[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = list[min(k + j * kLThreads, n - 1)];
#pragma unroll
    for (int j = 0; j < 4; ++j) count[j] = s.counts[start + e[j]], bias[j] = s.bias[start + e[j]];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (k + j * kLThreads < n) token(start + e[j], load_logit<T>(held + e[j]), count[j], bias[j]);
  }
  if (WRITE) return;
  key = wave_max_u64(key);
  if ((tid & 63) == 0) wbest[tid >> 6] = key;
  __syncthreads();
  if (tid == 0) {
#pragma unroll
    for (int w = 1; w < kLThreads / 64; ++w) key = u64_max(key, wbest[w]);
    p.keys[(int64_t)row * p.splits + split] = key;
  }
}

// A row's slices: as many as the greedy accept's, or as it takes of at most kSlice.
Split plan_slices(int B, int N, int V, int dtype) {
  const Split sp = plan_split(B, N, V);
  const int chunk = std::min(sp.chunk, dtype == DFLASH_DTYPE_F32 ? kSlice<float> : kSlice<uint16_t>);
  return Split{(int)ceil_div(V, chunk), chunk};
}

// Forget: only what a known bit is set for holds anything.  A thread eight tokens' bits.
__global__ __launch_bounds__(kLThreads) void state_reset_kernel(const dflash_logits_state s) {
  const int words = (s.V + 31) >> 5, b = blockIdx.y;
  const int w = blockIdx.x * kLThreads + threadIdx.x;
  if (w == 0) s.penalties[3 * b] = 1.f, s.penalties[3 * b + 1] = 0.f, s.penalties[3 * b + 2] = 0.f;
  if (w >= 4 * words) return;
  uint8_t* kp = reinterpret_cast<uint8_t*>(s.known + (int64_t)b * words) + w;
  uint32_t bits = *kp;
  if (bits == 0) return;
  *kp = 0;
  for (; bits; bits &= bits - 1) {
    const int v = 8 * w + __builtin_ctz(bits);
    if (v >= s.V) break;
    s.counts[(int64_t)b * s.V + v] = 0;
    s.bias[(int64_t)b * s.V + v] = 0.f;
  }
}

// Four tokens a thread.  In text a few tokens come again and again, and atomics on one address
// take turns (16 000 tokens of 32 sequences of which 5 % are one token: 50 us): a workgroup
// first adds up equal tokens, and the known bits of a word, in tables in LDS, whose place a
// token that finds it taken by another does without.  Integer sums and ORs: the result does
// not depend on the order.
constexpr int kAddTokens = 4 * kLThreads, kAddSlots = 1024;
__global__ __launch_bounds__(kLThreads) void state_add_kernel(const dflash_logits_state s, const int32_t* tokens,
                                                             int64_t row_stride, int n, const int32_t* lens,
                                                             int prompt) {
  __shared__ int32_t token_at[kAddSlots], times[kAddSlots], word_at[kAddSlots];
  __shared__ uint32_t bits_at[kAddSlots];
  const int b = blockIdx.y;
  const int end = lens != nullptr ? min(n, lens[b]) : n;
  if ((int)blockIdx.x * kAddTokens >= end) return;
  int32_t* counts = s.counts + (int64_t)b * s.V;
  uint32_t* known = s.known + (int64_t)b * ((s.V + 31) >> 5);
  int v[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int j = blockIdx.x * kAddTokens + k * kLThreads + threadIdx.x;
    v[k] = j < end ? tokens[b * row_stride + j] : -1;
  }
  for (int k = threadIdx.x; k < kAddSlots; k += kLThreads) token_at[k] = -1, times[k] = 0, word_at[k] = -1, bits_at[k] = 0;
  __syncthreads();
  auto add = [&](int t, int c) {
    if (prompt)
      atomicOr(reinterpret_cast<uint32_t*>(counts + t), ~kCountMask);
    else
      atomicAdd(counts + t, c);
  };
  auto learn = [&](int w, uint32_t bits) {
    if ((known[w] & bits) != bits) atomicOr(known + w, bits);
  };
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if ((uint32_t)v[k] >= (uint32_t)s.V) continue;
    const int slot = ((uint32_t)v[k] * 2654435761u) >> 22;
    const int was = atomicCAS(&token_at[slot], -1, v[k]);
    if (was == -1 || was == v[k])
      atomicAdd(&times[slot], 1);
    else
      add(v[k], 1);
    if (was == v[k]) continue;  // its bit is on its way
    const int w = v[k] >> 5, ws = w & (kAddSlots - 1);
    const int had = atomicCAS(&word_at[ws], -1, w);
    if (had == -1 || had == w)
      atomicOr(&bits_at[ws], 1u << (v[k] & 31));
    else
      learn(w, 1u << (v[k] & 31));
  }
  __syncthreads();
  for (int k = threadIdx.x; k < kAddSlots; k += kLThreads) {
    if (token_at[k] >= 0) add(token_at[k], times[k]);
    if (word_at[k] >= 0) learn(word_at[k], bits_at[k]);
  }
}

// A workgroup a sequence; of an id given twice the last stays.
__global__ __launch_bounds__(kLThreads) void state_set_bias_kernel(const dflash_logits_state s, const int32_t* ids,
                                                                  int64_t ids_stride, const float* values,
                                                                  int64_t values_stride, int n) {
  __shared__ int32_t id[DFLASH_LOGITS_MAX_BIAS];
  const int b = blockIdx.x;
  for (int j = threadIdx.x; j < n; j += kLThreads) id[j] = ids[b * ids_stride + j];
  __syncthreads();
  for (int j = threadIdx.x; j < n; j += kLThreads) {
    const int v = id[j];
    if ((uint32_t)v >= (uint32_t)s.V) continue;
    bool later = false;
    for (int k = j + 1; k < n; ++k) later |= id[k] == v;
    if (later) continue;
    s.bias[(int64_t)b * s.V + v] = values[b * values_stride + j];
    atomicOr(s.known + (int64_t)b * ((s.V + 31) >> 5) + (v >> 5), 1u << (v & 31));
  }
}

int check_state(const dflash_logits_state* s) {
  if (s == nullptr) return DFLASH_ERR_NULL;
  if (s->B < 0 || s->V <= 0 || s->V > INT32_MAX - 64 || s->B > 65535) return DFLASH_ERR_SHAPE;
  if (s->B == 0) return DFLASH_OK;
  for (const void* a : {(const void*)s->counts, (const void*)s->known, (const void*)s->bias, (const void*)s->penalties}) {
    if (a == nullptr) return DFLASH_ERR_NULL;
    if ((uintptr_t)a % 4) return DFLASH_ERR_ALIGN;
  }
  return DFLASH_OK;
}

template <bool WRITE, bool INPLACE>
hipError_t launch_process(const ProcessParams& p, int dtype, hipStream_t s) {
  const dim3 grid(p.rows, p.splits);
  if (dtype == DFLASH_DTYPE_F32)
    hipLaunchKernelGGL((process_kernel<float, WRITE, INPLACE>), grid, dim3(kLThreads), 0, s, p);
  else if (dtype == DFLASH_DTYPE_BF16)
    hipLaunchKernelGGL((process_kernel<uint16_t, WRITE, INPLACE>), grid, dim3(kLThreads), 0, s, p);
  else
    hipLaunchKernelGGL((process_kernel<F16Tag, WRITE, INPLACE>), grid, dim3(kLThreads), 0, s, p);
  return hipGetLastError();
}

// The checks that both entry points share, and their parameters.
int make_params(ProcessParams& p, const void* logits, int dtype, int64_t bs, int64_t rs,
                const dflash_logits_state* state, const int32_t* draft, int64_t dstride, int n_draft,
                const uint32_t* mask, int64_t mask_bs, int64_t mask_rs, int B, int N, int V) {
  if (B < 0 || N <= 0 || V <= 0 || n_draft < 0) return DFLASH_ERR_SHAPE;
  if (N > kMaxAcceptRows || (int64_t)B * N > INT32_MAX || V > INT32_MAX - 64) return DFLASH_ERR_SHAPE;
  if (B == 0) return DFLASH_OK;
  if (logits == nullptr || (n_draft > 0 && draft == nullptr)) return DFLASH_ERR_NULL;
  if (dtype != DFLASH_DTYPE_F32 && dtype != DFLASH_DTYPE_BF16 && dtype != DFLASH_DTYPE_F16)
    return DFLASH_ERR_UNSUPPORTED;
  const int elt = dtype == DFLASH_DTYPE_F32 ? 4 : 2;
  if ((uintptr_t)logits % elt || (uintptr_t)draft % 4 || (uintptr_t)mask % 4) return DFLASH_ERR_ALIGN;
  if (state != nullptr) {
    const int e = check_state(state);
    if (e) return e;
    if (state->B != B || state->V != V) return DFLASH_ERR_SHAPE;
    if ((n_draft < N - 1 ? n_draft : N - 1) > DFLASH_LOGITS_MAX_DRAFT) return DFLASH_ERR_SHAPE;
    p.counts = state->counts, p.known = state->known, p.bias = state->bias, p.penalties = state->penalties;
  }
  const Split sp = plan_slices(B, N, V, dtype);
  if (sp.splits > 65535) return DFLASH_ERR_SHAPE;
  p.logits = logits, p.bs = bs, p.rs = rs;
  p.draft = draft, p.dstride = dstride, p.n_draft = n_draft;
  p.mask = mask, p.mask_bs = mask_bs, p.mask_rs = mask_rs;
  p.N = N, p.V = V, p.chunk = sp.chunk, p.splits = sp.splits;
  p.rows = (unsigned)(B * N);
  return DFLASH_OK;
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" int dflash_logits_state_reset(const dflash_logits_state* state, void* stream) {
  const int e = check_state(state);
  if (e || state->B == 0) return e;
  const dim3 grid((unsigned)ceil_div(4 * ceil_div(state->V, 32), kLThreads), (unsigned)state->B);
  hipLaunchKernelGGL(state_reset_kernel, grid, dim3(kLThreads), 0, static_cast<hipStream_t>(stream), *state);
  return to_status(hipGetLastError());
}

extern "C" int dflash_logits_state_add(const dflash_logits_state* state, const int32_t* tokens, int64_t row_stride,
                                       int n, const int32_t* lens, int prompt, void* stream) {
  const int e = check_state(state);
  if (e) return e;
  if (n < 0) return DFLASH_ERR_SHAPE;
  if (n == 0 || state->B == 0) return DFLASH_OK;
  if (tokens == nullptr) return DFLASH_ERR_NULL;
  if ((uintptr_t)tokens % 4 || (uintptr_t)lens % 4) return DFLASH_ERR_ALIGN;
  const dim3 grid((unsigned)ceil_div(n, kAddTokens), (unsigned)state->B);
  hipLaunchKernelGGL(state_add_kernel, grid, dim3(kLThreads), 0, static_cast<hipStream_t>(stream), *state, tokens,
                     row_stride, n, lens, prompt);
  return to_status(hipGetLastError());
}

extern "C" int dflash_logits_state_set_bias(const dflash_logits_state* state, const int32_t* ids, int64_t ids_stride,
                                            const float* values, int64_t values_stride, int n, void* stream) {
  const int e = check_state(state);
  if (e) return e;
  if (n < 0 || n > DFLASH_LOGITS_MAX_BIAS) return DFLASH_ERR_SHAPE;
  if (n == 0 || state->B == 0) return DFLASH_OK;
  if (ids == nullptr || values == nullptr) return DFLASH_ERR_NULL;
  if ((uintptr_t)ids % 4 || (uintptr_t)values % 4) return DFLASH_ERR_ALIGN;
  hipLaunchKernelGGL(state_set_bias_kernel, dim3((unsigned)state->B), dim3(kLThreads), 0,
                     static_cast<hipStream_t>(stream), *state, ids, ids_stride, values, values_stride, n);
  return to_status(hipGetLastError());
}

extern "C" int dflash_logits_process(const void* logits, int logits_dtype, int64_t batch_stride, int64_t row_stride,
                                     const dflash_logits_state* state, const int32_t* draft, int64_t draft_stride,
                                     int n_draft, const uint32_t* mask, int64_t mask_batch_stride,
                                     int64_t mask_row_stride, void* out, int64_t out_batch_stride,
                                     int64_t out_row_stride, int B, int N, int V, void* stream) {
  ProcessParams p{};
  const int e = make_params(p, logits, logits_dtype, batch_stride, row_stride, state, draft, draft_stride, n_draft,
                            mask, mask_batch_stride, mask_row_stride, B, N, V);
  if (e || B == 0) return e;
  if (out == nullptr) return DFLASH_ERR_NULL;
  if ((uintptr_t)out % (logits_dtype == DFLASH_DTYPE_F32 ? 4 : 2)) return DFLASH_ERR_ALIGN;
  const bool inplace = out == logits;
  if (inplace && (out_batch_stride != batch_stride || out_row_stride != row_stride)) return DFLASH_ERR_SHAPE;
  p.out = out, p.obs = out_batch_stride, p.ors = out_row_stride;
  hipStream_t s = static_cast<hipStream_t>(stream);
  return to_status(inplace ? launch_process<true, true>(p, logits_dtype, s)
                           : launch_process<true, false>(p, logits_dtype, s));
}

extern "C" size_t dflash_greedy_accept_processed_workspace_bytes(int B, int N, int V) {
  if (B <= 0 || N <= 0 || V <= 0) return 0;
  return sizeof(uint64_t) * (size_t)B * N * plan_slices(B, N, V, DFLASH_DTYPE_F32).splits;
}

extern "C" int dflash_greedy_accept_processed(const void* logits, int logits_dtype, int64_t batch_stride,
                                              int64_t row_stride, const int32_t* draft, int64_t draft_stride,
                                              int n_draft, const dflash_logits_state* state, const uint32_t* mask,
                                              int64_t mask_batch_stride, int64_t mask_row_stride, int32_t* posterior,
                                              int32_t* matched, int32_t* bonus, int B, int N, int V, void* workspace,
                                              size_t workspace_bytes, void* stream) {
  ProcessParams p{};
  const int e = make_params(p, logits, logits_dtype, batch_stride, row_stride, state, draft, draft_stride, n_draft,
                            mask, mask_batch_stride, mask_row_stride, B, N, V);
  if (e || B == 0) return e;
  if (workspace == nullptr || (posterior == nullptr && matched == nullptr && bonus == nullptr)) return DFLASH_ERR_NULL;
  if (workspace_bytes < sizeof(uint64_t) * (size_t)B * N * p.splits) return DFLASH_ERR_WORKSPACE;
  if ((uintptr_t)workspace % 8) return DFLASH_ERR_ALIGN;
  p.keys = static_cast<uint64_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t h = launch_process<false, false>(p, logits_dtype, s);
  if (h != hipSuccess) return (int)h;
  return to_status(launch_accept_finalize(p.keys, p.splits, B, N, draft, draft_stride, n_draft, posterior, matched,
                                          bonus, s));
}
