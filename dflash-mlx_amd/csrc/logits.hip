// What a request asks of the logits: penalties for repeated tokens, biases and
// grammar masks, applied on the way to the greedy accept or written out for a
// sampler (include/dflash_logits.h has the formulas).
//
// All of it is bound by the logits' bytes (600 KB a row of 151 936 in fp32), so
// the state is kept such that a pass reads little else: a bit a token says
// whether the token has a count or a bias at all, and only where one of eight
// neighbouring bits is set are those eight counts and biases read.  Draft tokens
// before a row are counted from a list in LDS of those that fall into the
// workgroup's slice, mostly none.
#include <hip/hip_runtime.h>
#include <stdint.h>

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
  const uint8_t* known;
  const float* bias;
  const uint8_t* mask;
  float rep, pres, freq;
  const int32_t* drafts;
  int nd;
};

__device__ __forceinline__ int times_drafted(const RowState& s, int v) {
  int n = 0;
  for (int k = 0; k < s.nd; ++k) n += s.drafts[k] == v;
  return n;
}

// Which of entries 8c .. 8c + 7 have a count or a bias.
__device__ __forceinline__ uint32_t known_bits(const RowState& s, int c) {
  uint32_t bits = s.counts != nullptr ? s.known[c] : 0;
  for (int k = 0; k < s.nd; ++k)
    if ((s.drafts[k] >> 3) == c) bits |= 1u << (s.drafts[k] & 7);
  return bits;
}

// Eight whole entries 8c .. 8c + 7.
__device__ __forceinline__ void process8(const RowState& s, int c, uint32_t bits, uint32_t allowed, float (&x)[8]) {
  if (bits) {
    const u32x4_e4* cp = reinterpret_cast<const u32x4_e4*>(s.counts + 8 * c);
    const f32x4_e4* bp = reinterpret_cast<const f32x4_e4*>(s.bias + 8 * c);
    const u32x4 c0 = cp[0], c1 = cp[1];
    const f32x4 b0 = bp[0], b1 = bp[1];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (bits >> e & 1)
        x[e] = penalised(x[e], e < 4 ? c0[e & 3] : c1[e & 3], e < 4 ? b0[e & 3] : b1[e & 3], s.rep, s.pres, s.freq,
                         s.nd ? times_drafted(s, 8 * c + e) : 0);
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (!(allowed >> e & 1)) x[e] = -__builtin_inff();
}

// grid (rows, splits): one workgroup processes one slice of one row, and either
// writes it (WRITE; INPLACE: only what changes) or reduces it to an argmax key.
template <typename T, bool WRITE, bool INPLACE>
__global__ __launch_bounds__(kLThreads) void process_kernel(const ProcessParams p) {
  __shared__ int32_t drafts[DFLASH_LOGITS_MAX_DRAFT];
  __shared__ int nd_s;
  __shared__ uint64_t wbest[kLThreads / 64];
  const int row = blockIdx.x, split = blockIdx.y;
  const int b = row / p.N, i = row - b * p.N;
  const int start = split * p.chunk, end = min(p.V, start + p.chunk);  // chunk % 16 == 0
  const T* base = static_cast<const T*>(p.logits) + b * p.bs + i * p.rs;
  T* out = WRITE ? static_cast<T*>(p.out) + b * p.obs + i * p.ors : nullptr;
  RowState s{};
  const int n_before = p.counts != nullptr ? min(p.n_draft, i) : 0;
  if (p.counts != nullptr) {
    s.counts = p.counts + (int64_t)b * p.V;
    s.known = reinterpret_cast<const uint8_t*>(p.known + (int64_t)b * ((p.V + 31) >> 5));
    s.bias = p.bias + (int64_t)b * p.V;
    s.rep = p.penalties[3 * b], s.pres = p.penalties[3 * b + 1], s.freq = p.penalties[3 * b + 2];
  }
  if (p.mask != nullptr)
    s.mask = reinterpret_cast<const uint8_t*>(p.mask + b * p.mask_bs + i * p.mask_rs);
  if (n_before > 0) {  // wave 0 keeps the slice's drafts, in any order
    if (threadIdx.x < 64) {
      const int d = (int)threadIdx.x < n_before ? p.draft[b * p.dstride + threadIdx.x] : -1;
      const bool in = d >= start && d < end;
      const unsigned long long hit = __ballot(in);
      if (in) drafts[__popcll(hit & ((1ull << threadIdx.x) - 1))] = d;
      if (threadIdx.x == 0) nd_s = __popcll(hit);
    }
    __syncthreads();
    s.drafts = drafts;
    s.nd = nd_s;
  }
  uint64_t best = 0;
  const int c1 = start / 8 + (end - start) / 8;
  for (int c = start / 8 + threadIdx.x; c < c1; c += kLThreads) {
    const uint32_t allowed = s.mask != nullptr ? s.mask[c] : 0xffu;
    const uint32_t bits = known_bits(s, c);
    if (INPLACE && bits == 0 && allowed == 0xffu) continue;
    float x[8];
    load8<T>(base + 8 * c, x);
    process8(s, c, bits, allowed, x);
    if (WRITE) {
      store8<T>(out + 8 * c, x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) best = u64_max(best, argmax_key(x[e], 8 * c + e));
    }
  }
  // the row's last V % 8 entries, a lane each
  const int v = 8 * c1 + threadIdx.x;
  if (v < end) {
    float x = load_logit<T>(base + v);
    if (s.counts != nullptr && known_bits(s, v >> 3) >> (v & 7) & 1)
      x = penalised(x, (uint32_t)s.counts[v], s.bias[v], s.rep, s.pres, s.freq, times_drafted(s, v));
    if (s.mask != nullptr && !(s.mask[v >> 3] >> (v & 7) & 1)) x = -__builtin_inff();
    if (WRITE)
      out[v] = to_bits<T>(x);
    else
      best = u64_max(best, argmax_key(x, v));
  }
  if (WRITE) return;
  best = wave_max_u64(best);
  if ((threadIdx.x & 63) == 0) wbest[threadIdx.x >> 6] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int w = 1; w < kLThreads / 64; ++w) best = u64_max(best, wbest[w]);
    p.keys[(int64_t)row * p.splits + split] = best;
  }
}

// Forget: only what a known bit is set for holds anything.
__global__ __launch_bounds__(kLThreads) void state_reset_kernel(const dflash_logits_state s) {
  const int words = (s.V + 31) >> 5, b = blockIdx.y;
  const int w = blockIdx.x * kLThreads + threadIdx.x;
  if (w == 0) s.penalties[3 * b] = 1.f, s.penalties[3 * b + 1] = 0.f, s.penalties[3 * b + 2] = 0.f;
  if (w >= words) return;
  uint32_t* kp = s.known + (int64_t)b * words + w;
  uint32_t bits = *kp;
  if (bits == 0) return;
  *kp = 0;
  while (bits) {
    const int v = 32 * w + __builtin_ctz(bits);
    bits &= bits - 1;
    if (v >= s.V) break;
    s.counts[(int64_t)b * s.V + v] = 0;
    s.bias[(int64_t)b * s.V + v] = 0.f;
  }
}

// A thread a token.  Integer atomics: the result does not depend on their order.  A
// stale bit only costs the atomic that would have been spared.
__global__ __launch_bounds__(kLThreads) void state_add_kernel(const dflash_logits_state s, const int32_t* tokens,
                                                             int64_t row_stride, int n, const int32_t* lens,
                                                             int prompt) {
  const int b = blockIdx.y;
  const int j = blockIdx.x * kLThreads + threadIdx.x;
  if (j >= (lens != nullptr ? min(n, lens[b]) : n)) return;
  const int v = tokens[b * row_stride + j];
  if ((uint32_t)v >= (uint32_t)s.V) return;
  int32_t* count = s.counts + (int64_t)b * s.V + v;
  if (!prompt)
    atomicAdd(count, 1);
  else if (*count >= 0)
    atomicOr(reinterpret_cast<uint32_t*>(count), ~kCountMask);
  uint32_t* word = s.known + (int64_t)b * ((s.V + 31) >> 5) + (v >> 5);
  const uint32_t bit = 1u << (v & 31);
  if (!(*word & bit)) atomicOr(word, bit);
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
hipError_t launch_process(const ProcessParams& p, int dtype, int B, hipStream_t s) {
  const dim3 grid((unsigned)(B * p.N), (unsigned)p.splits);
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
  const Split sp = plan_split(B, N, V);
  p.logits = logits, p.bs = bs, p.rs = rs;
  p.draft = draft, p.dstride = dstride, p.n_draft = n_draft;
  p.mask = mask, p.mask_bs = mask_bs, p.mask_rs = mask_rs;
  p.N = N, p.V = V, p.chunk = sp.chunk, p.splits = sp.splits;
  return DFLASH_OK;
}

}  // namespace
}  // namespace dflash

using namespace dflash;

extern "C" int dflash_logits_state_reset(const dflash_logits_state* state, void* stream) {
  const int e = check_state(state);
  if (e || state->B == 0) return e;
  const dim3 grid((unsigned)ceil_div(ceil_div(state->V, 32), kLThreads), (unsigned)state->B);
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
  const dim3 grid((unsigned)ceil_div(n, kLThreads), (unsigned)state->B);
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
  return to_status(inplace ? launch_process<true, true>(p, logits_dtype, B, s)
                           : launch_process<true, false>(p, logits_dtype, B, s));
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
  if (workspace_bytes < dflash_greedy_accept_workspace_bytes(B, N, V)) return DFLASH_ERR_WORKSPACE;
  if ((uintptr_t)workspace % 8) return DFLASH_ERR_ALIGN;
  p.keys = static_cast<uint64_t*>(workspace);
  hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t h = launch_process<false, false>(p, logits_dtype, B, s);
  if (h != hipSuccess) return (int)h;
  return to_status(launch_accept_finalize(p.keys, p.splits, B, N, draft, draft_stride, n_draft, posterior, matched,
                                          bonus, s));
}
