/*
 * dflash_kv8.h — the 8-bit key/value cache of libdflash_gfx950.so and the
 * attention that reads it.  Conventions (return codes, streams, no allocation,
 * no synchronisation) are those of dflash_gdn.h.
 *
 * A cache of one attention layer holds, for B sequences, Hkv key/value heads of
 * width 128 and Smax positions (a multiple of 64):
 *
 *   codes   every complete block of 64 positions in 8 bits, with one fp32 scale
 *           per block and head for the keys and one for the values:
 *             k_codes [B, Hkv, Smax, 128]          k_scale [B, Hkv, Smax / 64]
 *             v_codes [B, Hkv, Smax / 64, 128, 64] v_scale [B, Hkv, Smax / 64]
 *           (values transposed inside a block: positions contiguous)
 *   tail    the latest two blocks of positions in bf16, position p in slot
 *           p % 128:
 *             tail_k [B, Hkv, 128, 128]   tail_vt [B, Hkv, 128, 128]
 *           (tail_vt transposed: [feature][slot])
 *
 * A scale that 64 positions share must not depend on draft tokens that are
 * rejected later, or decoding would depend on them: drafts go to the tail, and
 * a block is quantised, from the tail's bf16, by the first append whose
 * committed length covers it.  With L committed positions the blocks below
 * L / 64 are read from their codes and the positions from 64 (L / 64) on from
 * the tail.
 *
 * Quantisation of a block x of 64 x 128 values, a = max(max |x|, 2^-100):
 *   DFLASH_KV_INT8  scale = a / 127, code = rint(x * (127 / a))
 *   DFLASH_KV_E4M3  scale = the least power of two with a / scale <= 448,
 *                   code = e4m3(x / scale), to nearest, ties to even
 * A block that holds a NaN or an infinity has scale NaN and codes 0: all of it
 * reads as NaN.
 *
 * Lengths: lens[b] (device int32) is sequence b's committed length before the
 * call's tokens.  lens[b] < 0 marks a sequence that takes no part: nothing of it
 * is written to the cache, and an attention's or a read's rows of it are zero (the
 * append's queries are computed all the same).  Positions at or past Smax are never
 * written nor read; a length that draft tokens carry past Smax stands for the
 * positions below it.  Between two draft appends (at most 16 tokens) lens[b]
 * grows by at most the tokens of the first; it may fall (a rewind) to L as long as
 * the tail still holds what the next call reads: with W the largest position
 * written since the tail was last loaded, plus one, W < 64 (L / 64) + 64 where
 * L % 64 <= 16, else W < 64 (L / 64) + 128 (L = 0 takes nothing from it).
 * dflash_kv8_load sets any state anew.
 */
#ifndef DFLASH_KV8_H
#define DFLASH_KV8_H

#include "dflash_gdn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define DFLASH_KV_INT8 0
#define DFLASH_KV_E4M3 1

/* Every pointer 16-byte aligned, every array contiguous. */
typedef struct {
  void* k_codes;
  void* v_codes;
  float* k_scale;
  float* v_scale;
  void* tail_k;
  void* tail_vt;
  int32_t type; /* DFLASH_KV_INT8 or DFLASH_KV_E4M3 */
  int32_t B, Hkv, Smax;
} dflash_kv8_cache;

/*
 * dflash_attn_prep for this cache (custom_qwen35_model.py:496-522): from the
 * projection rows proj [B*T, proj_row_stride] bf16, [Hq x (query | gate), Hkv x
 * key, Hkv x value] of 128 each, q = rope(rms_norm(query) * q_norm_w) to
 * q_out [B, T, Hq, 128], and keys rope(rms_norm(key) * k_norm_w), rounded to bf16,
 * and values appended at positions lens[b] + t.
 *   prompt == 0: T <= 16 draft tokens.  They go to the tail; block lens[b] / 64 - 1
 *     is quantised from the tail if lens[b] % 64 <= 16 (it may have become complete
 *     since the last append; the same codes again otherwise), the cache's last block if
 *     Smax <= lens[b] <= Smax + 16.
 *   prompt != 0: T committed tokens (lens grows by T).  Every block that they complete
 *     is quantised, and the tail holds the last of those and the open block.
 * overflow (or NULL): [B], set to 1 for a sequence with a position outside
 * [0, Smax).  rot_dims in {0, 16, 32, 64, 128}; Hq a multiple of Hkv; proj, its rows
 * and q_out 16-byte aligned.
 */
int dflash_kv8_append(const dflash_kv8_cache* cache, const void* proj,
                      int64_t proj_row_stride, const void* q_norm_w,
                      const void* k_norm_w, const int32_t* lens, void* q_out,
                      int32_t* overflow, int T, int Hq, int rot_dims,
                      float rope_base, float eps, int prompt, void* stream);

/*
 * Load: positions [0, lens[b]) of every sequence (lens clamped to [0, min(S, Smax)])
 * from bf16 keys and values k, v [B, Hkv, S, 128], the last axis contiguous and
 * the others strided (k_strides, v_strides: b, h, position, in elements, multiples
 * of 8), complete blocks quantised, the last of them and the open block to the tail.
 */
int dflash_kv8_load(const dflash_kv8_cache* cache, const void* k,
                    const int64_t* k_strides, const void* v,
                    const int64_t* v_strides, const int32_t* lens, int S,
                    void* stream);

/*
 * Read: positions start + starts[b] + i, i < count, as bf16 to k_out and v_out
 * [B, Hkv, count, 128] (either may be NULL), as an attention at committed length
 * lens[b] would see them: blocks below lens[b] / 64 as their codes stand for
 * (block lens[b] / 64 - 1, if it may still wait for its codes, as they will stand
 * for), the rest from the tail, which has to hold them at that length (Lengths
 * above).  Positions outside [0, min(lens[b], Smax)) read as zero.  starts may be NULL.
 */
int dflash_kv8_read(const dflash_kv8_cache* cache, const int32_t* lens,
                    const int32_t* starts, int start, int count, void* k_out,
                    void* v_out, void* stream);

/*
 * dflash_attn_verify over this cache: the T <= 16 tokens of each sequence that
 * dflash_kv8_append (prompt == 0) has put at lens[b] attend to the positions 0 ..
 * lens[b] + t:
 *   out[b, t, h*128 ..] = bf16(softmax(scale * q k^T) v * sigmoid(gate))
 * with the gate of head h at h*256 + 128 of row b*T + t of gate_src.  T * Hq / Hkv
 * <= 64.  workspace: dflash_attn_verify_q8_workspace_bytes bytes (enough for any
 * smaller T and Hq too), its first 4 * B * Hkv bytes zero before the first call
 * (every call leaves them zero), not shared by calls that overlap in time.
 */
size_t dflash_attn_verify_q8_workspace_bytes(int B, int T, int Hq, int Hkv,
                                             int Smax);
int dflash_attn_verify_q8(const dflash_kv8_cache* cache, const void* q,
                          const int32_t* lens, const void* gate_src,
                          int64_t gate_row_stride, void* out, int T, int Hq,
                          float scale, void* workspace, size_t workspace_bytes,
                          void* stream);

/*
 * The same over P prompt rows a sequence that dflash_kv8_append (prompt != 0) has put
 * at lens[b]: row i attends to positions 0 .. lens[b] + i.  q [B, P, Hq, 128],
 * out [B, P, Hq*128].  workspace: dflash_attn_prefill_q8_workspace_bytes bytes for
 * these sizes, of any content, not shared by calls that overlap in time: few rows have
 * their keys split over workgroups, which meet there.  NULL (or 0 bytes needed): no split.
 */
size_t dflash_attn_prefill_q8_workspace_bytes(int B, int P, int Hq, int Hkv,
                                              int Smax);
int dflash_attn_prefill_q8(const dflash_kv8_cache* cache, const void* q,
                           const int32_t* lens, const void* gate_src,
                           int64_t gate_row_stride, void* out, int P, int Hq,
                           float scale, void* workspace, size_t workspace_bytes,
                           void* stream);

#ifdef __cplusplus
}
#endif

#endif /* DFLASH_KV8_H */
