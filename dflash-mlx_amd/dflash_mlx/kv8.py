"""The 8-bit key/value cache of an attention layer, and the ops over it.

A decode step reads the whole cache, so its bytes set the step's time at long
contexts; a cache in 8 bits halves them (and the memory).  ``QuantizedKVCache``
holds complete blocks of 64 positions as int8 or e4m3 codes with one fp32
scale per block and head, keys and values apart, and the latest two blocks of
positions in bf16 (the tail).  A block gets its codes only once all its
positions are committed, from the tail: what the cache holds of the kept
tokens never depends on draft tokens that were rejected.  A step at committed
length L reads the blocks below L // 64 from their codes, so a token that ends a
block is read in bf16 by the steps that start before its end and from its code
by those after.

The ops take the place of the bf16 cache's append (q/k RMSNorm, rotary, KV
append; custom_qwen35_model.py:496-522) and attention (causal SDPA over the
cache, sigmoid gate; :524-534):

* ``attn_prep_q8``: queries, and the new keys and values into the cache;
* ``attn_verify_q8``: attention of a draft block (1 to 16 tokens) a sequence;
* ``attn_prefill_q8``: attention of a prompt's rows;
* ``kv_load_q8`` / ``kv_read_q8``: bf16 keys and values into a cache and back.

``lens`` is always the committed length per sequence before the call's tokens
(device int32 [B]; negative: the sequence takes no part).  Layout, quantisation
and the contract on lengths are in include/dflash_kv8.h.  Every op runs
hand-written gfx950 kernels on torch's current stream of its tensors' device;
there is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .gated_delta import _require_device

BLOCK = 64   # positions that share a scale
SLOTS = 128  # tail slots: position p is in slot p % SLOTS
HEAD_DIM = 128
MAX_DRAFT = 16

_TYPES = {torch.int8: 0, torch.float8_e4m3fn: 1}
_I64x3 = ctypes.c_int64 * 3


class _CCache(ctypes.Structure):
    """dflash_kv8_cache of include/dflash_kv8.h."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("k_codes", "v_codes", "k_scale", "v_scale", "tail_k", "tail_vt")] + [
        (n, ctypes.c_int32) for n in ("type", "B", "Hkv", "Smax")]


class QuantizedKVCache:
    """Keys and values of B sequences and Hkv heads of width 128, Smax positions
    (a multiple of 64), in caller-owned tensors:

    k_codes [B, Hkv, Smax, 128] and v_codes [B, Hkv, Smax/64, 128, 64] (int8 or
    float8_e4m3fn), k_scale and v_scale [B, Hkv, Smax/64] fp32, tail_k [B, Hkv,
    128 slots, 128] and tail_vt [B, Hkv, 128, 128 slots] bf16; all contiguous, on
    one device."""

    __slots__ = ("k_codes", "v_codes", "k_scale", "v_scale", "tail_k", "tail_vt", "B", "Hkv", "Smax", "dtype",
                 "device", "_struct", "_ptr", "_lens_shape", "_ws_bytes", "_workspaces")

    def __init__(self, k_codes, v_codes, k_scale, v_scale, tail_k, tail_vt):
        _require_device("k_codes", k_codes)
        if k_codes.dtype not in _TYPES:
            raise TypeError(f"codes must be int8 or float8_e4m3fn, got {k_codes.dtype}")
        if k_codes.dim() != 4 or k_codes.shape[3] != HEAD_DIM:
            raise ValueError(f"k_codes must be [B, Hkv, Smax, {HEAD_DIM}], got {tuple(k_codes.shape)}")
        B, Hkv, Smax, D = k_codes.shape
        if Smax == 0 or Smax % BLOCK:
            raise ValueError(f"Smax must be a positive multiple of {BLOCK}, got {Smax}")
        nb, bf = Smax // BLOCK, torch.bfloat16
        for name, t, shape, dtype in (
                ("k_codes", k_codes, (B, Hkv, Smax, D), k_codes.dtype),
                ("v_codes", v_codes, (B, Hkv, nb, D, BLOCK), k_codes.dtype),
                ("k_scale", k_scale, (B, Hkv, nb), torch.float32), ("v_scale", v_scale, (B, Hkv, nb), torch.float32),
                ("tail_k", tail_k, (B, Hkv, SLOTS, D), bf), ("tail_vt", tail_vt, (B, Hkv, D, SLOTS), bf)):
            _require_device(name, t, k_codes.device)
            if t.dtype is not dtype:
                raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
            if tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {list(shape)}, got {list(t.shape)}")
        self.k_codes, self.v_codes, self.k_scale, self.v_scale = k_codes, v_codes, k_scale, v_scale
        self.tail_k, self.tail_vt = tail_k, tail_vt
        self.B, self.Hkv, self.Smax, self.dtype, self.device = B, Hkv, Smax, k_codes.dtype, k_codes.device
        self._struct = _CCache(k_codes.data_ptr(), v_codes.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(),
                               tail_k.data_ptr(), tail_vt.data_ptr(), _TYPES[k_codes.dtype], B, Hkv, Smax)
        self._ptr = ctypes.addressof(self._struct)
        self._lens_shape = (B,)
        self._ws_bytes = {}    # attn_verify_q8's, by (T, heads)
        self._workspaces = {}  # by stream: calls on one stream do not overlap

    @classmethod
    def zeros(cls, B: int, Hkv: int, Smax: int, dtype: torch.dtype, device) -> "QuantizedKVCache":
        """An empty cache: every position reads as zero."""
        if dtype not in _TYPES:
            raise TypeError(f"codes must be int8 or float8_e4m3fn, got {dtype}")
        if B < 0 or Hkv <= 0 or Smax <= 0 or Smax % BLOCK:
            raise ValueError(f"need B >= 0, Hkv > 0 and Smax a positive multiple of {BLOCK}, got {B}, {Hkv}, {Smax}")
        nb, D, bf = Smax // BLOCK, HEAD_DIM, torch.bfloat16
        z = lambda dt, *s: torch.zeros(*s, dtype=dt, device=device)  # noqa: E731
        codes = lambda *s: z(torch.uint8, *s).view(dtype)  # noqa: E731
        ones = lambda: torch.ones(B, Hkv, nb, dtype=torch.float32, device=device)  # noqa: E731
        return cls(codes(B, Hkv, Smax, D), codes(B, Hkv, nb, D, BLOCK), ones(), ones(), z(bf, B, Hkv, SLOTS, D),
                   z(bf, B, Hkv, D, SLOTS))

    def __repr__(self):
        return f"QuantizedKVCache({self.dtype}, B={self.B}, Hkv={self.Hkv}, Smax={self.Smax}, {self.device})"


def _call(fn: str, dev: torch.device, *args) -> None:
    """The entry point on the tensors' device and its current stream."""
    if torch.cuda.current_device() == dev.index:
        _lib.call(fn, *args, _lib.stream_handle(dev))
    else:
        with torch.cuda.device(dev):
            _lib.call(fn, *args, _lib.stream_handle(dev))


# The checks below test for what is right in one expression and say what is wrong
# only afterwards: a small call's time is all host work.

def _check_cache(cache) -> None:
    if not isinstance(cache, QuantizedKVCache):
        raise TypeError(f"cache must be a QuantizedKVCache, got {type(cache).__name__}")


def _check_lens(name: str, lens, cache) -> None:
    if isinstance(lens, torch.Tensor) and (lens.dtype is torch.int32 and lens.shape == cache._lens_shape
                                           and lens.device == cache.device and lens.is_contiguous()):
        return
    _require_device(name, lens, cache.device)
    if lens.dtype is not torch.int32:
        raise TypeError(f"{name} must be int32, got {lens.dtype}")
    raise ValueError(f"{name} must be contiguous [{cache.B}], got {tuple(lens.shape)}")


def _row_stride(name: str, proj, cache, T: int | None, width: int) -> int:
    """Row stride of the projection rows [B, T, >= width], which are evenly
    spaced and 16-byte aligned."""
    if isinstance(proj, torch.Tensor) and proj.dim() == 3:
        (b, t, w), (sb, st, se) = proj.shape, proj.stride()
        row = st if t > 1 else sb if b > 1 else max(st, w)
        if (proj.dtype is torch.bfloat16 and proj.device == cache.device and b == cache.B and (T is None or t == T)
                and w >= width and se == 1 and row >= w and (b == 1 or t == 1 or sb == t * row) and row % 8 == 0
                and proj.data_ptr() % 16 == 0):
            return row
    _require_device(name, proj, cache.device)
    if proj.dtype is not torch.bfloat16:
        raise TypeError(f"{name} must be bfloat16, got {proj.dtype}")
    if proj.dim() != 3 or proj.shape[0] != cache.B or (T is not None and proj.shape[1] != T) or proj.shape[2] < width:
        raise ValueError(f"{name} must be [{cache.B}, {'T' if T is None else T}, at least {width}], "
                         f"got {tuple(proj.shape)}")
    if proj.numel() == 0:
        return -(-width // 8) * 8
    raise ValueError(f"{name} rows must be contiguous, evenly spaced over [B, T] and 16-byte aligned, "
                     f"got strides {tuple(proj.stride())}")


def _check_queries(q, cache):
    if isinstance(q, torch.Tensor) and q.dim() == 4:
        b, t, h, d = q.shape
        if (q.dtype is torch.bfloat16 and b == cache.B and d == HEAD_DIM and h and h % cache.Hkv == 0
                and q.device == cache.device):
            return t, h
    _require_device("q", q, cache.device)
    if q.dtype is not torch.bfloat16:
        raise TypeError(f"q must be bfloat16, got {q.dtype}")
    raise ValueError(f"q must be [{cache.B}, T, a multiple of {cache.Hkv} heads, {HEAD_DIM}], got {tuple(q.shape)}")


_NORM_SHAPE = (HEAD_DIM,)


def _check_norm(name: str, w, cache) -> None:
    if isinstance(w, torch.Tensor) and (w.dtype is torch.bfloat16 and w.shape == _NORM_SHAPE
                                        and w.device == cache.device and w.is_contiguous()):
        return
    _require_device(name, w, cache.device)
    raise ValueError(f"{name} must be contiguous bfloat16 [{HEAD_DIM}], got {w.dtype} {tuple(w.shape)}")


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """t, or a contiguous 16-byte aligned copy."""
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def attn_prep_q8(proj, q_norm, k_norm, lens, cache: QuantizedKVCache, *, num_heads: int, rot_dims: int,
                 rope_base: float, eps: float = 1e-6, prompt: bool = False, overflow=None):
    """Queries [B, T, num_heads, 128] bf16 from the projection rows, the new keys
    and values appended to the cache at lens[b] + t.

    proj: bf16 [B, T, >= (2 num_heads + 2 Hkv) 128], rows evenly spaced and 16-byte
    aligned, laid out [heads x (query | gate), Hkv x key, Hkv x value]; q_norm, k_norm: bf16 [128] RMSNorm weights;
    rotary over the first rot_dims (0, 16, 32, 64 or 128) features.

    prompt=False: T <= 16 draft tokens, of which any number may be rejected (the
    next call's lens says how many were kept).  prompt=True: T committed tokens, all
    of them: lens grows by T.  (Prompts of several lengths, which padding would
    commit too: a call for each length, with lens -1 for the other sequences.)
    overflow (int32 [B], optional) is set to 1 for a sequence with positions
    outside the cache, lens -1 among them, which are not written."""
    _check_cache(cache)
    _check_lens("lens", lens, cache)
    if num_heads <= 0 or num_heads % cache.Hkv:
        raise ValueError(f"num_heads must be a positive multiple of {cache.Hkv}, got {num_heads}")
    row = _row_stride("proj", proj, cache, None, (2 * num_heads + 2 * cache.Hkv) * HEAD_DIM)
    T = proj.shape[1]
    if not prompt and T > MAX_DRAFT:
        raise ValueError(f"a draft append takes at most {MAX_DRAFT} tokens, got {T} (prompt=True for committed ones)")
    _check_norm("q_norm", q_norm, cache)
    _check_norm("k_norm", k_norm, cache)
    if overflow is not None:
        _check_lens("overflow", overflow, cache)
    q = torch.empty((cache.B, T, num_heads, HEAD_DIM), dtype=torch.bfloat16, device=cache.device)
    _call("dflash_kv8_append", cache.device, cache._ptr, proj.data_ptr(), row, q_norm.data_ptr(), k_norm.data_ptr(),
          lens.data_ptr(), q.data_ptr(), _lib.ptr(overflow), T, num_heads, int(rot_dims), float(rope_base), float(eps),
          int(bool(prompt)))
    return q


def attn_verify_q8_workspace_bytes(B: int, T: int, num_heads: int, Hkv: int, Smax: int) -> int:
    """Bytes of attn_verify_q8's workspace (for the current device)."""
    return int(_lib.load().dflash_attn_verify_q8_workspace_bytes(B, T, num_heads, Hkv, Smax))


def _verify_workspace(cache: QuantizedKVCache, T: int, Hq: int) -> torch.Tensor:
    """The cache's workspace of its device's current stream; of a captured graph its own."""
    if torch.cuda.current_device() != cache.device.index:  # (the capture's state is the current device's)
        with torch.cuda.device(cache.device):
            return _verify_workspace(cache, T, Hq)
    n = cache._ws_bytes.get((T, Hq))
    if n is None:
        n = cache._ws_bytes[(T, Hq)] = attn_verify_q8_workspace_bytes(cache.B, T, Hq, cache.Hkv, cache.Smax)
    capturing = torch.cuda.is_current_stream_capturing()
    stream = _lib.stream_handle(cache.device)
    ws = None if capturing else cache._workspaces.get(stream)
    if ws is None or ws.numel() < n:
        ws = torch.empty(n, dtype=torch.uint8, device=cache.device)
        ws[:4 * cache.B * cache.Hkv].zero_()
        if not capturing:
            cache._workspaces[stream] = ws
    return ws


def attn_verify_q8(q, cache: QuantizedKVCache, lens, proj, *, scale: float | None = None, workspace=None):
    """Attention of the T <= 16 tokens a sequence that attn_prep_q8 (prompt=False)
    appended at lens[b]: token t sees positions 0 .. lens[b] + t.

    q: bf16 [B, T, Hq, 128]; proj: the projection rows (the gate of head h at
    256 h + 128); T * Hq / Hkv <= 64; scale: 128 ** -0.5 by default.  workspace
    (optional): uint8, attn_verify_q8_workspace_bytes bytes, the first 4 B Hkv zero
    before its first use; calls that overlap in time must not share it.  By default
    the cache keeps one a stream, and a captured graph gets its own.  Returns
    softmax(scale q k^T) v * sigmoid(gate), bf16 [B, T, Hq * 128]."""
    _check_cache(cache)
    _check_lens("lens", lens, cache)
    T, Hq = _check_queries(q, cache)
    if T > MAX_DRAFT or T * (Hq // cache.Hkv) > 64:
        raise ValueError(f"at most {MAX_DRAFT} tokens and 64 query rows a key/value head, got T = {T}, {Hq} heads")
    row = _row_stride("proj", proj, cache, T, 2 * Hq * HEAD_DIM)
    out = torch.empty((cache.B, T, Hq * HEAD_DIM), dtype=torch.bfloat16, device=cache.device)
    if out.numel() == 0:
        return out
    if workspace is None:
        workspace = _verify_workspace(cache, T, Hq)
    else:
        _require_device("workspace", workspace, cache.device)
        if workspace.dtype is not torch.uint8 or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous uint8")
    q = _aligned(q)
    _call("dflash_attn_verify_q8", cache.device, cache._ptr, q.data_ptr(), lens.data_ptr(), proj.data_ptr(), row,
          out.data_ptr(), T, Hq, HEAD_DIM ** -0.5 if scale is None else float(scale), workspace.data_ptr(),
          workspace.numel())
    return out


def attn_prefill_q8_workspace_bytes(B: int, P: int, num_heads: int, Hkv: int, Smax: int) -> int:
    """Bytes of attn_prefill_q8's workspace: 0 where the rows alone fill the device."""
    return int(_lib.load().dflash_attn_prefill_q8_workspace_bytes(B, P, num_heads, Hkv, Smax))


def attn_prefill_q8(q, cache: QuantizedKVCache, lens, proj, *, scale: float | None = None):
    """attn_verify_q8 over the P rows a sequence that attn_prep_q8 (prompt=True)
    appended at lens[b]: row i sees positions 0 .. lens[b] + i."""
    _check_cache(cache)
    _check_lens("lens", lens, cache)
    P, Hq = _check_queries(q, cache)
    row = _row_stride("proj", proj, cache, P, 2 * Hq * HEAD_DIM)
    out = torch.empty((cache.B, P, Hq * HEAD_DIM), dtype=torch.bfloat16, device=cache.device)
    n = attn_prefill_q8_workspace_bytes(cache.B, P, Hq, cache.Hkv, cache.Smax)
    workspace = torch.empty(n, dtype=torch.uint8, device=cache.device) if n else None
    q = _aligned(q)
    _call("dflash_attn_prefill_q8", cache.device, cache._ptr, q.data_ptr(), lens.data_ptr(), proj.data_ptr(), row,
          out.data_ptr(), P, Hq, HEAD_DIM ** -0.5 if scale is None else float(scale),
          workspace.data_ptr() if n else None, n)
    return out


def kv_load_q8(k, v, lens, cache: QuantizedKVCache) -> None:
    """Positions [0, lens[b]) of every sequence from bf16 k, v [B, Hkv, S, 128]
    (last axis contiguous); lens is taken as at most S and Smax."""
    _check_cache(cache)
    _check_lens("lens", lens, cache)
    strides = []
    for name, t in (("k", k), ("v", v)):
        _require_device(name, t, cache.device)
        if t.dtype is not torch.bfloat16:
            raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
        if t.dim() != 4 or t.shape != (cache.B, cache.Hkv, k.shape[2], HEAD_DIM):
            raise ValueError(f"{name} must be [{cache.B}, {cache.Hkv}, S, {HEAD_DIM}], got {tuple(t.shape)}")
    if k.shape[2] == 0 or cache.B == 0:
        return
    # rows are loaded 16 bytes at a time
    k, v = (t if t.stride(3) == 1 and t.data_ptr() % 16 == 0 and all(s % 8 == 0 for s in t.stride()[:3])
            else _aligned(t) for t in (k, v))
    strides = [_I64x3(*t.stride()[:3]) for t in (k, v)]
    _call("dflash_kv8_load", cache.device, cache._ptr, k.data_ptr(), ctypes.addressof(strides[0]), v.data_ptr(),
          ctypes.addressof(strides[1]), lens.data_ptr(), k.shape[2])


def kv_read_q8(cache: QuantizedKVCache, lens, count: int, *, start=0):
    """(keys, values) bf16 [B, Hkv, count, 128] at positions start + i, as an
    attention at committed length lens[b] reads them; positions outside [0,
    lens[b]) are zero.  A length below one already written to is read after
    kv_rewind_q8, like any call at it.  start: an int, or int32 [B] on the device."""
    _check_cache(cache)
    _check_lens("lens", lens, cache)
    count = int(count)
    if count < 0:
        raise ValueError(f"count must not be negative, got {count}")
    starts = None
    if isinstance(start, torch.Tensor):
        _check_lens("start", start, cache)
        starts, start = start, 0
    elif not -2 ** 31 <= start < 2 ** 31:
        raise ValueError(f"start {start} is not a 32-bit position")
    k = torch.empty((cache.B, cache.Hkv, count, HEAD_DIM), dtype=torch.bfloat16, device=cache.device)
    v = torch.empty_like(k)
    _call("dflash_kv8_read", cache.device, cache._ptr, lens.data_ptr(), _lib.ptr(starts), int(start), count,
          k.data_ptr(), v.data_ptr())
    return k, v


def kv_rewind_q8(cache: QuantizedKVCache, length: int, written: int) -> int:
    """Make the tail ready for a call at committed length `length` of every sequence
    after positions up to `written` - 1 have been appended (rejected drafts
    included): what the call reads from the tail and later positions have
    overwritten comes back from the codes, rounded to bf16.  Returns what to pass as
    `written` next time, with the positions appended from here on.  Nothing is
    launched for the rewinds of a decode loop."""
    _check_cache(cache)
    length, written = int(length), int(written)
    if not 0 <= length <= cache.Smax or written < length:
        raise ValueError(f"need 0 <= length <= {cache.Smax} and written >= length, got {length} and {written}")
    blk, rest = divmod(length, BLOCK)

    def intact(x):
        # no later position has taken block x's slots, nor did a prompt or a load end where the
        # block after it does, which keeps that one alone
        return x < 0 or written < x * BLOCK + SLOTS

    def refill(x):
        # as read at a length past it: from its codes, which it got before its slots were taken
        lens = torch.full((cache.B,), (x + 2) * BLOCK + BLOCK // 2, dtype=torch.int32, device=cache.device)
        k, v = kv_read_q8(cache, lens, BLOCK, start=x * BLOCK)
        s = x * BLOCK % SLOTS
        cache.tail_k[:, :, s:s + BLOCK] = k
        cache.tail_vt[:, :, :, s:s + BLOCK] = v.transpose(2, 3)

    if rest and not intact(blk):
        refill(blk)
    if intact(blk - 1):
        return length
    if rest <= MAX_DRAFT:  # the next append may quantise block blk - 1 again
        refill(blk - 1)
        return length
    return min(written, blk * BLOCK + SLOTS - 1)  # (block blk is there, block blk - 1 is not)
