"""What a request asks of the logits: penalties for repeated tokens, biases and
grammar masks.

A ``LogitsState`` holds the counts, biases and penalties of B sequences;
``process_logits`` applies them (and a mask) to the logits of draft blocks, and
``greedy_accept(logits, draft, state=, mask=)`` (runtime.py) takes the greedy
tokens of the processed logits without storing them.  A block's row i knows the
tokens counted so far and the block's drafts 0 .. i - 1, so a verify step over
T rows gives what T single steps would.  The formulas and the layout are in
include/dflash_logits.h.

Masks are bitmasks: int32 [B, N, ceil(V / 32)] (an axis of B or N may be
expanded), token v allowed where bit v % 32 of word v // 32 is set.

Every op runs hand-written gfx950 kernels on torch's current stream of its
tensors' device; there is no CPU path.
"""
from __future__ import annotations

import ctypes

import torch

from . import _lib
from .gated_delta import _require_device
from .kv8 import _call

MAX_BIAS = 4096  # biases of one set_bias call
MAX_DRAFT = 64   # draft tokens that are counted for a sequence's rows

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


class _CState(ctypes.Structure):
    """dflash_logits_state of include/dflash_logits.h."""

    _fields_ = [(n, ctypes.c_void_p) for n in ("counts", "known", "bias", "penalties")] + [
        (n, ctypes.c_int32) for n in ("B", "V")]


class LogitsState:
    """Counts, biases and penalties of B sequences over V tokens, in caller-owned
    contiguous tensors on one device (``zeros`` makes them):

    counts int32 [B, V]: how often a token was generated, the sign bit set for
    tokens of the prompt; known int32 [B, ceil(V / 32)]: a bit for every token
    that has a count or a bias; bias fp32 [B, V]; penalties fp32 [B, 3]:
    repetition (> 0), presence, frequency.  ``state[b]`` and ``state[b0:b1]``
    are views of some sequences, e.g. to begin a request in one slot of a batch."""

    __slots__ = ("counts", "known", "bias", "penalties", "B", "V", "device", "_struct", "_ptr")

    def __init__(self, counts, known, bias, penalties):
        _require_device("counts", counts)
        if counts.dim() != 2 or counts.shape[1] == 0:
            raise ValueError(f"counts must be [B, V], got {tuple(counts.shape)}")
        B, V = counts.shape
        for name, t, shape, dtype in (("counts", counts, (B, V), torch.int32),
                                      ("known", known, (B, -(-V // 32)), torch.int32),
                                      ("bias", bias, (B, V), torch.float32),
                                      ("penalties", penalties, (B, 3), torch.float32)):
            _require_device(name, t, counts.device)
            if t.dtype is not dtype:
                raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
            if tuple(t.shape) != shape or not t.is_contiguous():
                raise ValueError(f"{name} must be contiguous {list(shape)}, got {list(t.shape)}")
        if B > 65535:
            raise ValueError(f"at most 65535 sequences, got {B}")
        self.counts, self.known, self.bias, self.penalties = counts, known, bias, penalties
        self.B, self.V, self.device = B, V, counts.device
        self._struct = _CState(counts.data_ptr(), known.data_ptr(), bias.data_ptr(), penalties.data_ptr(), B, V)
        self._ptr = ctypes.addressof(self._struct)

    @classmethod
    def zeros(cls, B: int, V: int, device) -> "LogitsState":
        """Nothing counted, no bias, no penalty."""
        if B < 0 or V <= 0:
            raise ValueError(f"need B >= 0 and V > 0, got {B} and {V}")
        z = lambda dt, *s: torch.zeros(*s, dtype=dt, device=device)  # noqa: E731
        penalties = z(torch.float32, B, 3)
        penalties[:, 0].fill_(1.0)
        return cls(z(torch.int32, B, V), z(torch.int32, B, -(-V // 32)), z(torch.float32, B, V), penalties)

    def __getitem__(self, rows) -> "LogitsState":
        if isinstance(rows, slice):
            if rows.step not in (None, 1):
                raise ValueError("a view takes neighbouring sequences")
        else:
            b = int(rows)
            if not -self.B <= b < self.B:
                raise IndexError(f"sequence {b} of {self.B}")
            b %= self.B
            rows = slice(b, b + 1)
        return LogitsState(self.counts[rows], self.known[rows], self.bias[rows], self.penalties[rows])

    def __repr__(self):
        return f"LogitsState(B={self.B}, V={self.V}, {self.device})"

    def reset(self) -> None:
        """Begin anew: nothing counted, no bias, no penalty.  Writes the known
        entries only."""
        _call("dflash_logits_state_reset", self.device, self._ptr)

    def set_penalties(self, repetition=1.0, presence=0.0, frequency=0.0) -> None:
        """Numbers, or a tensor or list of one a sequence.  Repetition penalties are positive (not
        looked at in a tensor on the device)."""
        for j, (name, p) in enumerate((("repetition", repetition), ("presence", presence), ("frequency", frequency))):
            if not isinstance(p, torch.Tensor):
                p = torch.tensor(p, dtype=torch.float32)
            if j == 0 and p.device.type == "cpu" and not bool((p > 0).all()):
                raise ValueError(f"the repetition penalty must be positive, got {repetition}")
            if p.dim() and tuple(p.shape) != (self.B,):
                raise ValueError(f"{name} must be a number or [{self.B}], got {tuple(p.shape)}")
            self.penalties[:, j].copy_(p)

    def set_bias(self, ids, values) -> None:
        """bias[b, ids[b, j]] = values[b, j], beside the biases that are there (of an
        id given twice the last counts; ids outside [0, V) are passed over).  ids int32
        [B, n] or [n], values fp32 of the same shape, n <= 4096; on the device or the
        host."""
        ids, values = self._rows("ids", ids, torch.int32), self._rows("values", values, torch.float32)
        if ids.shape != values.shape:
            raise ValueError(f"ids and values must be of one shape, got {tuple(ids.shape)}, {tuple(values.shape)}")
        if ids.shape[1] > MAX_BIAS:
            raise ValueError(f"at most {MAX_BIAS} biases a call, got {ids.shape[1]}")
        if ids.numel():
            _call("dflash_logits_state_set_bias", self.device, self._ptr, ids.data_ptr(), ids.stride(0),
                  values.data_ptr(), values.stride(0), ids.shape[1])

    def add(self, tokens, lens=None, *, prompt: bool = False) -> None:
        """Count tokens int32 [B, n] (or [n]; device or host), of sequence b the first
        lens[b] (int32 [B] on the device; all by default); ids outside [0, V) are passed
        over.  prompt: they are the prompt's, which the repetition penalty alone looks
        at.  After a verify step: add(posterior, matched + 1)."""
        tokens = self._rows("tokens", tokens, torch.int32)
        if lens is not None:
            _require_device("lens", lens, self.device)
            if lens.dtype is not torch.int32 or lens.shape != (self.B,) or not lens.is_contiguous():
                raise ValueError(f"lens must be contiguous int32 [{self.B}], got {lens.dtype} {tuple(lens.shape)}")
        if tokens.numel():
            _call("dflash_logits_state_add", self.device, self._ptr, tokens.data_ptr(), tokens.stride(0),
                  tokens.shape[1], _lib.ptr(lens), int(bool(prompt)))

    def _rows(self, name: str, t, dtype) -> torch.Tensor:
        """t as [B, n] of dtype on the device, rows contiguous."""
        if not isinstance(t, torch.Tensor):
            t = torch.tensor(t)
        if t.is_floating_point() and not dtype.is_floating_point and t.numel():
            raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
        if t.dim() == 1:
            t = t.expand(self.B, -1)
        if t.dim() != 2 or t.shape[0] != self.B:
            raise ValueError(f"{name} must be [{self.B}, n] or [n], got {tuple(t.shape)}")
        if t.device.type != "cpu":
            _require_device(name, t, self.device)
        if dtype is torch.int32 and t.dtype is not dtype:  # ids that 32 bits would wrap stay outside
            t = t.long().clamp(-1, self.V)
        t = t.to(device=self.device, dtype=dtype)
        return t if t.shape[1] < 2 or t.stride(1) == 1 else t.contiguous()


def check_mask(mask, B: int, N: int, V: int, dev):
    """(pointer, batch stride, row stride) of a bitmask [B, N, ceil(V / 32)]."""
    W = -(-V // 32)
    _require_device("mask", mask, dev)
    if mask.dtype is not torch.int32:
        raise TypeError(f"mask must be int32 words, got {mask.dtype}")
    if mask.dim() == 2:
        mask = mask.unsqueeze(0)
    if tuple(mask.shape) != (B, N, W):
        raise ValueError(f"mask must be [{B}, {N}, {W}], got {tuple(mask.shape)}")
    if W > 1 and mask.stride(2) != 1:
        raise ValueError("a mask's words must be contiguous")
    return mask.data_ptr(), mask.stride(0), mask.stride(1)


def check_state(state, B: int, V: int, dev) -> int | None:
    if state is None:
        return None
    if not isinstance(state, LogitsState):
        raise TypeError(f"state must be a LogitsState, got {type(state).__name__}")
    if state.B != B or state.V != V or state.device != dev:
        raise ValueError(f"logits of {B} sequences and {V} tokens on {dev}, but {state}")
    return state._ptr


def check_draft(draft, B: int, N: int, dev, counted: bool):
    """int32 [B, n] on the device with contiguous rows, or None."""
    if draft is None:
        return None
    if isinstance(draft, torch.Tensor):
        _require_device("draft", draft, dev)
        if draft.dtype is torch.int64:  # ids that 32 bits would wrap stay outside the vocabulary
            draft = draft.clamp(-1, 2 ** 31 - 1)
        draft = draft.to(torch.int32)
    else:
        draft = torch.tensor(draft, dtype=torch.int32).to(dev)
    if draft.dim() == 1:
        draft = draft.unsqueeze(0)
    if draft.dim() != 2 or draft.shape[0] != B:
        raise ValueError(f"draft must be [{B}, n], got {tuple(draft.shape)}")
    if counted and min(draft.shape[1], N - 1) > MAX_DRAFT:
        raise ValueError(f"at most {MAX_DRAFT} drafts are counted, got {draft.shape[1]} for {N} rows")
    return draft if draft.stride(-1) == 1 or draft.shape[1] < 2 else draft.contiguous()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """The two tensors' address ranges meet."""
    (a0, a1), (b0, b1) = ((t.data_ptr(), t.data_ptr() + t.element_size() * (
        1 + sum((n - 1) * s for n, s in zip(t.shape, t.stride())))) for t in (a, b))
    return a.numel() > 0 and b.numel() > 0 and a0 < b1 and b0 < a1


def process_logits(logits: torch.Tensor, state: LogitsState | None = None, draft=None, *, mask=None,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Logits [B, N, V] (or [N, V], B = 1; fp32, bf16 or fp16) under the state's
    penalties and biases and the mask, computed in fp32 and rounded once to their type.

    draft: [B, n] token ids, draft i known to the rows from i + 1 on (the block's tokens
    after its first, which is counted already).  mask: int32 words [B, N, ceil(V / 32)],
    or [N, ceil(V / 32)] for B = 1.  out: a tensor like the logits, or the logits
    themselves: then the entries that nothing changes keep their values, and eights of a
    row without a masked or known token are not touched."""
    _require_device("logits", logits, None)
    if logits.dtype not in _FLOATS:
        raise TypeError(f"logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if logits.dim() not in (2, 3):
        raise ValueError(f"logits must be [B, N, V] or [N, V], got {tuple(logits.shape)}")
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=logits.device)
    elif out is not logits:
        _require_device("out", out, logits.device)
        if out.dtype is not logits.dtype or out.shape != logits.shape:
            raise ValueError(f"out must be {logits.dtype} {list(logits.shape)}, got {out.dtype} {list(out.shape)}")
        if (out.data_ptr() != logits.data_ptr() or out.stride() != logits.stride()) and _overlap(out, logits):
            raise ValueError("out must be the logits themselves or lie apart from them")
    lg, res = (t.unsqueeze(0) if t.dim() == 2 else t for t in (logits, out))
    B, N, V = lg.shape
    dev = lg.device
    if lg.numel() == 0:
        return out
    if V > 1 and res.stride(2) != 1:
        raise ValueError("out's rows must be contiguous")
    (s0, n0), (s1, n1) = sorted((s, n) for s, n in ((res.stride(0), B), (res.stride(1), N)))
    if (n0 > 1 and s0 < V) or (n1 > 1 and s1 < (s0 * (n0 - 1) if n0 > 1 else 0) + V):
        raise ValueError(f"out's rows overlap, strides {tuple(res.stride())}")
    if V > 1 and lg.stride(2) != 1:
        lg = lg.contiguous()
    sp = check_state(state, B, V, dev)
    d = check_draft(draft, B, N, dev, state is not None)
    mp, mb, mr = check_mask(mask, B, N, V, dev) if mask is not None else (None, 0, 0)
    _call("dflash_logits_process", dev, lg.data_ptr(), _lib.dtype_tag(lg.dtype), lg.stride(0), lg.stride(1), sp,
          _lib.ptr(d), d.stride(0) if d is not None else 0, d.shape[1] if d is not None else 0, mp, mb, mr,
          res.data_ptr(), res.stride(0), res.stride(1), B, N, V)
    return out
