"""Projections in 8-bit integers.

A verify step streams the target's weights once for a few rows, and a prompt pass
is matrix products: weights in 8 bits halve the first's bytes and double the rate
of the matrix unit in the second.  Weights are quantised once per output channel
(``quantize_weight_i8``, or ``pack_weight_i8`` of codes from elsewhere), rows per
token as they come: ``linear_i8`` quantises and multiplies, ``quantize_rows_i8``
and ``matmul_i8`` are its two halves.  Sums of codes are exact 32-bit integers;
they are scaled in fp32 and rounded once.  Formats and formulas are in
include/dflash_int8.h.

Every op runs hand-written gfx950 kernels on torch's current stream of its
tensors' device; there is no CPU path.
"""
from __future__ import annotations

import torch

from . import _lib
from .gated_delta import _require_device
from .kv8 import _call
from .logits import _overlap

MAX_K = 131072  # features: the sum of products of codes stays in 32 bits

_OUT = {torch.float32: _lib.DFLASH_DTYPE_F32, torch.bfloat16: _lib.DFLASH_DTYPE_BF16,
        torch.float16: _lib.DFLASH_DTYPE_F16}
_IN = {torch.bfloat16: _lib.DFLASH_DTYPE_BF16, torch.float16: _lib.DFLASH_DTYPE_F16}


class Int8Weight:
    """A packed weight of N output channels and K features (quantize_weight_i8 and
    pack_weight_i8 make it): codes as the matrix unit's fragments, one fp32 scale a
    channel.  gated: the weight is [gate; up] and the products are silu(gate) * up."""

    __slots__ = ("codes", "scales", "N", "K", "gated", "cols", "device", "_codes_ptr", "_scales_ptr", "_gated", "_ws_bytes")

    def __init__(self, codes, scales, N: int, K: int, gated: bool):
        lib = _lib.load()
        _require_device("codes", codes)
        _require_device("scales", scales, codes.device)
        nbytes = int(lib.dflash_weight_i8_bytes(N, K, int(gated)))
        if nbytes == 0:
            raise ValueError(f"no packed weight of {N} channels and {K} features{' (gated)' if gated else ''}")
        if codes.dtype is not torch.int8 or not codes.is_contiguous() or codes.numel() != nbytes:
            raise ValueError(f"codes must be contiguous int8 [{nbytes}], got {codes.dtype} {list(codes.shape)}")
        n = int(lib.dflash_weight_i8_scales(N, int(gated)))
        if scales.dtype is not torch.float32 or not scales.is_contiguous() or scales.numel() != n:
            raise ValueError(f"scales must be contiguous float32 [{n}], got {scales.dtype} {list(scales.shape)}")
        self.codes, self.scales, self.N, self.K, self.gated = codes, scales, int(N), int(K), bool(gated)
        self.cols = self.N // 2 if self.gated else self.N
        self.device = codes.device
        self._codes_ptr, self._scales_ptr, self._gated = codes.data_ptr(), scales.data_ptr(), int(self.gated)
        self._ws_bytes = {}  # by entry point and rows

    def __repr__(self):
        return f"Int8Weight(N={self.N}, K={self.K}, gated={self.gated}, {self.device})"


def _matrix(name: str, t, dtypes) -> None:
    _require_device(name, t)
    if t.dtype not in dtypes:
        raise TypeError(f"{name} must be {' or '.join(str(d) for d in dtypes)}, got {t.dtype}")
    if t.dim() != 2:
        raise ValueError(f"{name} must be a matrix, got {tuple(t.shape)}")


def pack_weight_i8(codes: torch.Tensor, scale: torch.Tensor, *, gated: bool = False) -> Int8Weight:
    """int8 codes [N, K] and fp32 scales [N] as a packed weight.  gated: the rows are [gate; up].
    Codes of the largest K are at least -127: a sum of -128 * -128 would leave 32 bits."""
    _matrix("codes", codes, (torch.int8,))
    N, K = codes.shape
    dev = codes.device
    _require_device("scale", scale, dev)
    if scale.dtype is not torch.float32 or scale.shape != (N,):
        raise ValueError(f"scale must be float32 [{N}], got {scale.dtype} {tuple(scale.shape)}")
    lib = _lib.load()
    nbytes = int(lib.dflash_weight_i8_bytes(N, K, int(gated)))
    if nbytes == 0:
        raise ValueError(f"a weight of {N} channels and {K} features cannot be packed (at most {MAX_K} features, "
                         "an even number of channels if gated)")
    if K > 1 and codes.stride(1) != 1 or N > 1 and codes.stride(0) < K:
        codes = codes.contiguous()
    if K == MAX_K and bool((codes == -128).any()):
        raise ValueError(f"codes of {K} features must be at least -127")
    scale = scale.contiguous()
    packed = torch.empty(nbytes, dtype=torch.int8, device=dev)
    scales = torch.empty(int(lib.dflash_weight_i8_scales(N, int(gated))), dtype=torch.float32, device=dev)
    _call("dflash_weight_pack_i8", dev, codes.data_ptr(), codes.stride(0), scale.data_ptr(), packed.data_ptr(),
          scales.data_ptr(), N, K, int(bool(gated)))
    return Int8Weight(packed, scales, N, K, gated)


def quantize_weight_i8(weight: torch.Tensor, *, gated: bool = False) -> Int8Weight:
    """A bf16 or fp16 weight [N, K] quantised by channel and packed; made once at load time."""
    codes, scale = quantize_rows_i8(weight)
    return pack_weight_i8(codes, scale, gated=gated)


def _rows_of(x: torch.Tensor):
    """x [..., K] as rows [M, K] whose last axis is contiguous."""
    if x.dim() != 2:
        x = x.reshape(-1, x.shape[-1])
    if x.shape[1] > 1 and x.stride(1) != 1 or x.stride(0) < 0:
        x = x.contiguous()
    return x


def quantize_rows_i8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes int8 [..., K], scales fp32 [...]) of the rows of x (bf16 or fp16 [..., K]):
    a = max(max |x|, 2^-100), scale a / 127, code rint(127 x / a).  A row that holds a
    NaN or an infinity has scale NaN.  The codes' rows lie a multiple of 16 bytes apart."""
    _require_device("x", x)
    if x.dtype not in _IN:
        raise TypeError(f"x must be bfloat16 or float16, got {x.dtype}")
    if x.dim() == 0 or not 1 <= x.shape[-1] <= MAX_K:
        raise ValueError(f"x must be [..., K] with 1 to {MAX_K} features, got {tuple(x.shape)}")
    lead, K = x.shape[:-1], x.shape[-1]
    rows = _rows_of(x)
    M, dev = rows.shape[0], x.device
    Kp = -(-K // 16) * 16
    codes = torch.empty((M, Kp), dtype=torch.int8, device=dev)
    scale = torch.empty(lead, dtype=torch.float32, device=dev)
    if M:
        _call("dflash_quantize_rows_i8", dev, rows.data_ptr(), _IN[x.dtype], rows.stride(0), codes.data_ptr(), Kp,
              scale.data_ptr(), M, K)
    codes = codes.view(*lead, Kp)
    return (codes if Kp == K else codes[..., :K]), scale


def _workspace_bytes(fn: str, M: int, weight: Int8Weight) -> int:
    """The entry point's workspace for M rows (on the weight's device)."""
    n = weight._ws_bytes.get((fn, M))
    if n is None:
        with torch.cuda.device(weight.device):
            n = int(getattr(_lib.load(), fn)(M, weight.N, weight.K, weight._gated))
        if len(weight._ws_bytes) < 4096:
            weight._ws_bytes[(fn, M)] = n
    return n


def _output(out, out_dtype, lead, weight):
    """(the output tensor, its rows' stride)."""
    if out is None:
        if out_dtype not in _OUT:
            raise TypeError(f"out_dtype must be bfloat16, float16 or float32, got {out_dtype}")
        out = torch.empty((*lead, weight.cols), dtype=out_dtype, device=weight.device)
        return out, weight.cols
    _require_device("out", out, weight.device)
    if out.dtype not in _OUT:
        raise TypeError(f"out must be bfloat16, float16 or float32, got {out.dtype}")
    if tuple(out.shape) != (*lead, weight.cols):
        raise ValueError(f"out must be {[*lead, weight.cols]}, got {list(out.shape)}")
    if out.numel() == 0:
        return out, weight.cols
    if out.dim() == 1:
        rows = out.unsqueeze(0)
    else:
        try:
            rows = out.view(-1, weight.cols)
        except RuntimeError:
            raise ValueError("out's rows must be evenly spaced") from None
    if weight.cols > 1 and rows.stride(1) != 1 or rows.shape[0] > 1 and rows.stride(0) < weight.cols:
        raise ValueError(f"out's rows must be contiguous and apart, got strides {tuple(out.stride())}")
    return out, max(rows.stride(0), weight.cols)


def _check_apart(out, name: str, x) -> None:
    """Workgroups read x while others store."""
    if out.untyped_storage().data_ptr() == x.untyped_storage().data_ptr() and _overlap(out, x):
        raise ValueError(f"out must lie apart from {name}")


def _check_weight(weight, K: int, dev) -> None:
    if not isinstance(weight, Int8Weight):
        raise TypeError(f"weight must be an Int8Weight, got {type(weight).__name__}")
    if weight.K != K or weight.device != dev:
        raise ValueError(f"rows of {K} features on {dev}, but {weight}")


def matmul_i8(codes: torch.Tensor, scale: torch.Tensor, weight: Int8Weight, *, out_dtype: torch.dtype = torch.bfloat16,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """(codes @ weight codes^T) * scale * weight scales, [..., N] (gated: silu(gate) * up,
    [..., N / 2]) in out_dtype, or into out (whose type counts, and which lies apart from codes).

    codes: int8 [..., K], scale: fp32 [...], as quantize_rows_i8 gives them."""
    _require_device("codes", codes)
    if codes.dtype is not torch.int8:
        raise TypeError(f"codes must be int8, got {codes.dtype}")
    if codes.dim() == 0:
        raise ValueError("codes must be [..., K]")
    lead, K, dev = codes.shape[:-1], codes.shape[-1], codes.device
    _check_weight(weight, K, dev)
    _require_device("scale", scale, dev)
    if scale.dtype is not torch.float32 or scale.shape != lead:
        raise ValueError(f"scale must be float32 {list(lead)}, got {scale.dtype} {list(scale.shape)}")
    given = out is not None
    out, os = _output(out, out_dtype, lead, weight)
    if out.numel() == 0:
        return out
    if given:
        _check_apart(out, "codes", codes)
        _check_apart(out, "scale", scale)
    rows, Kp = _rows_of(codes), -(-K // 16) * 16
    M = rows.shape[0]
    # rows are read 16 bytes at a time, up to K rounded up to 16
    fits = rows.storage_offset() + (M - 1) * rows.stride(0) + Kp <= rows.untyped_storage().nbytes()
    s = rows.stride(0)
    if not fits or rows.data_ptr() % 16 or M > 1 and (s % 16 or not Kp <= s <= 1 << 23):
        rows = torch.nn.functional.pad(rows, (0, Kp - K)) if Kp > K else rows.clone(memory_format=torch.contiguous_format)
    scale = scale.contiguous()
    n = _workspace_bytes("dflash_gemm_i8_workspace_bytes", M, weight)
    ws = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _call("dflash_gemm_i8", dev, rows.data_ptr(), rows.stride(0) if M > 1 else Kp, scale.data_ptr(),
          weight._codes_ptr, weight._scales_ptr, out.data_ptr(), _OUT[out.dtype], os, M, weight.N, K, weight._gated,
          _lib.ptr(ws), n)
    return out


def linear_i8(x: torch.Tensor, weight: Int8Weight, *, out_dtype: torch.dtype | None = None,
              out: torch.Tensor | None = None) -> torch.Tensor:
    """x @ weight^T with x's rows quantised on the way: matmul_i8(*quantize_rows_i8(x), weight).

    x: bf16 or fp16 [..., K]; out_dtype: x's type by default; out lies apart from x."""
    _require_device("x", x)
    if x.dtype not in _IN:
        raise TypeError(f"x must be bfloat16 or float16, got {x.dtype}")
    if x.dim() == 0:
        raise ValueError("x must be [..., K]")
    lead, K, dev = x.shape[:-1], x.shape[-1], x.device
    _check_weight(weight, K, dev)
    given = out is not None
    out, os = _output(out, x.dtype if out_dtype is None else out_dtype, lead, weight)
    if out.numel() == 0:
        return out
    if given:
        _check_apart(out, "x", x)
    rows = _rows_of(x)
    M = rows.shape[0]
    n = _workspace_bytes("dflash_linear_i8_workspace_bytes", M, weight)
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    _call("dflash_linear_i8", dev, rows.data_ptr(), _IN[x.dtype], rows.stride(0), weight._codes_ptr, weight._scales_ptr,
          out.data_ptr(), _OUT[out.dtype], os, M, weight.N, K, weight._gated, ws.data_ptr(), n)
    return out
