"""The 8-bit projections' C entry points and Python checks: declared, exported, bound,
and refusing bad arguments before any launch (no GPU: nothing here computes)."""
from __future__ import annotations

import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent
NULL, SHAPE, UNSUPPORTED, ALIGN, WORKSPACE = -1, -2, -3, -4, -5
P = 0x1000  # stands for a device pointer: no call below gets as far as a launch


@pytest.fixture(scope="module")
def lib():
    from dflash_mlx import _lib

    return _lib.load()


def _pack(lib, codes=P, rs=200, scale=P, packed=P, packed_scale=P, N=64, K=200, gated=0):
    return lib.dflash_weight_pack_i8(codes, rs, scale, packed, packed_scale, N, K, gated, None)


def _quantize(lib, x=P, dtype=1, xs=200, codes=P, cs=208, scale=P, M=4, K=200):
    return lib.dflash_quantize_rows_i8(x, dtype, xs, codes, cs, scale, M, K, None)


def _gemm(lib, x=P, xs=208, sx=P, w=P, sw=P, out=P, dtype=1, os=64, M=4, N=64, K=200, gated=0, ws=P, nbytes=1 << 40):
    return lib.dflash_gemm_i8(x, xs, sx, w, sw, out, dtype, os, M, N, K, gated, ws, nbytes, None)


def test_every_declared_entry_point_is_exported_and_bound(lib):
    from dflash_mlx import _lib

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "dflash_int8.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(dflash_[a-z0-9_]+)\s*\(", text))
    assert names == {"dflash_weight_i8_bytes", "dflash_weight_i8_scales", "dflash_weight_pack_i8",
                     "dflash_quantize_rows_i8", "dflash_gemm_i8", "dflash_gemm_i8_workspace_bytes",
                     "dflash_linear_i8", "dflash_linear_i8_workspace_bytes", "dflash_add_rmsnorm_i8"}
    for name in names:
        assert hasattr(lib, name) and name in _lib.SIGNATURES


def test_sizes_of_packed_weights(lib):
    assert lib.dflash_weight_i8_bytes(1, 1, 0) == 2 * 1024
    assert lib.dflash_weight_i8_bytes(33, 129, 0) == 3 * 4 * 1024
    assert lib.dflash_weight_i8_bytes(34, 128, 1) == 2 * 2 * 2 * 1024
    assert lib.dflash_weight_i8_scales(33, 0) == 48 and lib.dflash_weight_i8_scales(34, 1) == 64
    for N, K, gated in ((0, 1, 0), (1, 0, 0), (1, 131073, 0), (3, 64, 1), (-2, 64, 1), (2 ** 28 + 1, 1, 0)):
        assert lib.dflash_weight_i8_bytes(N, K, gated) == 0
    assert lib.dflash_weight_i8_scales(3, 1) == 0


@pytest.mark.parametrize("call", [_pack, _gemm])
def test_weights_that_are_refused(lib, call):
    for kw in (dict(N=0), dict(K=0), dict(K=131073), dict(N=63, gated=1)):
        assert call(lib, **kw) == SHAPE


def test_packing_that_is_refused(lib):
    assert _pack(lib, rs=199) == SHAPE
    for name in ("codes", "scale", "packed", "packed_scale"):
        assert _pack(lib, **{name: None}) == NULL
    for name, p in (("scale", P + 2), ("packed", P + 8), ("packed_scale", P + 8)):
        assert _pack(lib, **{name: p}) == ALIGN


def test_rows_that_are_refused(lib):
    for kw in (dict(M=-1), dict(K=0), dict(K=131073), dict(xs=-1), dict(cs=192)):
        assert _quantize(lib, **kw) == SHAPE
    for name in ("x", "codes", "scale"):
        assert _quantize(lib, **{name: None}) == NULL
    assert _quantize(lib, dtype=0) == UNSUPPORTED
    for kw in (dict(x=P + 1), dict(codes=P + 8), dict(cs=209), dict(scale=P + 2)):
        assert _quantize(lib, **kw) == ALIGN
    assert _quantize(lib, M=0, x=None) == 0


def test_products_that_are_refused(lib):
    for kw in (dict(M=-1), dict(xs=192), dict(os=63), dict(xs=2 ** 23 + 16), dict(os=2 ** 26 + 1)):
        assert _gemm(lib, **kw) == SHAPE
    for name in ("x", "sx", "w", "sw", "out"):
        assert _gemm(lib, **{name: None}) == NULL
    assert _gemm(lib, dtype=3) == UNSUPPORTED
    for kw in (dict(x=P + 8), dict(xs=216), dict(sx=P + 2), dict(w=P + 8), dict(sw=P + 8), dict(out=P + 1),
               dict(out=P + 2, dtype=0)):
        assert _gemm(lib, **kw) == ALIGN
    assert _gemm(lib, M=0, x=None) == 0


def _linear(lib, x=P, xd=1, xs=200, w=P, sw=P, out=P, dtype=1, os=64, M=4, N=64, K=200, gated=0, ws=P, nbytes=1 << 40):
    return lib.dflash_linear_i8(x, xd, xs, w, sw, out, dtype, os, M, N, K, gated, ws, nbytes, None)


def test_linears_that_are_refused(lib):
    for kw in (dict(M=-1), dict(xs=-1), dict(os=63), dict(N=0), dict(K=131073), dict(N=63, gated=1), dict(os=1 << 27)):
        assert _linear(lib, **kw) == SHAPE
    for name in ("x", "w", "sw", "out", "ws"):
        assert _linear(lib, **{name: None}) == NULL
    assert _linear(lib, dtype=3) == UNSUPPORTED and _linear(lib, xd=0) == UNSUPPORTED
    for kw in (dict(x=P + 1), dict(w=P + 8), dict(sw=P + 8), dict(out=P + 1), dict(out=P + 2, dtype=0), dict(ws=P + 8)):
        assert _linear(lib, **kw) == ALIGN
    assert _linear(lib, nbytes=4 * 208 + 15) == WORKSPACE
    assert _linear(lib, M=0, x=None) == 0
    assert lib.dflash_linear_i8_workspace_bytes(4, 64, 200, 0) == 4 * 208 + 16
    assert lib.dflash_linear_i8_workspace_bytes(0, 64, 200, 0) == 0


def _norm(lib, h=P, r=P, w=P, out=P, cap=P, cap_stride=256, codes=P, cs=256, scale=P, M=4, H=256):
    return lib.dflash_add_rmsnorm_i8(h, r, w, out, cap, cap_stride, codes, cs, scale, M, H, 1e-6, None)


def test_norms_that_are_refused(lib):
    for kw in (dict(M=-1), dict(H=0), dict(H=8), dict(H=32784), dict(cs=240), dict(cap_stride=248)):
        assert _norm(lib, **kw) == SHAPE
    for name in ("h", "w", "out", "codes", "scale"):
        assert _norm(lib, **{name: None}) == NULL
    for name in ("h", "r", "w", "out", "cap", "codes"):
        assert _norm(lib, **{name: P + 8}) == ALIGN
    for kw in (dict(cs=264), dict(cap_stride=260), dict(scale=P + 2)):
        assert _norm(lib, **kw) == ALIGN
    assert _norm(lib, M=0, h=None) == 0


def test_python_refuses_host_tensors():
    from dflash_mlx import linear_i8, matmul_i8, pack_weight_i8, quantize_rows_i8, quantize_weight_i8

    x, c = torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 64, dtype=torch.int8)
    for bad in (lambda: quantize_rows_i8(x), lambda: quantize_weight_i8(x), lambda: linear_i8(x, None),
                lambda: pack_weight_i8(c, torch.ones(2)), lambda: matmul_i8(c, torch.ones(2), None)):
        with pytest.raises(ValueError, match="no CPU path"):
            bad()
