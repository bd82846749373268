"""The 8-bit cache's C entry points: declared, exported, bound, and refusing bad
arguments before any launch (no GPU: nothing here computes)."""
from __future__ import annotations

import ctypes
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


def _cache(**kw):
    from dflash_mlx.kv8 import _CCache

    f = dict(k_codes=P, v_codes=P, k_scale=P, v_scale=P, tail_k=P, tail_vt=P, type=0, B=2, Hkv=4, Smax=256)
    f.update(kw)
    return _CCache(**f)


def _append(lib, c, proj=P, stride=40 * 128, q_norm=P, k_norm=P, lens=P, q_out=P, T=4, Hq=16, rot=32, prompt=0):
    return lib.dflash_kv8_append(ctypes.addressof(c) if c is not None else None, proj, stride, q_norm, k_norm, lens,
                                 q_out, None, T, Hq, rot, 1e5, 1e-6, prompt, None)


def _verify(lib, c, q=P, lens=P, gate=P, stride=32 * 128, out=P, T=4, Hq=16, ws=P, nbytes=1 << 40):
    return lib.dflash_attn_verify_q8(ctypes.addressof(c), q, lens, gate, stride, out, T, Hq, 0.1, ws, nbytes, None)


def _prefill(lib, c, q=P, lens=P, gate=P, stride=32 * 128, out=P, T=40, Hq=16, ws=None, nbytes=0):
    return lib.dflash_attn_prefill_q8(ctypes.addressof(c), q, lens, gate, stride, out, T, Hq, 0.1, ws, nbytes, None)


def _read(lib, c, lens=P, count=5, k=P, v=P):
    return lib.dflash_kv8_read(ctypes.addressof(c), lens, None, 0, count, k, v, None)


def _load(lib, c, k=P, v=P, lens=P, S=100, ks=(1024, 256, 128), vs=(1024, 256, 128)):
    a, b = (ctypes.c_int64 * 3)(*ks), (ctypes.c_int64 * 3)(*vs)
    return lib.dflash_kv8_load(ctypes.addressof(c), k, ctypes.addressof(a), v, ctypes.addressof(b), lens, S, None)


def test_every_declared_entry_point_is_exported_and_bound(lib):
    from dflash_mlx import _lib

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "dflash_kv8.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(dflash_[a-z0-9_]+)\s*\(", text))
    assert names == {"dflash_kv8_append", "dflash_kv8_load", "dflash_kv8_read", "dflash_attn_verify_q8",
                     "dflash_attn_verify_q8_workspace_bytes", "dflash_attn_prefill_q8",
                     "dflash_attn_prefill_q8_workspace_bytes"}
    for name in names:
        assert hasattr(lib, name) and name in _lib.SIGNATURES


@pytest.mark.parametrize("call", [_append, _verify, _prefill, _read, _load])
def test_caches_that_are_refused(lib, call):
    for field in ("k_codes", "v_codes", "k_scale", "v_scale", "tail_k", "tail_vt"):
        assert call(lib, _cache(**{field: None})) == NULL
        assert call(lib, _cache(**{field: P + 8})) == ALIGN
    assert call(lib, _cache(type=2)) == UNSUPPORTED
    assert call(lib, _cache(type=-1)) == UNSUPPORTED
    for bad in (dict(Smax=0), dict(Smax=100), dict(Smax=-64), dict(Hkv=0), dict(B=-1), dict(B=1 << 30)):
        assert call(lib, _cache(**bad)) == SHAPE, bad
    # nothing to do, whatever the pointers
    assert call(lib, _cache(B=0, k_codes=None)) == 0


def test_append_refusals(lib):
    c = _cache()
    assert _append(lib, None) == NULL
    for name in ("proj", "q_norm", "k_norm", "lens", "q_out"):
        assert _append(lib, c, **{name: None}) == NULL, name
    assert _append(lib, c, T=17) == SHAPE           # more than a draft
    assert _append(lib, c, T=-1, prompt=1) == SHAPE
    assert _append(lib, c, T=2 ** 31 - 100, prompt=1) == SHAPE
    assert _append(lib, c, Hq=6) == SHAPE           # not a multiple of Hkv
    assert _append(lib, c, stride=40 * 128 - 8) == SHAPE
    assert _append(lib, c, rot=48) == UNSUPPORTED
    assert _append(lib, c, stride=40 * 128 + 4) == ALIGN
    assert _append(lib, c, proj=P + 8) == ALIGN
    assert _append(lib, c, T=0, proj=None) == 0


def test_verify_refusals(lib):
    c = _cache()
    for name in ("q", "lens", "gate", "out", "ws"):
        assert _verify(lib, c, **{name: None}) == NULL, name
    assert _verify(lib, c, T=17) == SHAPE
    assert _verify(lib, c, T=16, Hq=20) == SHAPE     # 80 rows a key/value head
    assert _verify(lib, c, Hq=18) == SHAPE
    assert _verify(lib, c, stride=32 * 128 - 4) == SHAPE
    assert _verify(lib, c, q=P + 8) == ALIGN
    assert _verify(lib, c, gate=P + 4) == ALIGN
    assert _verify(lib, c, out=P + 4) == ALIGN
    need = lib.dflash_attn_verify_q8_workspace_bytes(2, 4, 16, 4, 256)
    assert need > 0 and _verify(lib, c, nbytes=need - 1) == WORKSPACE
    assert _verify(lib, c, T=0) == 0
    for bad in ((0, 4, 16, 4, 256), (2, 0, 16, 4, 256), (2, 17, 16, 4, 256), (2, 4, 18, 4, 256), (2, 16, 20, 4, 256),
                (2, 4, 16, 4, 100)):
        assert lib.dflash_attn_verify_q8_workspace_bytes(*bad) == 0, bad


@pytest.mark.parametrize("B,Hkv,Smax", [(1, 4, 4096), (12, 1, 64), (300, 4, 1024), (256, 8, 64), (2000, 1, 8192)])
def test_verify_workspace_serves_smaller_calls(lib, B, Hkv, Smax):
    need = lib.dflash_attn_verify_q8_workspace_bytes
    sizes = {(T, rep): need(B, T, Hkv * rep, Hkv, Smax) for T in range(1, 17) for rep in (1, 2, 3, 4, 8, 16) if T * rep <= 64}
    for (T, rep), n in sizes.items():
        assert all(n >= m > 0 for (t, r), m in sizes.items() if t <= T and r <= rep), (T, rep)


def test_prefill_refusals(lib):
    c = _cache()
    for name in ("q", "lens", "gate", "out"):
        assert _prefill(lib, c, **{name: None}) == NULL, name
    assert _prefill(lib, c, T=-1) == SHAPE
    assert _prefill(lib, c, Hq=68, stride=136 * 128) == SHAPE  # 17 query heads a key/value head
    assert _prefill(lib, c, stride=32 * 128 - 8) == SHAPE
    assert _prefill(lib, c, stride=32 * 128 + 4) == ALIGN
    assert _prefill(lib, c, gate=P + 8) == ALIGN
    assert _prefill(lib, _cache(B=65536)) == SHAPE
    assert _prefill(lib, c, T=0) == 0


def test_prefill_workspace(lib):
    need = lib.dflash_attn_prefill_q8_workspace_bytes
    # one row block of four head groups over 32 turns of keys: split; a device's worth of row blocks: not
    n = need(1, 40, 16, 4, 4096)
    assert n > 0 and n % (40 * 16 * 129 * 4) == 0
    assert need(1, 100000, 16, 4, 4096) == 0 and need(64, 200, 16, 4, 4096) == 0
    assert need(1, 40, 16, 4, 256) == 0  # too few turns
    for bad in ((0, 40, 16, 4, 4096), (1, 0, 16, 4, 4096), (1, 40, 16, 0, 4096), (1, 40, 15, 4, 4096), (1, 40, 68, 4, 4096),
                (1, 40, 16, 4, 100), (1, 40, 16, 4, 0), (1, 40, 0, 4, 4096)):
        assert need(*bad) == 0, bad
    c = _cache(B=1, Smax=4096)
    assert _prefill(lib, c, ws=P, nbytes=n - 1) == WORKSPACE
    assert _prefill(lib, c, ws=P + 8, nbytes=n) == ALIGN


def test_read_and_load_refusals(lib):
    c = _cache()
    assert _read(lib, c, lens=None) == NULL
    assert _read(lib, c, k=None, v=None) == NULL
    assert _read(lib, c, count=-1) == SHAPE
    assert _read(lib, c, k=P + 8) == ALIGN
    assert _read(lib, c, count=0) == 0
    for name in ("k", "v", "lens"):
        assert _load(lib, c, **{name: None}) == NULL, name
    assert _load(lib, c, S=-1) == SHAPE
    assert _load(lib, c, ks=(1024, -256, 128)) == SHAPE
    assert _load(lib, c, vs=(1024, 256, 132)) == ALIGN
    assert _load(lib, c, v=P + 8) == ALIGN
    assert _load(lib, c, S=0) == 0


def test_python_refuses_cpu_tensors_and_bad_caches():
    import dflash_mlx as dm

    z = lambda dt, *s: torch.zeros(*s, dtype=dt)  # noqa: E731
    with pytest.raises(ValueError, match="no CPU path"):
        dm.QuantizedKVCache(z(torch.int8, 1, 1, 64, 128), z(torch.int8, 1, 1, 1, 128, 64), z(torch.float32, 1, 1, 1),
                            z(torch.float32, 1, 1, 1), z(torch.bfloat16, 1, 1, 128, 128), z(torch.bfloat16, 1, 1, 128, 128))
    with pytest.raises(TypeError, match="int8 or float8_e4m3fn"):
        dm.QuantizedKVCache.zeros(1, 1, 64, torch.bfloat16, "cpu")
    with pytest.raises(ValueError, match="multiple of 64"):
        dm.QuantizedKVCache.zeros(1, 1, 100, torch.int8, "cpu")
    with pytest.raises(TypeError, match="QuantizedKVCache"):
        dm.kv_read_q8(object(), None, 1)
