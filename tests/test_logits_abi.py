"""Logits processing's C entry points and Python checks: declared, exported, bound,
and refusing bad arguments before any launch (no GPU: nothing here computes)."""
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


def _state(**kw):
    from dflash_mlx.logits import _CState

    f = dict(counts=P, known=P, bias=P, penalties=P, B=2, V=100)
    f.update(kw)
    return _CState(**f)


def _ptr(s):
    return ctypes.addressof(s) if s is not None else None


def _reset(lib, s):
    return lib.dflash_logits_state_reset(_ptr(s), None)


def _add(lib, s, tokens=P, stride=5, n=5, lens=None, prompt=0):
    return lib.dflash_logits_state_add(_ptr(s), tokens, stride, n, lens, prompt, None)


def _bias(lib, s, ids=P, values=P, n=5):
    return lib.dflash_logits_state_set_bias(_ptr(s), ids, 5, values, 5, n, None)


def _process(lib, s, logits=P, dtype=0, bs=400, rs=100, draft=P, n_draft=3, mask=P, out=2 * P, obs=400, ors=100, B=2,
             N=4, V=100):
    return lib.dflash_logits_process(logits, dtype, bs, rs, _ptr(s), draft, 3, n_draft, mask, 16, 4, out, obs, ors, B, N,
                                     V, None)


def _accept(lib, s, logits=P, dtype=0, draft=P, n_draft=3, mask=P, post=P, matched=P, bonus=P, B=2, N=4, V=100, ws=P,
            nbytes=1 << 30):
    return lib.dflash_greedy_accept_processed(logits, dtype, 400, 100, draft, 3, n_draft, _ptr(s), mask, 16, 4, post,
                                              matched, bonus, B, N, V, ws, nbytes, None)


def test_every_declared_entry_point_is_exported_and_bound(lib):
    from dflash_mlx import _lib

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "dflash_logits.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(dflash_[a-z0-9_]+)\s*\(", text))
    assert names == {"dflash_logits_state_reset", "dflash_logits_state_add", "dflash_logits_state_set_bias",
                     "dflash_logits_process", "dflash_greedy_accept_processed",
                     "dflash_greedy_accept_processed_workspace_bytes"}
    for name in names:
        assert hasattr(lib, name) and name in _lib.SIGNATURES


@pytest.mark.parametrize("call", [_reset, _add, _bias, _process, _accept])
def test_states_that_are_refused(lib, call):
    for field in ("counts", "known", "bias", "penalties"):
        assert call(lib, _state(**{field: None})) == NULL
        assert call(lib, _state(**{field: P + 2})) == ALIGN
    assert call(lib, _state(V=0)) == SHAPE
    assert call(lib, _state(B=-1)) == SHAPE
    assert call(lib, _state(B=65536)) == SHAPE


@pytest.mark.parametrize("call", [_reset, _add, _bias])
def test_a_missing_state_is_refused_and_an_empty_one_is_no_work(lib, call):
    assert call(lib, None) == NULL
    assert call(lib, _state(B=0, counts=None)) == 0


def test_tokens_and_biases_that_are_refused(lib):
    s = _state()
    assert _add(lib, s, n=-1) == SHAPE
    assert _add(lib, s, tokens=None) == NULL
    assert _add(lib, s, tokens=P + 1) == ALIGN
    assert _add(lib, s, lens=P + 2) == ALIGN
    assert _add(lib, s, tokens=None, n=0) == 0
    assert _bias(lib, s, n=-1) == SHAPE
    assert _bias(lib, s, n=4097) == SHAPE
    assert _bias(lib, s, ids=None) == NULL and _bias(lib, s, values=None) == NULL
    assert _bias(lib, s, ids=P + 2) == ALIGN and _bias(lib, s, values=P + 2) == ALIGN
    assert _bias(lib, s, ids=None, n=0) == 0


@pytest.mark.parametrize("call", [_process, _accept])
def test_logits_that_are_refused(lib, call):
    s = _state()
    for kw in (dict(B=-1), dict(N=0), dict(V=0), dict(n_draft=-1), dict(N=16385), dict(V=2 ** 31 - 1), dict(V=99), dict(B=3)):
        assert call(lib, s, **kw) == SHAPE
    assert call(lib, s, N=66, n_draft=65) == SHAPE
    assert call(lib, s, logits=None) == NULL and call(lib, s, draft=None) == NULL
    assert call(lib, s, dtype=3) == UNSUPPORTED
    assert call(lib, s, logits=P + 2) == ALIGN and call(lib, s, dtype=1, logits=P + 1) == ALIGN
    assert call(lib, s, mask=P + 2) == ALIGN and call(lib, s, draft=P + 2) == ALIGN
    assert call(lib, s, B=0, logits=None) == 0


def test_outputs_that_are_refused(lib):
    s = _state()
    assert _process(lib, s, out=None) == NULL
    assert _process(lib, s, out=2 * P + 2) == ALIGN
    assert _process(lib, s, out=P, ors=200) == SHAPE  # in place means the same strides
    assert _accept(lib, s, post=None, matched=None, bonus=None) == NULL
    assert _accept(lib, s, ws=None) == NULL
    assert _accept(lib, s, nbytes=8) == WORKSPACE
    assert _accept(lib, s, ws=P + 4) == ALIGN


def test_python_refuses_host_tensors():
    from dflash_mlx import LogitsState, greedy_accept, process_logits

    with pytest.raises(ValueError, match="no CPU path"):
        LogitsState.zeros(1, 10, "cpu")
    with pytest.raises(ValueError):
        LogitsState.zeros(1, 0, "cpu")
    with pytest.raises(ValueError, match="no CPU path"):
        process_logits(torch.zeros(1, 2, 10))
    with pytest.raises(ValueError, match="no CPU path"):
        greedy_accept(torch.zeros(1, 2, 10), mask=torch.zeros(1, 2, 1, dtype=torch.int32))


def test_overlap_of_address_ranges():
    from dflash_mlx.logits import _overlap

    x = torch.zeros(4, 10)
    assert _overlap(x, x[1:3]) and _overlap(x[:3], x[2:])
    assert not _overlap(x[:2], x[2:]) and not _overlap(x[:0], x)
