"""The LM head's fp32 logits: C entry points declared, exported, bound, and refusing bad
arguments before any launch (no GPU: nothing here computes)."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

from dflash_mlx.adapters import LoadedTargetModel

ROOT = Path(__file__).resolve().parent.parent
NULL, SHAPE, UNSUPPORTED, ALIGN = -1, -2, -3, -4
P = 0x1000  # stands for a device pointer: no call below gets as far as a launch


@pytest.fixture(scope="module")
def lib():
    from dflash_mlx import _lib

    return _lib.load()


def _rows(lib, x=P, xs=256, w=P, ws=256, H=256, V=1000, out=P, os=1000, M=4):
    return lib.dflash_lm_head_logits(x, xs, w, ws, H, V, out, os, M, None)


def _tiled(lib, x=P, xs=256, w=P, H=256, V=1008, out=P, os=1008, M=4):
    return lib.dflash_lm_head_logits_tiled(x, xs, w, H, V, out, os, M, None)


def test_every_declared_entry_point_is_exported_and_bound(lib):
    from dflash_mlx import _lib

    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "dflash_lm_logits.h").read_text(), flags=re.S)
    names = set(re.findall(r"\b(dflash_[a-z0-9_]+)\s*\(", text))
    assert names == {"dflash_lm_head_logits", "dflash_lm_head_logits_tiled"}
    for name in names:
        assert hasattr(lib, name) and name in _lib.SIGNATURES


@pytest.mark.parametrize("call", [_rows, _tiled])
def test_calls_that_are_refused(lib, call):
    for kw in (dict(M=-1), dict(H=0), dict(V=0), dict(xs=248), dict(os=999)):
        assert call(lib, **kw) == SHAPE
    for kw in (dict(M=65), dict(H=200, xs=200)):
        assert call(lib, **kw) == UNSUPPORTED
    for name in ("x", "w", "out"):
        assert call(lib, **{name: None}) == NULL
    for kw in (dict(x=P + 8), dict(w=P + 8), dict(xs=260), dict(out=P + 2)):
        assert call(lib, **kw) == ALIGN
    assert call(lib, M=0, x=None) == 0
    assert _rows(lib, ws=248) == SHAPE and _rows(lib, ws=-1) == SHAPE and _rows(lib, ws=260) == ALIGN
    assert _tiled(lib, V=1000) == UNSUPPORTED


def test_targets_without_logits_of_their_own_for_the_argmax():
    """A model, or an adapter, that knows nothing of them gives its logits."""

    class Model:
        def lm_head_logits(self, hidden):
            return ("logits", hidden)

    class Own(Model):
        def lm_head_logits_fp32(self, hidden):
            return ("fp32", hidden)

    class Adapter:
        def lm_head_logits(self, model, hidden):
            return ("adapter", hidden)

    assert LoadedTargetModel(model=Model()).lm_head_logits_fp32(1) == ("logits", 1)
    assert LoadedTargetModel(model=Own()).lm_head_logits_fp32(1) == ("fp32", 1)
    assert LoadedTargetModel(model=Own(), adapter=Adapter()).lm_head_logits_fp32(1) == ("adapter", 1)
