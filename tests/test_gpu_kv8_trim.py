"""Keys and values of the hybrid target's 8-bit caches read straight after a trim, before
any forward has made the tail ready: what the cache read there before the trim."""
from __future__ import annotations

import pytest
import torch

from tests.kv8_util import BLOCK, DTYPES
from tests.test_gpu_kv8_model import _keys_values, _model, _tokens, weights  # noqa: F401

pytestmark = pytest.mark.gpu


def _near(x, y, n, dtype):
    """y [.., n, D], read after a trim to n, is what x read there: complete blocks bit for
    bit; the open block's values, where they come from the tail's bf16 again, within half a
    step of the code that x read (int8: 1 / 254 of the block's largest; e4m3: 2^-4 of the
    value, at least 2^-10 of the scale, which is at most 1 / 224 of the largest) and x's
    rounding to bf16 (2^-8; the largest is read off x, so it may be off by that and a step)."""
    whole = n // BLOCK * BLOCK
    assert y.shape[2] == n and torch.equal(x[:, :, :whole], y[:, :, :whole])
    if n == whole:
        return
    block = x[:, :, whole:whole + BLOCK].float()
    a, b = block[:, :, :n - whole], y[:, :, whole:].float()
    top = block.abs().amax((2, 3), keepdim=True) * (1 + 2.0 ** -3)
    step = top / 254 if dtype is torch.int8 else torch.maximum(2.0 ** -4 * b.abs(), 2.0 ** -10 / 224 * top)
    assert bool(((a - b).abs() <= step + 2.0 ** -8 * a.abs()).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cuts", [(1,), (20,), (60,), (64,), (70,), (100,), (129,), (200,), (260,), (265,), (300,),
                                  (40, 30), (138, 64, 54), (202, 54), (10, 64, 118, 64)])
def test_read_after_trims(weights, device, dtype, cuts):  # noqa: F811
    m = _model(weights, device, dtype)
    cache = m.make_cache()
    m.forward_dflash(_tokens(330), cache, [3])
    m.forward_dflash(_tokens(16, seed=3), cache, [3])
    cache[cache.attn_idx[0]].trim(16)  # a rejected block
    _trim_and_read(m, cache, 330, cuts, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [128, 320])
@pytest.mark.parametrize("cuts", [(1,), (47,), (50,), (60,), (64,), (80,), (110,), (64, 50)])
def test_read_after_trims_of_a_prompt_of_whole_blocks(weights, device, dtype, n, cuts):  # noqa: F811
    """The prompt leaves its last block in the tail, and none before it."""
    m = _model(weights, device, dtype)
    cache = m.make_cache()
    m.forward_dflash(_tokens(n), cache, [3])
    _trim_and_read(m, cache, n, cuts, dtype)


def _trim_and_read(m, cache, n, cuts, dtype):
    c = cache[cache.attn_idx[0]]
    before = [x.clone() for x in _keys_values(cache)]
    for cut in cuts:
        c.trim(cut)
        n -= cut
        for x, y in zip(before, _keys_values(cache)):
            _near(x, y, n, dtype)
    m.forward_dflash(_tokens(5, seed=4), cache, [3])
    c.trim(5)
    for x, y in zip(before, _keys_values(cache)):
        _near(x, y, n, dtype)
