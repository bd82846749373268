"""The hybrid target over caches in 8 bits (kv_dtype int8 or float8_e4m3fn).

The attention layer's cache is checked against the layer's own inputs through
the bf16 cache's run: hidden states of the two targets differ by what 8 bits
lose, so the cache is compared with the definition applied to its own tail and
codes, and the decode loop with itself: what a cache holds after blocks with
rejected drafts, trims and prompts is what the kept tokens alone leave."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from dflash_mlx.gdn_layer import GatedDeltaConfig
from dflash_mlx.hybrid_model import HybridConfig, HybridVerifyRunner, HybridWeights
from dflash_mlx.target import DeviceQuantizedKVCache, HybridTargetModel
from oracle import kv8_oracle as orc
from tests.kv8_util import BLOCK, D, DTYPES

pytestmark = pytest.mark.gpu

CFG = HybridConfig(hidden_size=256, num_hidden_layers=4, intermediate_size=512, vocab_size=1024,
                   num_attention_heads=4, num_key_value_heads=1, head_dim=128,
                   linear=GatedDeltaConfig(linear_num_key_heads=2, linear_num_value_heads=4))


@pytest.fixture(scope="module")
def weights(device):
    return HybridWeights.random(CFG, device, seed=5, on_device=False)


def _model(weights, device, dtype, **kw):
    return HybridTargetModel(CFG, weights, device, max_seq_len=512, block_size=16, kv_dtype=dtype, **kw)


def _tokens(n, seed=0):
    return torch.randint(0, 1024, (1, n), generator=torch.Generator().manual_seed(seed))


def _keys_values(cache):
    c = cache[cache.attn_idx[0]]
    assert isinstance(c, DeviceQuantizedKVCache)
    return c.keys, c.values


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("mode", ["prefill", "blocks"])
def test_hidden_states_near_the_bf16_cache(weights, device, dtype, mode):
    """A prompt and a block after it: normwise within 8 bits of the bf16 cache.

    One attention layer of four.  A value's error is at most half a step: 2^-4 of it in
    e4m3 and 1 / 254 of the block's largest in int8; a weight's, with scores of std about
    1, is of the same order.  Random signs average over some hundred keys, and the branch
    is one of four: 2^-4 bounds it many times over."""
    toks = _tokens(300)
    outs = []
    for dt in (torch.bfloat16, dtype):
        m = _model(weights, device, dt, prompt_pass=mode)
        cache = m.make_cache()
        h0, _ = m.forward_dflash(toks[:, :290], cache, [3])
        h1, t1, rec = m.forward_dflash(toks[:, 290:], cache, [3], return_rollback_records=True)
        outs.append(torch.cat((h0, h1), 1).float())
    err = (outs[0] - outs[1]).norm() / outs[0].norm()
    print(f"[kv8 model] {dtype} {mode}: {err:.2e} of the bf16 cache's hidden states", flush=True)
    assert torch.isfinite(outs[1]).all() and 0 < err <= 2.0 ** -4


@pytest.mark.parametrize("dtype", DTYPES)
def test_cache_of_kept_tokens(weights, device, dtype):
    """Blocks of which some drafts are rejected, twice with other rejected drafts: the
    caches hold the same, bit for bit, as no step reads a rejected token."""
    m = _model(weights, device, dtype)
    runs = []
    for rejected in (50, 900):  # seeds of the rejected drafts
        cache = m.make_cache()
        m.forward_dflash(_tokens(70), cache, [3])
        for i in range(14):
            keep = (5, 16, 1, 9, 13)[i % 5]
            block = torch.cat((_tokens(keep, seed=20 + i), _tokens(16 - keep, seed=rejected + i)), 1)
            _, _, rec = m.forward_dflash(block, cache, [3], return_rollback_records=True)
            for j in cache.attn_idx:
                cache[j].trim(16 - keep)
            m.rollback_linear_caches(cache, rec, keep)
        runs.append(_keys_values(cache))
    for a, b in zip(*runs):
        assert a.shape[2] > 2 * BLOCK and torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rewinds_past_the_tail(weights, device, dtype):
    """Trims by 1 to 300 positions, then another block: what is left of the cache reads
    as it did before, complete blocks bit for bit, the block that the cut opens again
    within its codes' rounding to bf16."""
    m = _model(weights, device, dtype)
    toks = _tokens(330)
    for cut in (1, 20, 60, 64, 70, 100, 129, 200, 265, 300):
        cache = m.make_cache()
        m.forward_dflash(toks, cache, [3])
        m.forward_dflash(_tokens(16, seed=3), cache, [3])
        k0, v0 = (x.clone() for x in _keys_values(cache))
        c = cache[cache.attn_idx[0]]
        c.trim(16 + cut)
        n = c.offset
        m.forward_dflash(_tokens(5, seed=4), cache, [3])
        c.trim(5)
        k1, v1 = _keys_values(cache)
        assert k1.shape[2] == n == 330 - cut
        whole = n // BLOCK * BLOCK
        safe = max(0, whole - BLOCK) if n % BLOCK <= 16 else whole
        for a, b in ((k0, k1), (v0, v1)):
            assert torch.equal(a[:, :, :safe], b[:, :, :safe]), cut
            # requantised from bf16 of its own values: the scale may move by a rounding (2^-8),
            # and a code that sits at a border then by one
            x, y = a[:, :, safe:n].float(), b[:, :, safe:n].float()
            assert float((x - y).abs().max() if x.numel() else 0) <= 2.0 ** -3 * float(a.float().abs().max()), cut
        out, _ = m.forward_dflash(_tokens(16, seed=5), cache, [3])
        assert torch.isfinite(out.float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_serving_step_captured(weights, device, dtype):
    """The device-driven step of three sequences: eager and as a replayed graph, the same
    tokens and caches; states loaded from bf16 keys and values."""
    B, T, Smax = 3, 16, 384
    g = torch.Generator().manual_seed(2)
    lens = [100, 63, 190]
    k = [torch.randn(B, 1, 256, D, generator=g).bfloat16().to(device)]
    v = [torch.randn(B, 1, 256, D, generator=g).bfloat16().to(device)]
    runs = []
    for graph in (False, True):
        run = HybridVerifyRunner(CFG, weights, B, T, Smax, device, kv_dtype=dtype)
        run.set_state(lens, k=k, v=v)
        if graph:
            run.capture_step()
        seen = []
        for i in range(8):
            run.tokens.copy_(torch.randint(0, 1024, (B, T), generator=torch.Generator().manual_seed(i)))
            run.replay() if graph else run.step()
            if i == 4:
                torch.cuda.synchronize()
            seen.append(torch.cat((run.posterior.flatten(), run.matched, run.lens)).clone())
        run.check_overflow()
        kv = run.kv[0]
        runs.append((torch.stack(seen).cpu(), kv.k_codes.view(torch.uint8).cpu(), kv.v_codes.view(torch.uint8).cpu(),
                     kv.tail_k.cpu(), kv.tail_vt.cpu()))
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    # the loaded history is quantised by the definition
    s, mul = orc.block_scale(k[0][2, :, :128].reshape(1, 2, BLOCK, D).cpu(), dtype)
    want = orc.block_codes(k[0][2, :, :128].reshape(1, 2, BLOCK, D).cpu(), mul, dtype).view(torch.uint8)
    assert torch.equal(runs[0][1][2, :, :128].view(1, 2, BLOCK, D), want)


@pytest.mark.parametrize("dtype", DTYPES)
def test_lengths_come_with_their_keys(weights, device, dtype):
    run = HybridVerifyRunner(CFG, weights, 1, 16, 128, device, kv_dtype=dtype)
    with pytest.raises(ValueError, match="keys and values"):
        run.set_state([5])
    run.set_state([0])
    with pytest.raises(TypeError, match="int8 or float8_e4m3fn"):
        HybridVerifyRunner(CFG, weights, 1, 16, 128, device, kv_dtype=torch.float16)


def test_refusals(weights, device):
    with pytest.raises(ValueError, match="64 query rows"):
        HybridVerifyRunner(dataclasses.replace(CFG, num_attention_heads=5), weights, 1, 16, 512, device, kv_dtype=torch.int8)
    with pytest.raises(ValueError, match="heads of 128"):
        HybridVerifyRunner(dataclasses.replace(CFG, head_dim=64), weights, 1, 16, 512, device, kv_dtype=torch.int8)
    with pytest.raises(TypeError, match="codes must be"):
        HybridVerifyRunner(CFG, weights, 1, 16, 512, device, kv_dtype=torch.float16)
