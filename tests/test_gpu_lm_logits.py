"""The logits that a verify step under a state, or a shaped generation, stores are the fp32
sums that the accept without logits compares: a state, mask or grammar that changes nothing
changes no token, however near the best two are."""
from __future__ import annotations

import dataclasses

import pytest
import torch

from dflash_mlx import DFlashGenerator, LogitsShaping, LogitsState, _lib, lm_head_argmax, tile_weight
from dflash_mlx.hybrid_model import HybridVerifyRunner, HybridWeights
from dflash_mlx.target import HybridTargetModel
from tests.logits_util import argmax_lowest
from tests.test_gpu_int8_model import CFG

pytestmark = pytest.mark.gpu


def _near_ties(w):
    """The rows again in the weight's second half, every 16th value a bf16 step up or down: the
    logits of a pair differ in their last fp32 bits, hardly ever in bf16."""
    half = w.shape[0] // 2
    twin = w[:half].clone()
    bits = twin.view(torch.int16)
    bits[:, ::16] += torch.randint(0, 2, bits[:, ::16].shape, generator=torch.Generator().manual_seed(3)).to(bits) * 2 - 1
    w[half:2 * half] = twin
    return w


@pytest.mark.parametrize("M", [1, 7, 16, 17, 32, 33, 48, 49, 64])
@pytest.mark.parametrize("V", [16, 1008, 4992, 1, 1003, 20011])
def test_sums_of_the_fused_accept(device, M, V):
    """Both layouts against 64 bits, and the argmax kernels' own choice among near ties.

    A product of bf16 values is exact in fp32; each of the H additions (and the join of up to
    four parts) is off by at most a step, 2^-23, of the magnitudes added up so far."""
    H = 320
    g = torch.Generator().manual_seed(M * V)
    x = torch.randn(M, H, generator=g).bfloat16()
    w = _near_ties(torch.randn(V, H, generator=g).bfloat16())
    want = x.double() @ w.double().T
    tol = (H + 4) * 2.0 ** -23 * (x.double().abs() @ w.double().abs().T)
    wide = torch.zeros(M, H + 24, dtype=torch.bfloat16, device=device)
    wide[:, 8:8 + H] = x.to(device)
    xd, wd = wide[:, 8:8 + H], w.to(device)
    for tiled in (False, True) if V % 16 == 0 else (False,):
        wt = tile_weight(wd) if tiled else None
        for first, extra in ((0, 0), (3, 5)):
            out = torch.full((M, V + extra + first), 7.0, device=device)
            view = out[:, first:first + V]
            if tiled:
                _lib.call("dflash_lm_head_logits_tiled", xd.data_ptr(), xd.stride(0), wt.data_ptr(), H, V, view.data_ptr(),
                          view.stride(0), M, _lib.stream_handle(device))
            else:
                _lib.call("dflash_lm_head_logits", xd.data_ptr(), xd.stride(0), wd.data_ptr(), H, H, V, view.data_ptr(),
                          view.stride(0), M, _lib.stream_handle(device))
            assert ((view.cpu().double() - want).abs() <= tol).all()
            assert (out[:, :first] == 7).all() and (out[:, first + V:] == 7).all()
            assert torch.equal(lm_head_argmax(xd, wd, weight_tiled=wt).cpu().long(), argmax_lowest(view.cpu()))


def _weights(device, V):
    cfg = dataclasses.replace(CFG, vocab_size=V)
    w = HybridWeights.random(cfg, device, seed=5, on_device=False)
    w.lm_head.copy_(_near_ties(w.lm_head.cpu()).to(device))
    return cfg, w


@pytest.mark.parametrize("V", [1024, 1003])
@pytest.mark.parametrize("layout", ["tiled", "rowmajor"])
@pytest.mark.parametrize("B,T", [(1, 1), (1, 16), (3, 5), (2, 16), (3, 16), (4, 16)])
def test_a_state_that_asks_for_nothing_changes_nothing(device, V, layout, B, T):
    cfg, w = _weights(device, V)
    plain = HybridVerifyRunner(cfg, w, B, T, 256, device, weight_layout=layout)
    states = HybridVerifyRunner(cfg, w, B, T, 256, device, weight_layout=layout,
                                logits_state=LogitsState.zeros(B, V, device))
    masked = HybridVerifyRunner(cfg, w, B, T, 256, device, weight_layout=layout, masked=True)
    apart = 0
    for k in range(4):
        tokens = torch.randint(0, V, (B, T), generator=torch.Generator().manual_seed(k)).int()
        for run in (plain, states, masked):
            run.set_state([0] * B)
            run.tokens.copy_(tokens)
            run.step()
        for run in (states, masked):
            assert run.logits.dtype is torch.float32
            for name in ("posterior", "matched", "bonus", "keep", "lens"):
                assert torch.equal(getattr(run, name), getattr(plain, name)), name
        apart += int((states.logits.bfloat16().cpu().float().argmax(-1) != states.posterior.view(-1).cpu()).sum())
    assert apart > 0 or B * T == 1  # (logits in bf16 would have)


def test_a_grammar_that_allows_everything_changes_nothing(device):
    """The mode that takes its tokens from the fused argmax, under a shaping."""
    V = 1024
    cfg, w = _weights(device, V)

    class Drafter:
        mask_token_id, target_layer_ids, block_size = 0, [1, 3], 8

        def make_cache(self):
            return []

        def __call__(self, noise_embedding, target_hidden, cache=None):
            return noise_embedding * 40

    prompt = torch.randint(0, V, (21,), generator=torch.Generator().manual_seed(3)).int()
    allowed = torch.full((V // 32,), -1, dtype=torch.int32)
    got = []
    for shaping in (None, LogitsShaping(token_mask=lambda t: allowed)):
        m = HybridTargetModel(cfg, w, device, max_seq_len=256, block_size=8)
        got.append(DFlashGenerator(m, Drafter()).generate_from_tokens(
            prompt, max_new_tokens=60, verify_mode="parallel-greedy-argmax", shaping=shaping).generated_tokens)
    assert got[0] == got[1]
    hidden = torch.randn(2, 70, cfg.hidden_size, generator=torch.Generator().manual_seed(4)).bfloat16().to(device)
    logits = m.lm_head_logits_fp32(hidden)
    assert logits.shape == (2, 70, V) and logits.dtype is torch.float32
    rows = hidden.view(140, -1)
    for m0 in range(0, 140, 64):
        assert torch.equal(m.lm_head_argmax(rows[m0:m0 + 64]).cpu().long(),
                           argmax_lowest(logits.view(140, V)[m0:m0 + 64].cpu()))


def test_blocks_that_are_kept_whole_are_the_callers_to_count(device):
    """accept_all leaves a state alone; the next commit counts as ever."""
    V = 1024
    cfg, w = _weights(device, V)
    state = LogitsState.zeros(1, V, device)
    run = HybridVerifyRunner(cfg, w, 1, 8, 256, device, logits_state=state)
    run.set_state([0])
    run.tokens.copy_(torch.arange(8, dtype=torch.int32)[None])
    run.forward()
    run.accept_all(8)
    run.lens.add_(8)
    assert state.counts.abs().sum() == 0 and state.known.abs().sum() == 0
    state.add([list(range(9))], prompt=True)
    run.tokens.copy_(torch.arange(8, 16, dtype=torch.int32)[None])
    run.step()
    counts = state.counts[0].cpu().long()
    made = torch.where(counts < 0, counts + 2 ** 31, counts)
    assert made.sum() == run.matched.item() + 1 and (counts[:9] < 0).all() and run.lens.item() == 8 + run.keep.item()
