"""The hybrid target with its weights in 8-bit integers, and its verify step under
penalties, biases and masks: everything of the set together, eager and captured."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import DFlashGenerator, LogitsShaping, LogitsState, linear_i8
from dflash_mlx.gdn_layer import GatedDeltaConfig
from dflash_mlx.hybrid_model import HybridConfig, HybridVerifyRunner, HybridWeights
from dflash_mlx.target import HybridTargetModel
from tests.logits_util import argmax_lowest, processed, words

pytestmark = pytest.mark.gpu

CFG = HybridConfig(hidden_size=256, num_hidden_layers=4, intermediate_size=512, vocab_size=1024,
                   num_attention_heads=4, num_key_value_heads=1, head_dim=128,
                   linear=GatedDeltaConfig(linear_num_key_heads=2, linear_num_value_heads=4))
V = CFG.vocab_size


@pytest.fixture(scope="module")
def weights(device):
    return HybridWeights.random(CFG, device, seed=5, on_device=False)


def _tokens(*shape, seed=0):
    return torch.randint(0, V, shape, generator=torch.Generator().manual_seed(seed))


@pytest.mark.parametrize("mode", ["prefill", "blocks"])
@pytest.mark.parametrize("kv", [torch.bfloat16, torch.int8])
def test_hidden_states_near_the_bf16_target(weights, device, mode, kv):
    """A prompt and a block after it.

    A projection is off by 1.2e-2 of itself (both operands' half steps, see the projections'
    tests), a branch has two in a row with a nonlinearity between that at most doubles it:
    5e-2 of the branch.  Eight branches with independent errors, none larger than the
    residual stream: 5e-2 of it where they make it up; three times that bounds it."""
    toks = _tokens(1, 300)
    outs = []
    for dt in (torch.bfloat16, torch.int8):
        m = HybridTargetModel(CFG, weights, device, max_seq_len=512, block_size=16, prompt_pass=mode, kv_dtype=kv,
                              weight_dtype=dt)
        cache = m.make_cache()
        h0, t0 = m.forward_dflash(toks[:, :290], cache, [1, 3])
        h1, t1, _ = m.forward_dflash(toks[:, 290:], cache, [1, 3], return_rollback_records=True)
        outs.append((torch.cat((h0, h1), 1).float(), torch.cat((t0, t1), 1).float()))
        logits = m.lm_head_logits(h1)
        assert logits.dtype is (torch.float32 if dt is torch.int8 else torch.bfloat16)
        if dt is torch.int8:
            assert torch.equal(logits, linear_i8(h1, weights.lm_head_i8, out_dtype=torch.float32))
            assert torch.equal(m.lm_head_argmax(h1), logits.argmax(-1).int())
    for a, b in zip(*outs):
        err = (a - b).norm() / a.norm()
        print(f"[int8 model] {mode} {kv}: {err:.2e} of the bf16 target's", flush=True)
        assert torch.isfinite(b).all() and 0 < err <= 0.15


def test_modes_agree_over_the_int8_target(weights, device):
    """The verify modes that share the block forward take the same tokens, shaped or not."""

    class Drafter:
        mask_token_id, target_layer_ids, block_size = 0, [1, 3], 8

        def make_cache(self):
            return []

        def __call__(self, noise_embedding, target_hidden, cache=None):
            return noise_embedding * 40

    prompt = _tokens(21, seed=3).int()
    for shaping in (None, (1.5, 0.5, 0.1)):
        got = {}
        for mode in ("parallel-replay", "parallel-lazy-logits", "parallel-greedy-argmax"):
            m = HybridTargetModel(CFG, weights, device, max_seq_len=256, block_size=8, weight_dtype=torch.int8)
            res = DFlashGenerator(m, Drafter()).generate_from_tokens(
                prompt, max_new_tokens=24, verify_mode=mode, verify_chunk_size=3,
                shaping=LogitsShaping(*shaping) if shaping else None)
            got[mode] = res.generated_tokens
        assert got["parallel-replay"] == got["parallel-lazy-logits"] == got["parallel-greedy-argmax"]
        assert len(got["parallel-replay"]) == 24
        if shaping:
            assert len(set(got["parallel-replay"])) > 1


B, T, SMAX = 3, 5, 256


def _state(device):
    s = LogitsState.zeros(B, V, device)
    s.set_penalties(torch.tensor([1.0, 1.3, 1.6]), torch.tensor([0.0, 0.4, 0.2]), torch.tensor([0.0, 0.1, 0.3]))
    s.set_bias([[5, 6], [7, 8], [9, 10]], [[1.0, -1.0], [2.0, -2.0], [0.5, 3.0]])
    s.add(_tokens(B, 30, seed=9).int(), prompt=True)
    return s


def _runner(weights, device, dtype, state, masked):
    run = HybridVerifyRunner(CFG, weights, B, T, SMAX, device, weight_dtype=dtype, logits_state=state, masked=masked)
    run.set_state([0] * B)
    return run


def test_norms_that_leave_codes_and_norms_that_do_not(weights, device):
    """Hidden sizes without whole 16s quantise in a launch of their own, as the codes' own
    norm does: about one value in 2^10 lies near enough to a bf16 border that it rounds the
    other way, by one code at most, where every code is off by 0.29 (rms) as it is.  So the
    two differ by 2^-5 / 0.29, a ninth, of what either is off (0.15 at most, see above)."""
    out = []
    for codes in (True, False):
        run = _runner(weights, device, torch.int8, None, False)
        assert run.norm_codes
        run.norm_codes = codes
        run.tokens.copy_(_tokens(B, T, seed=4).int())
        run.step()
        out.append(run.xn.float())
    err = (out[0] - out[1]).norm() / out[1].norm()
    print(f"[int8 model] norms with and without codes: {err:.2e}", flush=True)
    assert torch.isfinite(out[0]).all() and err <= 0.15 / 9


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.int8])
@pytest.mark.parametrize("masked", [False, True])
def test_steps_under_a_state(weights, device, dtype, masked):
    """Eager steps: the accept is that of the stored logits by the definition, the counts
    are those of the tokens kept; a captured step replays to the same bits."""
    s, s2 = _state(device), _state(device)
    run, cap = _runner(weights, device, dtype, s, masked), _runner(weights, device, dtype, s2, masked)
    first = _tokens(B, 1, seed=1).int()
    for st in (s, s2):
        st.add(first)
    block = torch.cat((first, _tokens(B, T - 1, seed=2).int()), 1)
    cap.step()  # (a graph's first run outside it)
    cap.set_state([0] * B, conv=[torch.zeros_like(c) for c in cap.conv], rec=[torch.zeros_like(r) for r in cap.state])
    for k in range(2):
        (s2[k] if k else s2).reset()
    fresh = _state(device)
    for name in ("counts", "known", "bias", "penalties"):
        getattr(s2, name).copy_(getattr(fresh, name))
    s2.add(first)
    cap.capture_step()
    for k in range(5):
        for r in (run, cap):
            r.tokens.copy_(block)
        if masked:
            allowed = torch.rand(B, T, V, generator=torch.Generator().manual_seed(k)) < 0.5
            allowed[1] = True
            for r in (run, cap):
                r.mask.copy_(words(allowed))
        c = s.counts.cpu().long()
        made, prompt = torch.where(c < 0, c + 2 ** 31, c), c < 0
        run.step()
        cap.replay()
        steps, _ = processed(run.logits.view(B, T, V).cpu(), made, prompt, s.bias.cpu(), s.penalties.cpu(),
                             block[:, 1:].tolist(), allowed if masked else None, torch.float32)
        post = argmax_lowest(steps)
        assert torch.equal(run.posterior.cpu().long(), post)
        matched = run.matched.tolist()
        for b in range(B):
            n = 0
            while n < T - 1 and block[b, n + 1] == post[b, n]:
                n += 1
            assert matched[b] == n
            for t in post[b, :n + 1].tolist():
                made[b, t] += 1
        c = s.counts.cpu().long()
        assert torch.equal(torch.where(c < 0, c + 2 ** 31, c), made)
        for name in ("posterior", "matched", "bonus", "lens", "keep", "xn"):
            assert torch.equal(getattr(run, name), getattr(cap, name)), name
        assert torch.equal(s.counts, s2.counts) and torch.equal(s.known, s2.known)
        # the next block: the bonus, some of its drafts what the target is likely to take
        nxt = torch.cat((run.bonus.cpu()[:, None], _tokens(B, T - 1, seed=20 + k).int()), 1)
        nxt[0, 1:] = post[0, :T - 1].int()
        block = nxt


def test_refusals(weights, device):
    with pytest.raises(ValueError, match="weight_dtype"):
        HybridVerifyRunner(CFG, weights, 1, 4, 64, device, weight_dtype=torch.float16)
    with pytest.raises(ValueError, match="logits_state"):
        HybridVerifyRunner(CFG, weights, 2, 4, 64, device, logits_state=LogitsState.zeros(1, V, device))
    away = LogitsState.zeros(1, V, device)
    away.device = torch.device("cuda", 7)
    with pytest.raises(ValueError, match="logits_state"):
        HybridVerifyRunner(CFG, weights, 1, 4, 64, device, logits_state=away)
