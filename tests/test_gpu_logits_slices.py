"""Logits processing where a workgroup's slice of a row is as long as it gets: 4096 entries of
fp32, 8192 of 16 bits, in turns of 2048.  (Few rows are split further: slices of 2048 at most.)

Tolerances and exact greedy tokens as in the tests of short slices."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import LogitsState, _lib, greedy_accept, process_logits
from tests.logits_util import accept, argmax_lowest, counts_of, processed, words
from tests.test_gpu_logits import TYPES, _check

pytestmark = pytest.mark.gpu

B, N, V = 32, 16, 40011  # 512 rows: 8192 x 4 + 7243 entries, or 4096 x 9 + 3147


def _slices(dtype):
    n = _lib.load().dflash_greedy_accept_processed_workspace_bytes(B, N, V) // (8 * B * N)
    assert n == 10  # of fp32
    return 4096 if dtype is torch.float32 else 8192


def _inputs(dtype, history, mask, seed):
    """Logits in steps of 1/2 (ties everywhere), the largest planted behind the first turn."""
    g = torch.Generator().manual_seed(seed)
    logits = (2 * torch.randn(B, N, V, generator=g)).round() / 2
    chunk = _slices(dtype)
    for b in range(B):
        for i in range(N):
            at = torch.randint(2048, chunk, (3,), generator=g) + chunk * torch.randint(0, 4, (3,), generator=g)
            logits[b, i, at.clamp_max(V - 1)] = 20.0  # three equal ones
    logits[1, 2, chunk - 1] = logits[1, 2, 2100] = torch.nan  # the first of two NaN
    logits[2, 3, V - 1] = torch.inf
    logits[3, :, :] = -torch.inf
    logits[3, 4, chunk + 2049] = -100.0
    prompt = [torch.randint(0, V, (history,), generator=g).tolist() for _ in range(B)]
    made = [torch.randint(0, V, (history // 3,), generator=g).tolist() for _ in range(B)]
    draft = torch.randint(0, V, (B, N - 1), generator=g)
    draft[:, 5] = draft[:, 2]  # one twice
    draft[7] = torch.arange(2048 - 7, 2048 + 8)  # over the border of two turns
    draft[8] = torch.arange(chunk - 7, chunk + 8)
    for b in range(9, B):
        draft[b, 1] = prompt[b][0]
        draft[b, 3] = V - 1 - b % 5
    pen = torch.stack((1 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g) - 0.3), 1)
    allowed = torch.rand(B, N, V, generator=g) < 0.7 if mask else None
    if mask:
        allowed[10], allowed[11, 3], allowed[12, 4] = True, False, False
        allowed[12, 4, V - 2] = True
    return logits.to(dtype), prompt, made, draft.tolist(), pen, allowed


def _run(device, dtype, logits, prompt, made, draft, pen, allowed):
    s = LogitsState.zeros(B, V, device)
    s.set_penalties(pen[:, 0], pen[:, 1], pen[:, 2])
    ids = torch.stack([(torch.arange(8) * 4999 + 3 * b) % V for b in range(B)])
    values = torch.linspace(-3, 3, 8).repeat(B, 1)
    s.set_bias(ids.int().to(device), values.to(device))
    for tokens, is_prompt in ((prompt, True), (made, False)):
        s.add(torch.tensor(tokens, dtype=torch.int32, device=device), prompt=is_prompt)
    bias = torch.zeros(B, V).scatter_(1, ids, values)
    c, p = counts_of(prompt, made, V)
    m = words(allowed).to(device) if allowed is not None else None
    d = torch.tensor(draft, dtype=torch.int32, device=device)
    lg = logits.to(device)

    want, size = processed(logits, c, p, bias, pen, draft, allowed)
    nan = want.isnan()
    want, size = want.masked_fill_(nan, 0), size.masked_fill_(nan, 0)
    inf = want.isposinf()
    outs = [process_logits(lg, s, d, mask=m)]
    again = lg.clone()
    outs.append(process_logits(again, s, d, mask=m, out=again))
    for out in outs:
        out = out.cpu()
        assert torch.equal(out.isnan(), nan) and torch.equal(out.isposinf(), inf)
        dead = nan | inf | logits.isneginf()  # (their magnitudes are none)
        assert out[logits.isneginf()].isneginf().all()
        _check(out.masked_fill(dead, 0), want.masked_fill(dead, 0), size.masked_fill(dead, 0), dtype)
    del want, size, outs

    steps, _ = processed(logits, c, p, bias, pen, draft, allowed, torch.float32)
    post = argmax_lowest(steps)
    agree = [post[b, :N - 1].tolist()[:b % N] + draft[b][b % N:] for b in range(B)]
    steps, _ = processed(logits, c, p, bias, pen, agree, allowed, torch.float32)
    post = argmax_lowest(steps)
    got, matched, bonus = greedy_accept(lg, torch.tensor(agree, dtype=torch.int32, device=device), state=s, mask=m)
    assert torch.equal(got.cpu().long(), post)
    want_m, want_b = accept(post, agree)
    assert matched.tolist() == want_m and bonus.tolist() == want_b
    return post


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("mask", [False, True])
def test_slices_of_several_turns(device, dtype, mask):
    post = _run(device, dtype, *_inputs(dtype, 900, mask, seed=1))
    if not mask:
        assert post[1, 2] == 2100 and post[2, 3] == V - 1
        assert (post % _slices(dtype) >= 2048).float().mean() > 0.5
    else:
        assert post[11, 3] == 0 and post[12, 4] in (0, V - 2)


@pytest.mark.parametrize("dtype,mask", [(torch.float32, True), (torch.bfloat16, False), (torch.float16, True)])
def test_more_known_tokens_than_are_listed(device, dtype, mask):
    """Sequences that know every token, or every second: more than 2048 of a slice, and allowed."""
    logits, prompt, made, draft, pen, allowed = _inputs(dtype, 30000, mask, seed=2)
    for b in range(0, B, 3):
        prompt[b] = [(t * (1 + b % 2)) % V for t in range(30000)]
        made[b] = [V - 1 - t for t in range(10000)]
    _run(device, dtype, logits, prompt, made, draft, pen, allowed)
