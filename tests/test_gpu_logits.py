"""Logits processing against its definition in 64 bits, and the greedy accept under it.

Tolerance of a processed logit: the steps round once each (a division or product, the
product frequency * count, two subtractions, the bias), each by at most 2^-24 of a value
no larger than the terms' magnitudes together: 5 * 2^-24 of that sum, and half a step of
the output's type.  Greedy tokens are compared with the same steps in fp32, where they
have to be equal."""
from __future__ import annotations

import random

import pytest
import torch

from dflash_mlx import LogitsState, greedy_accept, process_logits
from tests.logits_util import accept, argmax_lowest, counts_of, processed, words

pytestmark = pytest.mark.gpu

TYPES = (torch.float32, torch.bfloat16, torch.float16)


def _case(B, N, V, dtype, seed=0, mask=True, n_draft=None, history=30):
    """Inputs on the host: logits, token lists, biases, penalties, drafts, allowed."""
    g = torch.Generator().manual_seed(seed)
    r = random.Random(seed)
    logits = (3 * torch.randn(B, N, V, generator=g)).to(dtype)
    prompt = [[r.randrange(V) for _ in range(r.randrange(history + 1))] for _ in range(B)]
    made = [[r.randrange(min(V, 50)) for _ in range(r.randrange(history + 1))] for _ in range(B)]
    nb = min(V, 8)
    ids = torch.stack([torch.randperm(V, generator=g)[:nb] for _ in range(B)]).int()
    values = 4 * torch.randn(B, nb, generator=g)
    pen = torch.stack((1 + torch.rand(B, generator=g), torch.rand(B, generator=g), torch.rand(B, generator=g) - 0.3), 1)
    n = N - 1 if n_draft is None else n_draft
    draft = [[r.randrange(min(V, 60)) for _ in range(n)] for _ in range(B)]
    allowed = torch.rand(B, N, V, generator=g) < 0.6 if mask else None
    return logits, prompt, made, ids, values, pen, draft, allowed


def _state(device, B, V, prompt, made, ids, values, pen):
    s = LogitsState.zeros(B, V, device)
    s.set_penalties(pen[:, 0], pen[:, 1], pen[:, 2])
    s.set_bias(ids.to(device), values.to(device))
    for tokens, is_prompt in ((prompt, True), (made, False)):
        n = max(len(t) for t in tokens)
        lens = torch.tensor([len(t) for t in tokens], dtype=torch.int32, device=device)
        padded = torch.tensor([t + [0] * (n - len(t)) for t in tokens], dtype=torch.int32).view(B, n)
        s.add(padded.to(device), lens, prompt=is_prompt)
    return s


def _dense(ids, values, V):
    return torch.zeros(len(ids), V).scatter_(1, ids.long(), values)


def _check(got, want, size, dtype):
    got = got.cpu()
    assert torch.equal(torch.isneginf(got), torch.isneginf(want))
    live = ~torch.isneginf(want)
    tol = 5 * 2.0 ** -24 * size + torch.finfo(dtype).eps / 2 * want.abs() + torch.finfo(dtype).tiny
    bad = ((got.double() - want).abs() > tol) & live
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} beyond the tolerance"


SHAPES = [(1, 1, 1), (1, 1, 7), (2, 3, 8), (1, 4, 33), (3, 2, 1000), (2, 16, 4099), (1, 5, 20011), (33, 1, 515)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("mask", [False, True])
def test_processed_and_accepted(device, shape, dtype, mask):
    B, N, V = shape
    logits, prompt, made, ids, values, pen, draft, allowed = _case(B, N, V, dtype, seed=B + N + V, mask=mask)
    s = _state(device, B, V, prompt, made, ids, values, pen)
    c, p = counts_of(prompt, made, V)
    m = words(allowed).to(device) if mask else None
    bias = _dense(ids, values, V)
    d = torch.tensor(draft, dtype=torch.int32).view(B, N - 1).to(device)
    want, size = processed(logits, c, p, bias, pen, draft, allowed)
    _check(process_logits(logits.to(device), s, d, mask=m), want, size, dtype)
    same = logits.to(device)
    assert process_logits(same, s, d, mask=m, out=same) is same
    _check(same, want, size, dtype)

    steps, _ = processed(logits, c, p, bias, pen, draft, allowed, torch.float32)
    post = argmax_lowest(steps)
    # drafts that agree for a while
    agree = [post[b, :N - 1].tolist()[:b % N] + draft[b][b % N:] for b in range(B)]
    steps, _ = processed(logits, c, p, bias, pen, agree, allowed, torch.float32)
    post = argmax_lowest(steps)
    got, matched, bonus = greedy_accept(logits.to(device), torch.tensor(agree, dtype=torch.int32).view(B, N - 1).to(device),
                                        state=s, mask=m)
    assert torch.equal(got.cpu().long(), post)
    want_m, want_b = accept(post, agree)
    assert matched.tolist() == want_m and bonus.tolist() == want_b
    none, m2, b2 = greedy_accept(logits.to(device), agree, state=s, mask=m, want_posterior=False)
    assert none is None and torch.equal(m2, matched) and torch.equal(b2, bonus)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(device, dtype):
    """Rows that begin at any element, batches inside a wider buffer, [N, B] orders."""
    B, N, V = 2, 3, 1003
    logits, prompt, made, ids, values, pen, draft, allowed = _case(B, N, V, dtype, seed=3)
    s = _state(device, B, V, prompt, made, ids, values, pen)
    c, p = counts_of(prompt, made, V)
    want, size = processed(logits, c, p, _dense(ids, values, V), pen, draft, allowed)
    m = words(allowed).to(device)
    d = torch.tensor(draft, dtype=torch.int32).to(device)
    for first in (0, 1, 3):
        wide = torch.full((N, B, V + 9), 7.0, dtype=dtype, device=device)
        wide[:, :, first:first + V] = logits.to(device).transpose(0, 1)
        view = wide[:, :, first:first + V].transpose(0, 1)
        out = torch.full((B, N, V + 5), 9.0, dtype=dtype, device=device)
        process_logits(view, s, d, mask=m, out=out[:, :, 2:2 + V])
        _check(out[:, :, 2:2 + V], want, size, dtype)
        assert (out[:, :, :2] == 9).all() and (out[:, :, 2 + V:] == 9).all()
        post = greedy_accept(view, d, state=s, mask=m)[0]
        assert torch.equal(post, greedy_accept(logits.to(device), d, state=s, mask=m)[0])
        process_logits(view, s, d, mask=m, out=view)
        _check(view, want, size, dtype)
        assert (wide[:, :, :first] == 7).all() and (wide[:, :, first + V:] == 7).all()
    # every other entry: a copy
    two = torch.stack((logits, logits), -1).view(B, N, 2 * V)[:, :, ::2].to(device)
    spread = torch.empty(B, N, 2 * V, dtype=dtype, device=device)[:, :, ::2]
    spread.copy_(two)
    _check(process_logits(spread, s, d, mask=m), want, size, dtype)


def test_masks(device):
    """Empty rows, shared masks, NaN and infinities under them; without a state."""
    B, N, V = 2, 4, 777
    logits = torch.randn(B, N, V)
    logits[0, 1, 5], logits[0, 2, 6], logits[1, 0, 7], logits[1, 1, 8] = torch.nan, torch.inf, -torch.inf, torch.nan
    allowed = torch.rand(N, V) < 0.5
    allowed[1, 5], allowed[2, 6], allowed[3] = False, False, False
    allowed[0, 7], allowed[1, 8] = True, True
    mask = words(allowed).to(device)
    lg = logits.to(device)
    want = torch.where(allowed, logits, torch.full_like(logits, -torch.inf))
    shared = mask.expand(B, N, -1)
    out = process_logits(lg, mask=shared)
    assert torch.equal(out.cpu().nan_to_num(nan=123.0), want.nan_to_num(nan=123.0))
    post, matched, bonus = greedy_accept(lg, None, mask=shared)
    assert torch.equal(post.cpu().long(), argmax_lowest(want))
    assert post[:, 3].tolist() == [0, 0] and post[1, 1] == 8  # nothing left; a NaN ranks above all
    assert bonus.tolist() == post[:, 0].tolist() and matched.tolist() == [0, 0]
    # one mask for all rows of a sequence, [N, V] logits
    one = mask[:1].expand(N, -1)
    assert torch.equal(process_logits(lg[0], mask=one).cpu().nan_to_num(nan=1.0),
                       torch.where(allowed[0], logits[0], torch.full_like(logits[0], -torch.inf)).nan_to_num(nan=1.0))


def test_not_finite_logits_under_penalties(device):
    """Infinities keep their place, a NaN stays one."""
    V = 40
    logits = torch.zeros(1, 1, V)
    logits[0, 0, :4] = torch.tensor([torch.inf, -torch.inf, torch.nan, -0.0])
    s = LogitsState.zeros(1, V, device)
    s.set_penalties(1.5, 0.5, 0.25)
    s.add([[0, 1, 2, 3]])
    out = process_logits(logits.to(device), s)[0, 0].cpu()
    assert out[0] == torch.inf and out[1] == -torch.inf and torch.isnan(out[2]) and out[3] == -0.75
    assert greedy_accept(logits.to(device), state=s)[0].item() == 2


def test_drafts(device):
    """Repeated drafts, drafts of the prompt, outside the vocabulary, more or fewer than the rows."""
    V, N = 300, 6
    logits = torch.randn(1, N, V)
    s = LogitsState.zeros(1, V, device)
    s.set_penalties(1.3, 0.7, 0.4)
    s.add([[9, 9, 11]])
    s.add([[9, 12]], prompt=True)
    c, p = counts_of([[9, 12]], [[9, 9, 11]], V)
    pen = torch.tensor([[1.3, 0.7, 0.4]])
    for draft in ([9, 9, 9, 12, 12], [-1, 299, 300, 2 ** 31 - 1, -2 ** 31], [5], [], [1, 2, 3, 4, 5, 6, 7, 8]):
        want, size = processed(logits, c, p, torch.zeros(1, V), pen, [draft], None)
        got = process_logits(logits.to(device), s, torch.tensor([draft], dtype=torch.int32, device=device))
        _check(got, want, size, torch.float32)
    assert torch.equal(process_logits(logits.to(device), s), process_logits(logits.to(device), s, [[]]))


def test_a_block_is_as_its_tokens_one_by_one(device):
    """Row i of a block equals the single row after counting the drafts before it, bit for bit."""
    B, N, V = 3, 16, 5000
    logits, prompt, made, ids, values, pen, draft, _ = _case(B, N, V, torch.float32, seed=11)
    s = _state(device, B, V, prompt, made, ids, values, pen)
    d = torch.tensor(draft, dtype=torch.int32).to(device)
    block = process_logits(logits.to(device), s, d)
    for i in range(N):
        assert torch.equal(process_logits(logits[:, i:i + 1].to(device), s)[:, 0], block[:, i])
        if i < N - 1:
            s.add(d[:, i:i + 1])


def test_64_drafts(device):
    V, N = 500, 65
    logits = torch.randn(1, N, V)
    draft = [[(7 * i) % 40 for i in range(64)]]
    s = LogitsState.zeros(1, V, device)
    s.set_penalties(1.2, 0.1, 0.05)
    c, p = counts_of([[]], [[]], V)
    want, size = processed(logits, c, p, torch.zeros(1, V), torch.tensor([[1.2, 0.1, 0.05]]), draft, None)
    _check(process_logits(logits.to(device), s, draft), want, size, torch.float32)
    with pytest.raises(ValueError, match="at most 64 drafts"):
        process_logits(torch.zeros(1, 66, V, device=device), s, [[0] * 65])


def test_state(device):
    """Counts by token, invalid ids, lengths, views of one sequence, reset."""
    B, V = 3, 97
    s = LogitsState.zeros(B, V, device)
    tokens = torch.tensor([[5, 5, 96, -1, 97], [0, 1, 2, 3, 4], [5, 5, 5, 5, 5]], dtype=torch.int32, device=device)
    lens = torch.tensor([5, 0, 4], dtype=torch.int32, device=device)
    s.add(tokens, lens)
    s.add(tokens[:, 1:3], prompt=True)
    s.add(tokens[:, ::2])  # a stride
    s.add(torch.tensor([[2 ** 32 + 5], [-2 ** 32 + 5], [V]], device=device))  # 64 bits: still outside
    want = torch.zeros(B, V, dtype=torch.int64)
    want[0, 5], want[0, 96], want[2, 5] = 2 + 1, 1 + 1, 4 + 3
    want[1, 0] += 1
    want[1, 2] += 1
    want[1, 4] += 1
    for b, ts in enumerate(([5, 96], [1, 2], [5, 5])):
        for t in set(ts):
            want[b, t] -= 2 ** 31
    assert torch.equal(s.counts.cpu().long(), want)
    known = (s.known.cpu()[:, :, None] >> torch.arange(32) & 1).view(B, -1)[:, :V].bool()
    assert torch.equal(known, want != 0)
    before = s.counts.clone()
    one = s[1]
    one.set_bias([2, 90, 2], [1.0, 2.0, -3.0])
    one.set_penalties(2.0, presence=0.5)
    assert s.bias[1, 2] == -3 and s.bias[1, 90] == 2 and s.bias[0].abs().sum() == 0
    assert s.penalties.tolist() == [[1, 0, 0], [2, 0.5, 0], [1, 0, 0]]
    one.reset()
    assert s.counts[1].abs().sum() == 0 and s.bias[1].abs().sum() == 0 and s.known[1].abs().sum() == 0
    assert s.penalties[1].tolist() == [1, 0, 0]
    assert torch.equal(s.counts[0], before[0]) and torch.equal(s.counts[2], before[2])
    s[-1].reset()
    s[0:1].reset()
    assert s.counts.abs().sum() == 0 and s.known.abs().sum() == 0


def test_many_equal_tokens(device):
    """Every lane counts one token."""
    V = 1000
    s = LogitsState.zeros(2, V, device)
    s.add(torch.full((2, 70001), 3, dtype=torch.int32, device=device))
    s.add(torch.full((2, 70001), 3, dtype=torch.int32, device=device), prompt=True)
    assert s.counts[:, 3].tolist() == [70001 - 2 ** 31] * 2 and (s.counts != 0).sum() == 2


def test_bias_4096_with_duplicates(device):
    V = 5000
    s = LogitsState.zeros(1, V, device)
    ids = torch.randint(0, 1000, (1, 4096), generator=torch.Generator().manual_seed(1)).int()
    values = torch.randn(1, 4096)
    s.set_bias(ids.to(device), values.to(device))
    want = torch.zeros(V)
    for i, v in zip(ids[0].tolist(), values[0].tolist()):
        want[i] = v
    assert torch.equal(s.bias[0].cpu(), want)
    s.set_bias([1], [-torch.inf])
    out = process_logits(torch.ones(1, 1, V, device=device), s)
    assert out[0, 0, 1] == -torch.inf


def test_captured(device):
    """A graph of reset, counting, processing and accept, replayed on other inputs."""
    B, N, V = 2, 4, 3001
    logits, prompt, made, ids, values, pen, draft, allowed = _case(B, N, V, torch.bfloat16, seed=21)
    lg, d, m = logits.to(device), torch.tensor(draft, dtype=torch.int32).to(device), words(allowed).to(device)
    tokens = torch.tensor([[1, 2, 3], [4, 5, 5]], dtype=torch.int32, device=device)
    s = LogitsState.zeros(B, V, device)
    eager = LogitsState.zeros(B, V, device)

    def step(state):
        state.add(tokens)
        out = process_logits(lg, state, d, mask=m)
        return (out, *greedy_accept(lg, d, state=state, mask=m))

    for st in (s, eager):
        st.set_penalties(1.4, 0.3, 0.2)
    step(eager)
    eager.reset()
    eager.set_penalties(1.4, 0.3, 0.2)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = step(s)
    for k in range(4):
        lg.copy_((logits.float() * (1 + k)).bfloat16())
        tokens.add_(k)
        graph.replay()
        for a, b in zip(outs, step(eager)):
            assert torch.equal(a, b)
        torch.cuda.synchronize()
    assert torch.equal(s.counts, eager.counts)


def test_other_stream(device):
    """The ops go to the current stream."""
    V = 151936
    lg = torch.randn(1, 16, V, device=device)
    s = LogitsState.zeros(1, V, device)
    s.set_penalties(1.5)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(20):
            lg.add_(1)
        s.add(torch.arange(1000, dtype=torch.int32, device=device)[None])
        out = process_logits(lg, s)
        post = greedy_accept(lg, state=s)[0]
    side.synchronize()
    assert torch.equal(out.argmax(-1).int(), post)
    assert torch.equal(out[:, :, 1000:], lg[:, :, 1000:])


def test_refusals(device):
    s = LogitsState.zeros(2, 64, device)
    lg = torch.zeros(2, 3, 64, device=device)
    for bad in (lambda: process_logits(lg[:1], s), lambda: process_logits(lg[:, :, :63], s),
                lambda: process_logits(lg, s, out=lg[:, :2]), lambda: process_logits(lg[0, 0]),
                lambda: process_logits(lg, s, mask=torch.zeros(2, 3, 3, dtype=torch.int32, device=device)),
                lambda: process_logits(lg, s, [[1]]),
                lambda: process_logits(lg, s, out=torch.zeros(1, 3, 64, device=device).expand(2, 3, 64)),
                lambda: process_logits(lg[:, :2], s, out=lg[:, 1:]),
                lambda: greedy_accept(lg, state=s, mask=torch.zeros(2, 2, 2, dtype=torch.int32, device=device)),
                lambda: s.set_bias([[1, 2]], [[1.0, 2.0]]), lambda: s.set_bias([1], [1.0, 2.0]),
                lambda: s.set_bias([0] * 4097, [0.0] * 4097), lambda: s.set_penalties(repetition=0.0),
                lambda: s.set_penalties(presence=[1.0, 2.0, 3.0]), lambda: s.add(torch.zeros(3, 1, dtype=torch.int32)),
                lambda: s.add([[1], [2]], torch.zeros(1, dtype=torch.int32, device=device)), lambda: s[0:2:2],
                lambda: LogitsState(s.counts, s.known[:1], s.bias, s.penalties)):
        with pytest.raises(ValueError):
            bad()
    for bad in (lambda: process_logits(lg.double(), s), lambda: process_logits(lg, 5),
                lambda: process_logits(lg, s, mask=torch.zeros(2, 3, 2, device=device)), lambda: s.add([[1.5], [2.0]])):
        with pytest.raises(TypeError):
            bad()
    with pytest.raises(IndexError):
        s[2]
    assert process_logits(lg[:0], LogitsState.zeros(0, 64, device)).shape == (0, 3, 64)
