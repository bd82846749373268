"""Penalties, biases and a grammar in the decode loop: every verify mode takes the tokens
that one-by-one decoding under the definition takes, whatever the drafts were.

The target is a host model whose logits are a function of the tokens so far (a seeded row
for each state of its hash), on the device; the reference processes them in fp32 by the
definition, where the greedy tokens have to be equal."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import DFlashGenerator, LogitsShaping
from dflash_mlx import runtime as rt
from tests.logits_util import argmax_lowest, counts_of, processed, words
from tests.test_runtime_loop import FakeModel, KVCache, _advance

pytestmark = pytest.mark.gpu

V, BS, N_NEW = 61, 8, 40
PROMPT = [5, 17, 42, 8, 5, 5, 23, 11]
BIAS = {3: 4.0, 7: -30.0, 60: 2.5}


def _row(h: int) -> torch.Tensor:
    return 3 * torch.randn(V, generator=torch.Generator().manual_seed(int(h) % (2 ** 31)))


class Target(FakeModel):
    """Hidden states are the hash; negative ones stand for a token (the drafter's)."""

    def __init__(self, device):
        super().__init__()
        self.device = device

    def forward_dflash(self, inputs, cache, layer_ids, return_rollback_records=False):
        out = super().forward_dflash(inputs, cache, layer_ids, return_rollback_records)
        return (out[1][..., :1],) + tuple(out[1:])

    def lm_head_logits(self, hidden):
        rows = [_row(h) if h >= 0 else 50 * torch.nn.functional.one_hot(torch.tensor(int(-h) - 1), V).float()
                for h in hidden.reshape(-1).tolist()]
        return torch.stack(rows).view(*hidden.shape[:-1], V).to(self.device)

    def lm_head_argmax(self, hidden):
        return self.lm_head_logits(hidden).argmax(-1).int()

    def embed_tokens(self, tokens):
        return torch.as_tensor(tokens).double()[..., None]


class Drafter:
    """Proposes the reference's continuation, wrong at plan[k] of block k."""

    mask_token_id, target_layer_ids, block_size = 0, [1], BS

    def __init__(self, full, plan):
        self.full, self.plan, self.calls, self.at = full, plan, 0, None

    def make_cache(self):
        return [KVCache()]

    def __call__(self, noise_embedding, target_hidden, cache=None):
        self.at = len(PROMPT) if self.at is None else self.at + target_hidden.shape[1]
        toks = [self.full[self.at + i] for i in range(noise_embedding.shape[1])]
        wrong = self.plan[self.calls % len(self.plan)]
        if wrong is not None:
            toks[wrong] = (toks[wrong] + 1) % V
        self.calls += 1
        return torch.tensor([[[-float(t) - 1] for t in toks]], dtype=torch.float64)


def _grammar(tokens):
    """After an even number of tokens an even token, after a token below 5 anything."""
    if tokens[-1] < 5:
        return None
    allowed = torch.zeros(V, dtype=torch.bool)
    allowed[len(tokens) % 2::2] = True
    return words(allowed)


def _reference(penalties, bias, grammar, n):
    """Token by token by the definition."""
    h = 0
    for t in PROMPT:
        h = _advance(h, t)
    dense = torch.zeros(1, V)
    for t, v in bias.items():
        dense[0, t] = v
    out = []
    for _ in range(n):
        made, prompt = counts_of([PROMPT], [out], V)
        w = grammar(PROMPT + out) if grammar else None
        allowed = None if w is None else (w[:, None] >> torch.arange(32) & 1).bool().view(1, 1, -1)[..., :V]
        row, _ = processed(_row(h).view(1, 1, V), made, prompt, dense, torch.tensor([penalties]), None, allowed,
                           torch.float32)
        out.append(int(argmax_lowest(row)[0, 0]))
        h = _advance(h, out[-1])
    return out


CASES = {"penalties": ((1.4, 0.6, 0.3), {}, None), "biases": ((1.0, 0.0, 0.0), BIAS, None),
         "grammar": ((1.0, 0.0, 0.0), {}, _grammar), "all": ((1.3, 0.5, 0.2), BIAS, _grammar)}


@pytest.mark.parametrize("mode", rt.VERIFY_MODES)
@pytest.mark.parametrize("case", CASES)
def test_every_mode_decodes_as_one_by_one(device, case, mode, monkeypatch):
    penalties, bias, grammar = CASES[case]
    want = _reference(penalties, bias, grammar, N_NEW + 2 * BS)
    plain = _reference((1.0, 0.0, 0.0), {}, None, N_NEW)
    assert want[:N_NEW] != plain
    runs, begin = [], LogitsShaping.begin
    monkeypatch.setattr(LogitsShaping, "begin", lambda s, p: runs.append(begin(s, p)) or runs[-1])
    shaping = LogitsShaping(*penalties, logit_bias=bias, token_mask=grammar)
    drafter = Drafter(PROMPT + want, [3, None, 1, 5, 7])
    res = DFlashGenerator(Target(device), drafter).generate_from_tokens(
        torch.tensor(PROMPT), max_new_tokens=N_NEW, verify_mode=mode, verify_chunk_size=3, shaping=shaping)
    assert res.generated_tokens == want[:N_NEW]
    assert max(res.metrics["acceptance_lengths"]) == BS  # right drafts pass
    shaping, = runs
    made, prompt = counts_of([PROMPT], [shaping.tokens[len(PROMPT):]], V)
    if shaping._waiting == []:
        counts = shaping.state.counts.cpu()[0].long()
        assert torch.equal(torch.where(counts < 0, counts + 2 ** 31, counts), made[0])
        assert torch.equal(counts < 0, prompt[0])


def test_a_shaping_that_asks_for_nothing_changes_nothing(device):
    want = _reference((1.0, 0.0, 0.0), {}, None, N_NEW + 2 * BS)
    for shaping in (None, LogitsShaping()):
        res = DFlashGenerator(Target(device), Drafter(PROMPT + want, [2])).generate_from_tokens(
            torch.tensor(PROMPT), max_new_tokens=N_NEW, shaping=shaping)
        assert res.generated_tokens == want[:N_NEW]


def test_a_shaping_is_used_again_and_streams(device):
    want = _reference((1.4, 0.6, 0.3), {}, None, N_NEW + 2 * BS)
    shaping = LogitsShaping(1.4, 0.6, 0.3)
    for _ in range(2):
        events = list(DFlashGenerator(Target(device), Drafter(PROMPT + want, [4, None])).stream_from_tokens(
            torch.tensor(PROMPT), max_new_tokens=N_NEW, shaping=shaping))
        assert [t for e in events for t in e.token_ids] == want[:N_NEW]


def test_two_generations_at_once(device):
    want = _reference((1.4, 0.6, 0.3), {}, None, N_NEW + 2 * BS)
    shaping = LogitsShaping(1.4, 0.6, 0.3)
    streams = [DFlashGenerator(Target(device), Drafter(PROMPT + want, plan)).stream_from_tokens(
        torch.tensor(PROMPT), max_new_tokens=N_NEW, shaping=shaping) for plan in ([4, None], [1, 6])]
    got = [[], []]
    live = [0, 1]
    while live:  # an event of each in turn
        for i in list(live):
            event = next(streams[i], None)
            if event is None:
                live.remove(i)
            else:
                got[i] += event.token_ids
    assert got == [want[:N_NEW]] * 2


@pytest.mark.parametrize("bad", [torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int64),
                                 torch.zeros(1, 2, dtype=torch.int32)])
def test_a_grammar_of_another_form_is_refused(device, bad):
    with pytest.raises(ValueError, match="token_mask"):
        DFlashGenerator(Target(device), Drafter(PROMPT + [1] * 60, [None])).generate_from_tokens(
            torch.tensor(PROMPT), max_new_tokens=4, shaping=LogitsShaping(token_mask=lambda t: bad))


def test_sampling_keeps_to_the_grammar(device):
    torch.manual_seed(0)
    shaping = LogitsShaping(1.2, token_mask=_grammar)
    filler = [1] * (N_NEW + 3 * BS)
    res = DFlashGenerator(Target(device), Drafter(PROMPT + filler, [None])).generate_from_tokens(
        torch.tensor(PROMPT), max_new_tokens=N_NEW, temperature=0.7, shaping=shaping)
    toks = PROMPT + res.generated_tokens
    for i in range(len(PROMPT), len(toks)):
        assert toks[i - 1] < 5 or toks[i] % 2 == i % 2


def test_refusals():
    with pytest.raises(ValueError):
        LogitsShaping(repetition_penalty=0.0)
    with pytest.raises(ValueError):
        LogitsShaping(logit_bias={i: 1.0 for i in range(4097)})
