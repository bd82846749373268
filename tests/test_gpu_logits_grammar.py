"""A grammar is asked about nothing but what may be taken: drafts are proposed without it, so
a block may hold prefixes that it has ruled out, about which it need not know anything."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from dflash_mlx import DFlashGenerator, LogitsShaping
from dflash_mlx import runtime as rt
from tests.logits_util import words
from tests.test_gpu_logits_generate import N_NEW, PROMPT, BS, Drafter, Target, V, _grammar, _reference

SAMPLED = [m for m in rt.VERIFY_MODES if m != "parallel-greedy-argmax"]


def _allows(w, token):
    return w is None or bool(w[token // 32] >> token % 32 & 1)


class Strict:
    """A grammar that ends the program when asked about a text that it does not allow.  A
    text of which nothing may follow goes on with token 0."""

    def __init__(self, grammar):
        self.grammar, self.asked = grammar, 0

    def __call__(self, tokens):
        for i in range(len(PROMPT), len(tokens)):
            w = self.grammar(tokens[:i])
            dead = w is not None and not bool(w.any())
            assert tokens[i] == 0 if dead else _allows(w, tokens[i]), f"asked about {tokens[len(PROMPT):]}"
        self.asked += 1
        return self.grammar(tokens)


def _with_dead_ends(tokens):
    """_grammar, but nothing may follow a token of 40 to 43."""
    return torch.zeros(-(-V // 32), dtype=torch.int32) if 40 <= tokens[-1] < 44 else _grammar(tokens)


GRAMMARS = {"alternating": _grammar, "dead ends": _with_dead_ends}


@pytest.mark.gpu
@pytest.mark.parametrize("mode", rt.VERIFY_MODES)
@pytest.mark.parametrize("grammar", GRAMMARS)
def test_greedy(device, grammar, mode):
    """Drafts that are right for a while and then mostly forbidden."""
    want = _reference((1.2, 0.3, 0.1), {}, GRAMMARS[grammar], N_NEW + 2 * BS)
    strict = Strict(GRAMMARS[grammar])
    res = DFlashGenerator(Target(device), Drafter(PROMPT + want, [3, None, 1, 5, 7])).generate_from_tokens(
        torch.tensor(PROMPT), max_new_tokens=N_NEW, verify_mode=mode, verify_chunk_size=3,
        shaping=LogitsShaping(1.2, 0.3, 0.1, token_mask=strict))
    assert res.generated_tokens == want[:N_NEW] and strict.asked >= N_NEW
    if grammar == "dead ends":
        assert any(40 <= t < 44 for t in want[:N_NEW - 1])
    assert max(res.metrics["acceptance_lengths"]) == BS


@pytest.mark.gpu
@pytest.mark.parametrize("mode", SAMPLED)
@pytest.mark.parametrize("grammar", GRAMMARS)
def test_sampled(device, grammar, mode):
    """Near the greedy tokens, so that drafts pass, and far from them."""
    want = _reference((1.0, 0.0, 0.0), {}, GRAMMARS[grammar], N_NEW + 2 * BS)
    for temperature in (0.02, 1.5):
        torch.manual_seed(1)
        strict = Strict(GRAMMARS[grammar])
        res = DFlashGenerator(Target(device), Drafter(PROMPT + want, [3, None, 1, 5, 7])).generate_from_tokens(
            torch.tensor(PROMPT), max_new_tokens=N_NEW, temperature=temperature, verify_mode=mode, verify_chunk_size=3,
            shaping=LogitsShaping(token_mask=strict))
        assert len(res.generated_tokens) == N_NEW
        strict(PROMPT + res.generated_tokens)  # every token is one that may follow


@pytest.mark.gpu
@pytest.mark.parametrize("mode", rt.VERIFY_MODES)
def test_long_blocks(device, mode):
    """A state counts 64 drafts; a grammar alone needs no state."""
    block = 70
    want = _reference((1.0, 0.0, 0.0), {}, _grammar, 100 + 2 * block)

    def drafter():
        d = Drafter(PROMPT + want, [None, 66])
        d.block_size = block
        return d

    args = dict(max_new_tokens=100, verify_mode=mode, verify_chunk_size=block)
    res = DFlashGenerator(Target(device), drafter()).generate_from_tokens(
        torch.tensor(PROMPT), shaping=LogitsShaping(token_mask=_grammar), **args)
    assert res.generated_tokens == want[:100] and max(res.metrics["acceptance_lengths"]) == block
    if mode not in ("stream", "chunked"):
        with pytest.raises(ValueError, match="at most 64 drafts"):
            DFlashGenerator(Target(device), drafter()).generate_from_tokens(
                torch.tensor(PROMPT), shaping=LogitsShaping(1.1, token_mask=_grammar), **args)


def test_rows_behind_a_forbidden_draft(monkeypatch):
    """The grammar is asked about the rows up to the first draft that it rules out (no GPU)."""
    state = SimpleNamespace(**dict.fromkeys(("counts", "known", "bias", "penalties"), torch.zeros(1)), add=lambda t: None)

    def ready(shaping, n, dev):
        shaping._extra = state
        return state

    monkeypatch.setattr(LogitsShaping, "_ready", ready)
    W = -(-V // 32)
    none = torch.zeros(W, dtype=torch.int32)
    even = words(torch.arange(V) % 2 == 0)

    def masks(grammar, drafts, n=4, before=()):
        asked = []
        shaping = LogitsShaping(1.5, token_mask=lambda t: asked.append(t) or grammar(t)).begin([7])
        mask = shaping.rows(n, V, "cpu", before, drafts)[1]
        assert mask.shape == (1, n, W) and mask.dtype is torch.int32
        return mask[0], asked

    m, asked = masks(lambda t: even, [2, 3, 4])
    assert asked == [[7], [7, 2]] and torch.equal(m[:2], even.expand(2, W)) and (m[2:] == -1).all()
    m, asked = masks(lambda t: even, [2, 4, 3], before=[8])
    assert asked == [[7, 8], [7, 8, 2], [7, 8, 2, 4]] and (m[3] == -1).all()
    m, asked = masks(lambda t: None, [1, 2, 3])
    assert len(asked) == 4 and (m == -1).all()
    # nothing may follow: the token taken is 0
    m, asked = masks(lambda t: none if len(t) == 2 else None, [5, 0, 9])
    assert asked == [[7], [7, 5], [7, 5, 0], [7, 5, 0, 9]] and (m[1] == 0).all()
    m, asked = masks(lambda t: none if len(t) == 2 else None, [5, 1, 9])
    assert asked == [[7], [7, 5]] and (m[1] == 0).all() and (m[2:] == -1).all()
    # drafts outside the vocabulary, and rows behind the last draft
    for out in (V, -1, 2 ** 31):
        m, asked = masks(lambda t: even, [2, out, 4])
        assert asked == [[7], [7, 2]]
    m, asked = masks(lambda t: even, [2, 4, 6], n=3)
    assert len(asked) == 3
