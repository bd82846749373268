"""kv_rewind_q8's bookkeeping on the CPU: a cache of one feature whose values are the
numbers of the tokens, through appends, rejected drafts and any chain of rewinds.  Before
every append at length L the tail has to hold the open block's tokens below L and, where
the append may quantise the block before it (L % 64 <= 16), all of that block's."""
from __future__ import annotations

import random

import pytest
import torch

from dflash_mlx import kv8

BLOCK, SLOTS, SMAX = kv8.BLOCK, kv8.SLOTS, 640


class Sequence:
    def __init__(self, monkeypatch):
        self.cache = object.__new__(kv8.QuantizedKVCache)
        self.cache.B, self.cache.Smax, self.cache.device = 1, SMAX, torch.device("cpu")
        self.cache.tail_k = torch.full((1, 1, SLOTS, 1), -1.0)
        self.cache.tail_vt = torch.full((1, 1, 1, SLOTS), -1.0)
        self.codes = torch.full((SMAX // BLOCK, BLOCK), -1.0)
        self.kept = torch.zeros(0)  # the committed tokens' numbers
        self.written = self.tokens = 0
        monkeypatch.setattr(kv8, "kv_read_q8", self._read)

    @property
    def length(self):
        return len(self.kept)

    def _read(self, cache, lens, count, *, start=0):
        L, blk = int(lens[0]), start // BLOCK
        assert start % BLOCK == 0 and count == BLOCK  # a length at which the block is read from its codes:
        assert blk < min(L, SMAX) // BLOCK and (L % BLOCK > 16 or blk < L // BLOCK - 1)
        x = self.codes[blk].clone().view(1, 1, BLOCK, 1)
        return x, x

    def _slots(self, lo, hi):
        p = torch.arange(lo, hi) % SLOTS
        assert torch.equal(self.cache.tail_k[0, 0, p, 0], self.cache.tail_vt[0, 0, 0, p])
        return self.cache.tail_k[0, 0, p, 0]

    def append(self, T, keep, prompt=False):
        L = self.length
        blk = L // BLOCK
        assert torch.equal(self._slots(blk * BLOCK, L), self.kept[blk * BLOCK:]), f"the open block at {L}"
        if blk and L % BLOCK <= 16:
            self.codes[blk - 1] = self._slots((blk - 1) * BLOCK, blk * BLOCK)
        if blk:
            assert torch.equal(self.codes[:blk].flatten(), self.kept[:blk * BLOCK]), f"codes at {L}"
        T = min(T, SMAX - L)
        new = self.tokens + 1.0 + torch.arange(T)
        self.tokens += T
        self.kept = torch.cat((self.kept, new[:keep]))
        lo = L
        if prompt:  # codes of what it completes; the tail takes the last block with codes and the open one
            done = self.length // BLOCK
            self.codes[blk:done] = self.kept[blk * BLOCK:done * BLOCK].view(-1, BLOCK)
            lo = max(L, (done - 1) * BLOCK)
        p = torch.arange(lo, L + T) % SLOTS
        self.cache.tail_k[0, 0, p, 0] = self.cache.tail_vt[0, 0, 0, p] = new[lo - L:]
        self.written = max(self.written, L + T)

    def rewind(self, length):
        self.written = kv8.kv_rewind_q8(self.cache, length, self.written)
        self.kept = self.kept[:length]


def test_two_rewinds_in_a_row(monkeypatch):
    s = Sequence(monkeypatch)
    for _ in range(8):
        s.append(16, 16)
    s.append(10, 0)  # rejected drafts at 128 .. 137, in the slots of 0 .. 9
    s.rewind(128)
    s.rewind(74)
    s.append(5, 5)


@pytest.mark.parametrize("n,length", [(448, 384), (448, 398), (448, 330), (128, 64), (450, 384), (447, 384)])
def test_a_rewind_after_a_prompt(monkeypatch, n, length):
    """One that ends a block leaves no earlier one in the tail."""
    s = Sequence(monkeypatch)
    s.append(n, n, prompt=True)
    s.rewind(length)
    s.append(5, 5)


@pytest.mark.parametrize("seed", range(20))
def test_any_chain_of_appends_and_rewinds(monkeypatch, seed):
    rng = random.Random(seed)
    s = Sequence(monkeypatch)
    again = False
    for _ in range(1500):
        if rng.random() < (0.4 if again else 0.97) and s.length + 16 <= SMAX:
            if rng.random() < 0.1:
                n = min(rng.randint(1, 200), SMAX - s.length)
                if rng.random() < 0.5:  # up to a block's end
                    n = max(1, (s.length + n) // BLOCK * BLOCK - s.length)
                s.append(n, n, prompt=True)
            else:
                T = rng.randint(1, 16)
                s.append(T, rng.choice([T, T, rng.randint(0, T)]))
            again = False
        else:
            length = rng.randint(max(0, s.length - 150), s.length)
            if rng.random() < 0.6:  # lengths at a block's end and up to 16 past it are the ones to go wrong
                length = length // BLOCK * BLOCK + rng.choice([0, 0, 1, 10, 16, 17])
            s.rewind(min(s.length, length))
            again = True
