"""Arguments of the logits operators that look like others."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import LogitsState, greedy_accept, process_logits

pytestmark = pytest.mark.gpu


def test_drafts_of_64_bits(device):
    """An id that 32 bits would wrap is outside the vocabulary, and agrees with no token."""
    V = 50
    s = LogitsState.zeros(1, V, device)
    s.set_penalties(1.0, 5.0, 1.0)
    logits = torch.zeros(1, 4, V, device=device)
    logits[..., 7] = 1.0
    for bad in (2 ** 32 + 7, -2 ** 32 + 7, 2 ** 63 - 1, -2 ** 63, 2 ** 31 + 7):
        draft = torch.tensor([[bad, 9, 7]], device=device)
        want = process_logits(logits, s, torch.tensor([[-1, 9, 7]], dtype=torch.int32, device=device))
        assert torch.equal(process_logits(logits, s, draft), want)
        post, matched, bonus = greedy_accept(logits, draft, state=s)
        assert post[0, 0] == 7 and matched.item() == 0 and bonus.item() == 7
    draft = torch.tensor([[7, 0, 0]], device=device)  # the others count as ever
    assert greedy_accept(logits, draft, state=s)[1].item() == 2
