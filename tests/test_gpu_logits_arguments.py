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


def test_penalties_of_the_host_are_looked_at(device):
    s = LogitsState.zeros(2, 50, device)
    for bad in (0.0, -1.0, float("nan"), [1.0, 0.0], torch.tensor([1.0, 0.0]), torch.tensor(-2.0), torch.tensor(float("nan"))):
        with pytest.raises(ValueError, match="positive"):
            s.set_penalties(bad)
    assert s.penalties.tolist() == [[1.0, 0.0, 0.0]] * 2
    s.set_penalties(torch.tensor([1.5, 2.0]), torch.tensor(-0.5), [0.25, 0.5])
    assert s.penalties.tolist() == [[1.5, -0.5, 0.25], [2.0, -0.5, 0.5]]
    s.set_penalties(torch.tensor([2.0, 3.0], device=device))
    assert s.penalties[:, 0].tolist() == [2.0, 3.0]
