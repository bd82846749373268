"""Logits processed in place: what nothing changes keeps its value, and its bytes where its eight
holds nothing that changes."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import LogitsState, process_logits
from tests.logits_util import words

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,ints,nan", [(torch.float32, torch.int32, 0x7F800123), (torch.bfloat16, torch.int16, 0x7F81),
                                            (torch.float16, torch.int16, 0x7C05)])
@pytest.mark.parametrize("B,N,V", [(1, 3, 1003), (4, 16, 20011)])
def test_untouched_entries(device, dtype, ints, nan, B, N, V):
    g = torch.Generator().manual_seed(V)
    logits = torch.randn(B, N, V, generator=g).to(dtype)
    logits.view(ints).masked_fill_(torch.rand(B, N, V, generator=g) < 0.2, nan)  # a NaN's other bits go on the way
    allowed = torch.rand(B, N, V, generator=g) > 0.03
    s = LogitsState.zeros(B, V, device)
    s.set_penalties(1.5, 0.5, 0.25)
    tokens = torch.randint(0, V, (B, V // 40), generator=g).int()
    draft = torch.randint(0, V, (B, N - 1), generator=g).int()
    s.add(tokens)
    lg = logits.to(device)
    want = process_logits(lg, s, draft.to(device), mask=words(allowed).to(device)).cpu()
    process_logits(lg, s, draft.to(device), mask=words(allowed).to(device), out=lg)
    got = lg.cpu()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(nan=1), want.nan_to_num(nan=1))
    known = torch.zeros(B, N, V, dtype=torch.bool)
    known.scatter_(2, tokens.long()[:, None].expand(B, N, -1), True)
    for i in range(1, N):
        known[:, i].scatter_(1, draft[:, :i].long(), True)
    change = known | ~allowed
    pad = -V % 8
    eights = torch.nn.functional.pad(change, (0, pad)).view(B, N, -1, 8).any(-1).repeat_interleave(8, -1)[..., :V]
    assert 0 < eights.sum() < eights.numel() / 1.2
    assert torch.equal(got.view(ints)[~eights], logits.view(ints)[~eights])
    keep = ~change
    assert torch.equal(got[keep].nan_to_num(nan=1), logits[keep].nan_to_num(nan=1))
