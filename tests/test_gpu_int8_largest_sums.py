"""Sums of the largest magnitude that codes from elsewhere can make: exact, or refused."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import matmul_i8, pack_weight_i8

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M", [1, 16, 33, 100, 300])
def test_codes_of_minus_128(device, M):
    """2^14 K stays in 32 bits below the largest K; scales of one power of two keep it exact."""
    for K, code in ((131071, -128), (131072, -127)):
        x = torch.full((M, K), -128, dtype=torch.int8, device=device)
        w = torch.full((20, K), code, dtype=torch.int8, device=device)
        w[3] = 127
        scale = torch.full((M,), 2.0 ** -7, device=device)
        out = matmul_i8(x, scale, pack_weight_i8(w, torch.full((20,), 0.5, device=device)), out_dtype=torch.float32)
        want = torch.full((M, 20), 128 * -code * K, dtype=torch.float64)
        want[:, 3] = -128 * 127 * K
        assert torch.equal(out.cpu(), (want.float() * 2.0 ** -8))


def test_a_sum_that_32_bits_do_not_hold_is_refused(device):
    w = torch.full((4, 131072), -127, dtype=torch.int8, device=device)
    scale = torch.ones(4, device=device)
    pack_weight_i8(w, scale)
    w[2, 70000] = -128
    with pytest.raises(ValueError, match="-127"):
        pack_weight_i8(w, scale)
    pack_weight_i8(w[:, 1:], scale)
