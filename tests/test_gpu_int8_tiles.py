"""The products' tile kernels, each at shapes well inside its own range, with workgroups of one
tile and of several, few and many turns of their slots, in every output type, against the definition
in 64 bits (tolerances as in the tests of the projections).  That the shapes take the kernel
that they stand for is read off a trace."""
from __future__ import annotations

import pytest
import torch

from dflash_mlx import matmul_i8, pack_weight_i8, quantize_rows_i8
from tests.test_gpu_int8 import check, product, rows, weight

pytestmark = pytest.mark.gpu

OUT = (torch.bfloat16, torch.float16, torch.float32)
WIDE, NARROW = "256 x 256", "128 x 128"
# rows, channels, features, gated, tile: whole tiles and ends of them in every direction
CASES = [
    (2050, 4100, 1000, False, WIDE),   # 153 tiles: one a workgroup
    (2050, 4100, 1000, True, WIDE),
    (4096, 4096, 1024, True, WIDE),    # nothing but whole tiles
    (5000, 6001, 320, False, WIDE),    # 480: two for most
    (4100, 18000, 200, True, WIDE),    # 1207, four k-steps each
    (3000, 20002, 391, True, WIDE),
    (3000, 20003, 391, False, WIDE),
    (96, 70001, 640, False, NARROW),   # 547 on 512 places
    (96, 140002, 640, True, NARROW),   # 1094
    (1030, 16401, 200, False, NARROW),
    (2050, 9002, 640, True, NARROW),
    (1024, 2304, 640, True, NARROW),
]


def _tile_of(run):
    """The tile kernel that `run` launches, by its template's channel waves."""
    from torch.profiler import ProfilerActivity, profile

    with profile(activities=[ProfilerActivity.CUDA, ProfilerActivity.CPU]) as prof:
        run()
        torch.cuda.synchronize()
    names = [e.key for e in prof.key_averages() if "prompt_i8_kernel" in e.key]
    print("[int8 tiles]", names, flush=True)
    if not names:
        pytest.skip("no kernel names in this trace")
    (name,) = names
    return WIDE if "Shape<4" in name or "ShapeILi4" in name else NARROW


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:3])) + ("-gated" if c[3] else ""))
def test_tiles(device, case):
    M, N, K, gated, tile = case
    x = rows(M, K, torch.bfloat16, seed=M + N + K)
    w_codes, w_scale = weight(N, K, seed=N + K)
    w = pack_weight_i8(w_codes.to(device), w_scale.to(device), gated=gated)
    codes, scale = quantize_rows_i8(x.to(device))
    want, gate = product(codes.cpu(), scale.cpu(), w_codes, w_scale, gated)
    for dtype in OUT:
        out = torch.full((M, w.cols + 8), 7.0, dtype=dtype, device=device)
        view = out[:, 4:4 + w.cols]
        matmul_i8(codes, scale, w, out=view)
        check(view, want, gate if gated else None)
        assert (out[:, :4] == 7).all() and (out[:, 4 + w.cols:] == 7).all()
        # again, beside other work: the same bits
        again = [matmul_i8(codes, scale, w, out_dtype=dtype) for _ in range(3)]
        assert all(torch.equal(a, view) for a in again)


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(map(str, c[:3])) + ("-gated" if c[3] else ""))
def test_the_shapes_take_their_tiles(device, case):
    M, N, K, gated, tile = case
    if torch.cuda.get_device_properties(device).multi_processor_count != 256:
        pytest.skip("the shapes are chosen for 256 compute units")
    w = pack_weight_i8(torch.ones(N, K, dtype=torch.int8, device=device), torch.ones(N, device=device), gated=gated)
    codes, scale = torch.ones(M, -(-K // 16) * 16, dtype=torch.int8, device=device)[:, :K], torch.ones(M, device=device)
    assert _tile_of(lambda: matmul_i8(codes, scale, w)) == tile
