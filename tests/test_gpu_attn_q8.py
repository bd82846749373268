"""Attention over the 8-bit key/value cache against the same cache in 64 bits.

The bound on an output's error is derived in tests/kv8_util.attention_error:
the weights' and the output's rounding to bf16."""
from __future__ import annotations

import pytest
import torch

from tests.kv8_util import BLOCK, D, DTYPES, SLOTS, attention_error, loaded, proj_rows, random_kv, raw

pytestmark = pytest.mark.gpu


def _case(device, dtype, T, Hq, Hkv, lens, Smax, seed, prompt, qstd=1.5, pad=16):
    """A cache holding lens + T positions, as after the rows' append."""
    B = len(lens)
    k, v = random_kv(B, Hkv, Smax, seed, spread=False)
    g = torch.Generator().manual_seed(seed + 1)
    k = (k.float() * (0.3 + torch.rand(B, Hkv, Smax // BLOCK, generator=g).repeat_interleave(BLOCK, 2)[..., None])).bfloat16()
    held = [min(max(L, 0) + (T if L >= 0 else 0), Smax) for L in lens]
    # complete blocks are quantised up to the committed length only
    cache, _ = loaded(device, k, v, held if prompt else [min(L, Smax) for L in lens], Smax, dtype, fill=0xFF)
    if not prompt:
        for b, L in enumerate(lens):
            if L >= 0:
                p = torch.arange(min(L, Smax), held[b])
                cache.tail_k[b, :, p % SLOTS] = k[b, :, p].to(device)
                cache.tail_vt[b, :, :, p % SLOTS] = v[b, :, p].transpose(1, 2).to(device)
    q = (qstd * torch.randn(B, T, Hq, D, generator=g)).bfloat16()
    proj = proj_rows(B, T, Hq, Hkv, seed + 2, pad)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=device)
    ends = [(n, (n if prompt else min(max(L, 0), Smax)) // BLOCK) for n, L in zip(held, lens)]
    return cache, lens_d, k, v, q, proj, ends


def _check(device, dtype, T, Hq, Hkv, lens, Smax, seed, prompt, scale=None, qstd=1.5):
    import dflash_mlx as dm

    cache, lens_d, k, v, q, proj, ends = _case(device, dtype, T, Hq, Hkv, lens, Smax, seed, prompt, qstd)
    before = raw(cache)
    attend = dm.attn_prefill_q8 if prompt else dm.attn_verify_q8
    got = attend(q.to(device), cache, lens_d, proj.to(device), scale=scale).cpu()
    assert all(torch.equal(a, b) for a, b in zip(before, raw(cache)))
    live = [b for b, L in enumerate(lens) if L >= 0]
    assert all((got[b] == 0).all() for b in range(len(lens)) if b not in live)
    pick = lambda x: [x[b] for b in live]  # noqa: E731
    worst = attention_error(got[live], q[live], pick(k), pick(v), proj[live], [min(L, Smax) for L in pick(lens)], pick(ends),
                            dtype, D ** -0.5 if scale is None else scale)
    print(f"[attn q8] {dtype} T={T} {Hq}:{Hkv} lens={lens} prompt={prompt}: {worst:.3f} of the bound", flush=True)
    assert worst <= 1.0


VERIFY = [
    # T, Hq, Hkv, lens, Smax
    (1, 4, 1, [0], 64),
    (1, 16, 4, [500], 576),
    (16, 16, 4, [0], 64),
    (16, 16, 4, [1000], 1024),
    (16, 4, 4, [63, 64, 65, 127, 128, 129], 192),
    (5, 8, 8, [300, 0, 1, 767], 832),
    (3, 12, 4, [200, 5000, 64], 5056),
    (16, 8, 4, [77, 129], 256),
    (4, 16, 1, [129, 40], 192),     # sixteen query heads on one key/value head
    (1, 64, 1, [200], 256),         # sixty-four
    (2, 5, 1, [90], 128),
    (1, 8, 2, list(range(0, 140)), 192),  # more sequences than lanes
    (7, 4, 2, [-1, 100, -5, 60], 128),    # two take no part
    (16, 4, 1, [56, 64], 64),             # the rows run over the cache's end
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,Hkv,lens,Smax", VERIFY)
def test_verify(device, dtype, T, Hq, Hkv, lens, Smax):
    _check(device, dtype, T, Hq, Hkv, lens, Smax, seed=T + Hq + len(lens), prompt=False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,Hkv,lens,Smax", [
    (16, 16, 4, [2000, 70, -1, 900, 0, 1300], 2048),  # many heads of 64 rows, in parts and whole
    (8, 8, 2, [1500] + [40] * 20 + [-1, 700], 1536),  # of 32 rows
    (16, 1, 1, [4000], 4032),                         # one head of 16 rows in few parts
    (16, 2, 2, [2500, 100], 2560),
    (1, 8, 4, [(37 * i) % 190 - (i % 50 == 7) * 500 for i in range(270)] + [1400], 1472),  # more heads than workgroups
    (2, 16, 4, [(53 * i) % 130 for i in range(256)] + [700, 1000], 1024),
    (5, 17, 17, [(29 * i) % 140 for i in range(64)], 192),
])
def test_verify_merges(device, dtype, T, Hq, Hkv, lens, Smax):
    _check(device, dtype, T, Hq, Hkv, lens, Smax, seed=T + Hq + len(lens), prompt=False)


PROMPT = [
    (1, 4, 1, [0], 64),
    (17, 16, 4, [0], 64),
    (37, 8, 4, [5], 128),
    (300, 16, 4, [130], 448),
    (200, 3, 1, [0, 60], 320),
    (64, 16, 4, [448], 512),
    (130, 4, 4, [70, 0, 1], 256),
    (100, 8, 1, [33], 192),     # eight query heads a key/value head: two groups of four
    (70, 5, 1, [10], 128),      # five: one by one
    (90, 6, 1, [64], 192),      # six: two groups of three
    (40, 4, 2, [-1, 30], 128),
    (80, 4, 2, [20, 64], 64),   # rows past the cache's end see all of it
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,Hkv,lens,Smax", PROMPT)
def test_prompt(device, dtype, T, Hq, Hkv, lens, Smax):
    _check(device, dtype, T, Hq, Hkv, lens, Smax, seed=T + Hq + len(lens), prompt=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,Hkv,lens,Smax", [
    (1, 4, 1, [3900], 4032),              # one row block: as many splits as turns allow
    (33, 16, 4, [2000, 130, -1, 0], 2112),  # sequences of many splits, of two, of one and none
    (600, 8, 4, [700], 1344),
    (70, 3, 1, [1900, 1980], 1984),
    (129, 4, 4, [1500], 1664),
])
def test_prompt_with_split_keys(device, dtype, T, Hq, Hkv, lens, Smax):
    import dflash_mlx as dm

    assert dm.attn_prefill_q8_workspace_bytes(len(lens), T, Hq, Hkv, Smax) > 0
    _check(device, dtype, T, Hq, Hkv, lens, Smax, seed=T + Hq + len(lens), prompt=True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_split_keys_that_are_not_finite(device, dtype):
    """An infinite value is in its rows whatever its split weighs, a NaN block in the
    rows of every split that joins it, and neither in other rows."""
    import dflash_mlx as dm

    T, Hq, Hkv, L = 40, 4, 2, 1100
    cache, lens_d, k, v, q, proj, ends = _case(device, dtype, T, Hq, Hkv, [L], 1216, 5, True)
    attend = lambda: dm.attn_prefill_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(T, Hq, D)  # noqa: E731
    clean = attend()
    cache.tail_vt[0, 1, 17, 1120 % SLOTS] = float("inf")
    cache.tail_k[0, 1, 1120 % SLOTS] = -8 * q[0, 25, 2].to(device)  # its weight in row 25 of head 2 underflows
    got = attend()
    assert got[20:, 2:, 17].isinf().sum() >= 1 and not torch.isfinite(got[20:, 2:, 17].float()).any()
    assert torch.equal(got[:20], clean[:20]) and torch.equal(got[:, :2], clean[:, :2])
    assert torch.isfinite(got[20:, 2:, :17].float()).all() and torch.isfinite(got[20:, 2:, 18:].float()).all()
    for t in (cache.tail_vt, cache.tail_k):
        t.nan_to_num_(posinf=0.5)
    cache.v_scale[0, 0, 2] = float("nan")
    assert attend()[:, :2].isnan().all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_split_prompt_captured_and_on_two_streams(device, dtype):
    import dflash_mlx as dm

    T, Hq, Hkv, lens = 50, 8, 2, [1500, 200]
    cache, lens_d, k, v, q, proj, ends = _case(device, dtype, T, Hq, Hkv, lens, 1600, 9, True)
    qd, pd = q.to(device), proj.to(device)
    attend = lambda: dm.attn_prefill_q8(qd, cache, lens_d, pd)  # noqa: E731
    want = attend()
    torch.cuda.synchronize()
    outs, streams = [], [torch.cuda.Stream(device) for _ in range(2)]
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            outs.append(attend())
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = attend()
    for _ in range(3):
        captured.zero_()
        graph.replay()
        assert torch.equal(attend(), want)
        torch.cuda.synchronize()
        assert torch.equal(captured, want)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prompt", [False, True])
@pytest.mark.parametrize("scale", [0.5, -0.1, 0.0])
def test_scales(device, dtype, prompt, scale):
    _check(device, dtype, 9, 8, 2, [150, 64], 256, seed=4, prompt=prompt, scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prompt", [False, True])
def test_peaked_scores(device, dtype, prompt):
    """Queries of std 8: a row's weight sits on a few keys, the maximum moves often."""
    _check(device, dtype, 16, 4, 2, [700], 768, seed=6, prompt=prompt, qstd=8.0)


@pytest.mark.parametrize("dtype", DTYPES)
def test_value_scales_of_every_size(device, dtype):
    """Blocks whose values differ by 2^60: the output follows the largest, the
    sum of weights counts all."""
    import dflash_mlx as dm

    cache, lens_d, k, v, q, proj, ends = _case(device, dtype, 4, 4, 2, [400], 448, 8, False)
    mag = torch.tensor([1.0, 2.0 ** -60, 2.0 ** 20, 1.0, 2.0 ** 40, 2.0 ** -30, 1.0]).repeat_interleave(BLOCK)
    v = (v.float() * mag[:, None]).bfloat16()
    dm.kv_load_q8(k.to(device), v.to(device), lens_d, cache)
    p = torch.arange(400, 404)
    cache.tail_k[0, :, p % SLOTS] = k[0, :, p].to(device)
    cache.tail_vt[0, :, :, p % SLOTS] = v[0, :, p].transpose(1, 2).to(device)
    got = dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device)).cpu()
    assert attention_error(got, q, k, v, proj, [400], ends, dtype, D ** -0.5) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,rep,prompt", [(2, 1, False), (16, 2, False), (16, 4, False), (40, 2, True)])
@pytest.mark.parametrize("large", [2.0 ** 20, 2.0 ** 110])
def test_zero_values_beside_large_ones(device, dtype, T, rep, prompt, large):
    """One block's values are large, all others zero (their scale is the least there is)
    or, beside the largest, ordinary: the sum of weights counts every block."""
    import dflash_mlx as dm

    L, Smax = 1000 if prompt else 1040, 1088
    cache, lens_d, k, v, q, proj, ends = _case(device, dtype, T, 2 * rep, 2, [L], Smax, 8, prompt, qstd=0.5)
    held = ends[0][0]
    v[:, :, 64:128] = (v[:, :, 64:128].float() * large).bfloat16()
    if large < 2.0 ** 100:
        v[:, :, :64] = 0
        v[:, :, 128:] = 0
    dm.kv_load_q8(k.to(device), v.to(device), torch.tensor([held if prompt else L], dtype=torch.int32, device=device), cache)
    p = torch.arange(L // BLOCK * BLOCK if not prompt else held // BLOCK * BLOCK, held)
    cache.tail_k[0, :, p % SLOTS] = k[0, :, p].to(device)
    cache.tail_vt[0, :, :, p % SLOTS] = v[0, :, p].transpose(1, 2).to(device)
    attend = dm.attn_prefill_q8 if prompt else dm.attn_verify_q8
    got = attend(q.to(device), cache, lens_d, proj.to(device)).cpu()
    assert attention_error(got, q, k, v, proj, [L], ends, dtype, D ** -0.5) <= 1.0


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_values_that_are_not_finite(device, dtype, bad):
    """A draft token's value that is not finite is seen by its own row and the
    later ones, in its feature alone; key NaNs by all features of those rows."""
    import dflash_mlx as dm

    T, Hq, Hkv, L = 6, 4, 2, 130
    cache, lens_d, k, v, q, proj, ends = _case(device, dtype, T, Hq, Hkv, [L], 192, 3, False)
    clean = dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(T, Hq, D)
    cache.tail_vt[0, 1, 17, (L + 3) % SLOTS] = bad
    got = dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(T, Hq, D)
    hit = torch.zeros(T, Hq, D, dtype=torch.bool)
    hit[3:, 2:, 17] = True  # key/value head 1: query heads 2 and 3
    assert not torch.isfinite(got[hit].float()).any()
    assert torch.equal(got[~hit], clean[~hit])
    cache.tail_vt[0, 1, 17, (L + 3) % SLOTS] = 0.5
    cache.tail_k[0, 0, (L + 4) % SLOTS, 5] = float("nan")
    got = dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(T, Hq, D)
    assert got[4:, :2].isnan().all() and torch.isfinite(got[:4].float()).all() and torch.isfinite(got[4:, 2:].float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompt_values_that_are_not_finite(device, dtype):
    """In a prompt: the last partial block's by feature, a quantised block's as NaN
    of the whole block, and neither by earlier rows."""
    import dflash_mlx as dm

    T, Hq, Hkv, L = 150, 4, 2, 0
    cache, lens_d, k, v, q, proj, ends = _case(device, dtype, T, Hq, Hkv, [L], 192, 3, True)
    clean = dm.attn_prefill_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(T, Hq, D)
    cache.tail_vt[0, 1, 17, 140 % SLOTS] = float("inf")
    got = dm.attn_prefill_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(T, Hq, D)
    hit = torch.zeros(T, Hq, D, dtype=torch.bool)
    hit[140:, 2:, 17] = True
    assert not torch.isfinite(got[hit].float()).any()
    assert torch.equal(got[~hit], clean[~hit])
    cache.tail_vt[0, 1, 17, 140 % SLOTS] = 0.5
    for scales in (cache.k_scale, cache.v_scale):
        good = scales[0, 0, 1].clone()
        scales[0, 0, 1] = float("nan")  # positions 64 .. 127 of key/value head 0
        got = dm.attn_prefill_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(T, Hq, D)
        scales[0, 0, 1] = good
        assert got[64:, :2].isnan().all()
        assert torch.equal(got[:64], clean[:64])
        assert torch.isfinite(got[64:, 2:].float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("L", [10, 40, 1])
def test_prompt_rows_before_a_block_that_reads_as_nan(device, dtype, L):
    """Rows of one tile on both sides of the block's first position."""
    import dflash_mlx as dm

    T, Hq, Hkv = 150, 4, 2
    cache, lens_d, k, v, q, proj, ends = _case(device, dtype, T, Hq, Hkv, [L], 192, 3, True)
    attend = lambda: dm.attn_prefill_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(T, Hq, D)  # noqa: E731
    clean = attend()
    for scales in (cache.k_scale, cache.v_scale):
        good = scales[0, 0, 1].clone()
        scales[0, 0, 1] = float("nan")  # positions 64 .. 127 of key/value head 0
        got = attend()
        scales[0, 0, 1] = good
        assert got[64 - L:, :2].isnan().all()
        assert torch.equal(got[:64 - L], clean[:64 - L]) and torch.equal(got[:, 2:], clean[:, 2:])


@pytest.mark.parametrize("dtype", DTYPES)
def test_verify_blocks_that_read_as_nan(device, dtype):
    import dflash_mlx as dm

    cache, lens_d, k, v, q, proj, _ = _case(device, dtype, 2, 4, 2, [200, 200], 256, 3, False)
    for scales in (cache.k_scale, cache.v_scale):
        good = scales[1, 0, 2].clone()
        scales[1, 0, 2] = float("nan")
        got = dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device)).cpu().view(2, 2, 4, D)
        scales[1, 0, 2] = good
        assert got[1, :, :2].isnan().all()
        assert torch.isfinite(got[0].float()).all() and torch.isfinite(got[1, :, 2:].float()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,lens", [(1, [3000, 17, 900]), (16, [3000, 17, 900])])
def test_calls_on_two_streams_and_captured(device, dtype, T, lens):
    """Two streams at once over one cache, and two graphs captured on one stream and
    replayed beside each other and eager calls: all as the call alone."""
    import dflash_mlx as dm

    Hq, Hkv, Smax = 8, 2, 3136
    cache, lens_d, k, v, q, proj, _ = _case(device, dtype, T, Hq, Hkv, lens, Smax, 5, False)
    qs = [q.to(device), (q.float() * -0.5).bfloat16().to(device)]
    proj = proj.to(device)
    want = [dm.attn_verify_q8(x, cache, lens_d, proj) for x in qs]
    again = [dm.attn_verify_q8(x, cache, lens_d, proj) for x in qs]
    assert all(torch.equal(a, b) for a, b in zip(want, again))  # whichever part comes last
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(10):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(dm.attn_verify_q8(qs[i], cache, lens_d, proj))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])
    side = torch.cuda.Stream()
    graphs, outs = [], []
    for x in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            outs.append(dm.attn_verify_q8(x, cache, lens_d, proj))
        graphs.append(g)
    for turn in range(6):
        for o in outs:
            o.fill_(0)
        torch.cuda.synchronize()
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                graphs[i].replay()
        eager = dm.attn_verify_q8(qs[turn % 2], cache, lens_d, proj)
        torch.cuda.synchronize()
        assert torch.equal(eager, want[turn % 2])
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), turn


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_workspace_serves_every_shape(device, dtype):
    """One workspace for calls of growing and falling sizes: every call leaves its
    counts zero, and one that is too small is refused."""
    import dflash_mlx as dm
    from dflash_mlx import _lib

    Hq, Hkv, Smax = 8, 2, 4096
    n = dm.attn_verify_q8_workspace_bytes(3, 16, Hq, Hkv, Smax)
    ws = torch.zeros(n, dtype=torch.uint8, device=device)
    for T in (1, 16, 4, 8, 1, 3):
        cache, lens_d, k, v, q, proj, _ = _case(device, dtype, T, Hq, Hkv, [4000, 100, 2000], Smax, T, False)
        assert dm.attn_verify_q8_workspace_bytes(3, T, Hq, Hkv, Smax) <= n
        a = dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device), workspace=ws)
        b = dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device))
        assert torch.equal(a, b) and (ws[:4 * 3 * Hkv] == 0).all()
    with pytest.raises(_lib.DFlashError, match="workspace"):
        dm.attn_verify_q8(q.to(device), cache, lens_d, proj.to(device), workspace=ws[:1024])


def test_refusals(device):
    import dflash_mlx as dm

    cache, lens, k, v, q, proj, _ = _case(device, torch.int8, 4, 4, 2, [100, 30], 128, 1, False)
    q, proj = q.to(device), proj.to(device)
    w = torch.ones(D, dtype=torch.bfloat16, device=device)
    prep = dict(num_heads=4, rot_dims=32, rope_base=1e5)
    for fn, exc, text in (
            (lambda: dm.attn_verify_q8(q.float(), cache, lens, proj), TypeError, "q must be bfloat16"),
            (lambda: dm.attn_verify_q8(q[:1], cache, lens, proj), ValueError, "q must be"),
            (lambda: dm.attn_verify_q8(q[:, :, :3], cache, lens, proj), ValueError, "q must be"),
            (lambda: dm.attn_verify_q8(q.cpu(), cache, lens, proj), ValueError, "no CPU path"),
            (lambda: dm.attn_verify_q8(q, cache, lens.long(), proj), TypeError, "lens must be int32"),
            (lambda: dm.attn_verify_q8(q, cache, lens[:1], proj), ValueError, "lens must be contiguous"),
            (lambda: dm.attn_verify_q8(q, cache, lens.cpu(), proj), ValueError, "no CPU path"),
            (lambda: dm.attn_verify_q8(q, cache, lens, proj[:, :3]), ValueError, "proj must be"),
            (lambda: dm.attn_verify_q8(q, cache, lens, proj[..., :900]), ValueError, "proj must be"),
            (lambda: dm.attn_verify_q8(q, cache, lens, proj[..., 1:]), ValueError, "16-byte aligned"),
            (lambda: dm.attn_verify_q8(q.repeat(1, 5, 1, 1)[:, :17], cache, lens, proj.repeat(1, 5, 1)[:, :17]), ValueError,
             "at most 16 tokens"),
            (lambda: dm.attn_verify_q8(q.repeat(1, 4, 5, 1), cache, lens, proj.repeat(1, 4, 1)), ValueError, "64 query rows"),
            (lambda: dm.attn_verify_q8(q, cache, lens, proj, workspace=torch.zeros(9)), ValueError, "no CPU path"),
            (lambda: dm.attn_verify_q8(q, None, lens, proj), TypeError, "QuantizedKVCache"),
            (lambda: dm.attn_prefill_q8(q, cache, lens, proj[:, :2]), ValueError, "proj must be"),
            (lambda: dm.attn_prep_q8(proj.repeat(1, 5, 1), w, w, lens, cache, **prep), ValueError, "at most 16 tokens"),
            (lambda: dm.attn_prep_q8(proj, w[:64], w, lens, cache, **prep), ValueError, "q_norm must be"),
            (lambda: dm.attn_prep_q8(proj, w, w.float(), lens, cache, **prep), ValueError, "k_norm must be"),
            (lambda: dm.attn_prep_q8(proj, w, w, lens, cache, num_heads=3, rot_dims=32, rope_base=1e5), ValueError,
             "num_heads"),
            (lambda: dm.attn_prep_q8(proj, w, w, lens, cache, num_heads=4, rot_dims=48, rope_base=1e5), RuntimeError,
             "not supported"),
            (lambda: dm.attn_prep_q8(proj[..., :1400], w, w, lens, cache, **prep), ValueError, "proj must be"),
            (lambda: dm.kv_read_q8(cache, lens, -1), ValueError, "count"),
            (lambda: dm.kv_read_q8(cache, lens, 4, start=lens.long()), TypeError, "start must be int32"),
            (lambda: dm.kv_read_q8(cache, lens, 4, start=2 ** 31), ValueError, "32-bit"),
            (lambda: dm.kv_load_q8(k.to(device), v.to(device).float(), lens, cache), TypeError, "v must be bfloat16"),
            (lambda: dm.kv_load_q8(k.to(device), v.to(device)[:, :, :5], lens, cache), ValueError, "v must be"),
            (lambda: dm.kv_rewind_q8(cache, 129, 200), ValueError, "length"),
            (lambda: dm.kv_rewind_q8(cache, 50, 49), ValueError, "written")):
        with pytest.raises(exc, match=text):
            fn()
    # empty calls
    assert dm.attn_verify_q8(q[:, :0], cache, lens, proj[:, :0]).shape == (2, 0, 512)
    assert dm.attn_prefill_q8(q[:, :0], cache, lens, proj[:, :0]).shape == (2, 0, 512)
    assert dm.attn_prep_q8(proj[:, :0], w, w, lens, cache, **prep).shape == (2, 0, 4, D)
    assert dm.kv_read_q8(cache, lens, 0)[0].shape == (2, 2, 0, D)
    none = dm.QuantizedKVCache.zeros(0, 2, 64, torch.int8, device)
    assert dm.attn_verify_q8(q[:0], none, lens[:0], proj[:0]).shape == (0, 4, 512)
