"""The 8-bit cache's operators as a program uses them together: a prompt, then blocks of
drafts of which some are kept, eager and as replays of one captured graph, every
attention against 64 bits over what the cache's own codes and tail stand for."""
from __future__ import annotations

import pytest
import torch

from oracle import kv8_oracle as orc
from tests.kv8_util import BLOCK, D, DTYPES, EPS, SLOTS, THETA, raw
from tests.test_gpu_kv8 import proj_rows

pytestmark = pytest.mark.gpu

B, HQ, HKV, SMAX, P, T = 3, 8, 2, 512, 150, 6
KEEP = [(1, 6, 3), (6, 6, 6), (2, 1, 5), (4, 6, 1), (6, 3, 6), (5, 5, 2), (6, 6, 6), (3, 6, 4)]


def _held(cache, b, n, done):
    """fp64 keys and values [Hkv, n, D] of positions [0, n): codes below `done` blocks,
    the tail from there on."""
    c = done * BLOCK
    k = cache.k_codes[b].cpu().float().double() * cache.k_scale[b].cpu().double().repeat_interleave(BLOCK, 1)[..., None]
    v = cache.v_codes[b].cpu().float().double() * cache.v_scale[b].cpu().double()[..., None, None]
    v = v.transpose(-2, -1).reshape(HKV, SMAX, D)
    p = torch.arange(c, n)
    k[:, c:n] = cache.tail_k[b].cpu().double()[:, p % SLOTS]
    v[:, c:n] = cache.tail_vt[b].cpu().double()[:, :, p % SLOTS].transpose(1, 2)
    return k[:, :n], v[:, :n]


def _check(out, q, rows, cache, lens, rows_n, prompt):
    """attention_error's bound (tests/kv8_util.py), over the values the cache holds."""
    out, q = out.cpu().view(B, rows_n, HQ, D).double(), q.cpu()
    gate = rows.cpu()[:, :, :2 * HQ * D].view(B, rows_n, HQ, 2, D)[:, :, :, 1]
    for b, L in enumerate(lens):
        if L < 0:
            assert (out[b] == 0).all()
            continue
        n = L + rows_n
        k, v = _held(cache, b, n, (n if prompt else L) // BLOCK)
        ref, spread = orc.attention(q[b], k, v, gate[b], L, 0, cache.dtype, D ** -0.5)
        bound = 2.0 ** -8 * (spread + ref.abs()) + 2.0 ** -10 * spread + 1e-30
        assert bool(((out[b] - ref).abs() <= bound).all()), (b, L)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("starts", [(0, 0, 0), (70, -1, 33)])
def test_prompt_and_blocks(device, dtype, starts):
    import dflash_mlx as dm

    g = torch.Generator().manual_seed(4)
    qn, kn = ((1 + 0.2 * torch.randn(D, generator=g)).bfloat16().to(device) for _ in range(2))
    old = [torch.randn(B, HKV, 128, D, generator=g).bfloat16().to(device) for _ in range(2)]
    prompt = proj_rows(B, P, HQ, HKV, 5, 24).to(device)
    blocks = [proj_rows(B, T, HQ, HKV, 6 + i, 24).to(device) for i in range(len(KEEP))]
    keep = [torch.tensor([k if L >= 0 else 0 for k, L in zip(ks, starts)], dtype=torch.int32, device=device) for ks in KEEP]
    runs = []
    for form in ("eager", "graph"):
        stream = torch.cuda.Stream(device)
        with torch.cuda.stream(stream):
            cache = dm.QuantizedKVCache.zeros(B, HKV, SMAX, dtype, device)
            lens = torch.tensor(starts, dtype=torch.int32, device=device)
            dm.kv_load_q8(*old, lens, cache)
            overflow = torch.zeros(B, dtype=torch.int32, device=device)
            block = torch.empty_like(blocks[0])

            def prep(rows, prompt):
                return dm.attn_prep_q8(rows, qn, kn, lens, cache, num_heads=HQ, rot_dims=32, rope_base=THETA, eps=EPS,
                                       prompt=prompt, overflow=overflow)

            def step():
                q = prep(block, False)
                return q, dm.attn_verify_q8(q, cache, lens, block), *dm.kv_read_q8(cache, lens, 96, start=lens)

            q = prep(prompt, True)
            outs = [dm.attn_prefill_q8(q, cache, lens, prompt)]
            if form == "eager":
                torch.cuda.synchronize()
                _check(outs[0], q, prompt, cache, starts, P, True)
            lens += torch.where(lens < 0, 0, P).int()
            if form == "graph":
                block.copy_(blocks[0])
                step()  # (what a first call sets up)
                torch.cuda.synchronize()
                graph = torch.cuda.CUDAGraph()
                with torch.cuda.graph(graph, stream=stream):
                    res = step()
            for i, rows in enumerate(blocks):
                block.copy_(rows)
                if form == "eager":
                    res = step()
                    torch.cuda.synchronize()
                    _check(res[1], res[0], rows, cache, lens.tolist(), T, False)
                else:
                    graph.replay()
                    if i % 3 == 1:
                        torch.cuda.synchronize()
                outs += [r.clone() for r in res]
                lens += keep[i]
        torch.cuda.synchronize()
        assert overflow.tolist() == [int(L < 0) for L in starts]
        runs.append((outs, raw(cache)))
    (a, ca), (b, cb) = runs
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and all(torch.equal(x, y) for x, y in zip(ca, cb))


@pytest.mark.parametrize("dtype", DTYPES)
def test_offsets_past_32_bits(device, dtype):
    """Codes of more than 2^31 bytes: the last sequence, 130 937 positions long, appended
    to, read and attended to at the cache's far end."""
    import dflash_mlx as dm

    n, smax, L, hq = 40, 131072, 130937, 4
    cache = dm.QuantizedKVCache.zeros(n, HKV * 2, smax, dtype, device)
    assert cache.k_codes.numel() > 2 ** 31
    g = torch.Generator().manual_seed(3)
    k, v = (torch.randn(1, HKV * 2, L, D, generator=g).bfloat16() for _ in range(2))
    lens = torch.full((n,), -1, dtype=torch.int32, device=device)
    lens[-1] = L
    dm.kv_load_q8(*(x.to(device).expand(n, -1, -1, -1) for x in (k, v)), lens, cache)
    w = torch.ones(D, dtype=torch.bfloat16, device=device)
    for T, prompt in ((3, False), (70, True)):
        rows = proj_rows(1, T, hq, HKV * 2, 8 + T).to(device).expand(n, -1, -1).contiguous()
        q = dm.attn_prep_q8(rows, w, w, lens, cache, num_heads=hq, rot_dims=32, rope_base=THETA, eps=EPS, prompt=prompt)
        out = (dm.attn_prefill_q8 if prompt else dm.attn_verify_q8)(q, cache, lens, rows).cpu().view(n, T, hq, D)
        assert (out[:-1] == 0).all()
        done = (L + (T if prompt else 0)) // BLOCK
        kk, vv = (orc.held(x[0], L // BLOCK, dtype) for x in (k, v))
        p = torch.arange(L // BLOCK * BLOCK, L + T)
        new = [cache.tail_k[-1].cpu()[:, p % SLOTS], cache.tail_vt[-1].cpu()[:, :, p % SLOTS].transpose(1, 2)]
        kk, vv = (torch.cat((x[:, :p[0]], orc.held(y, done - L // BLOCK, dtype)), 1) for x, y in zip((kk, vv), new))
        gate = rows[-1:].cpu()[:, :, :2 * hq * D].view(1, T, hq, 2, D)[0, :, :, 1]
        ref, spread = orc.attention(q[-1].cpu(), kk, vv, gate, L, 0, dtype, D ** -0.5)
        bound = 2.0 ** -8 * (spread + ref.abs()) + 2.0 ** -10 * spread + 1e-30
        assert bool(((out[-1].double() - ref).abs() <= bound).all()), (T, prompt)
        at = L + (T if prompt else 0)
        got = dm.kv_read_q8(cache, torch.where(lens < 0, lens, at), 150, start=at - 150)
        for x, want in zip(got, (kk, vv)):
            assert torch.equal(x[-1].cpu(), want[:, at - 150:at].float().bfloat16()) and (x[:-1] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_prompts_of_several_lengths(device, dtype):
    """A call for each length, the other sequences at -1: every sequence's cache and rows
    are those of a cache of its own."""
    import dflash_mlx as dm

    sizes = (130, 64, 7)
    w = torch.ones(D, dtype=torch.bfloat16, device=device)
    rows = [proj_rows(1, n, HQ, HKV, 30 + n).to(device) for n in sizes]
    kw = dict(num_heads=HQ, rot_dims=32, rope_base=THETA, eps=EPS, prompt=True)

    def lens(*x):
        return torch.tensor(x, dtype=torch.int32, device=device)

    cache = dm.QuantizedKVCache.zeros(len(sizes), HKV, 192, dtype, device)
    for b, (n, r) in enumerate(zip(sizes, rows)):
        own = dm.QuantizedKVCache.zeros(1, HKV, 192, dtype, device)
        want = dm.attn_prefill_q8(dm.attn_prep_q8(r, w, w, lens(0), own, **kw), own, lens(0), r)
        batch = torch.full((len(sizes), *r.shape[1:]), float("nan"), dtype=r.dtype, device=device)
        batch[b] = r[0]
        at = lens(*(0 if i == b else -1 for i in range(len(sizes))))
        got = dm.attn_prefill_q8(dm.attn_prep_q8(batch, w, w, at, cache, **kw), cache, at, batch)
        assert torch.equal(got[b], want[0]) and (got[[i for i in range(len(sizes)) if i != b]] == 0).all()
        for x, y in zip(dm.kv_read_q8(cache, lens(*sizes), n), dm.kv_read_q8(own, lens(n), n)):
            assert torch.equal(x[b], y[0])
