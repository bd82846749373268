"""The 8-bit key/value cache: quantising, loading, reading back and appending.

Codes, scales and the values read back are compared bit for bit with the
definition (oracle/kv8_oracle.py); appended queries and keys with their
formula in 64 bits, and the bf16 cache's append (dflash_attn_prep) with both."""
from __future__ import annotations

import pytest
import torch

from oracle import kv8_oracle as orc
from tests.kv8_util import (BLOCK, D, DTYPES, EPS, THETA, appended, appended_keys, expected_read, loaded, norm_rotated,
                            proj_rows, random_kv, raw, rounded_right, tail_holds)

pytestmark = pytest.mark.gpu


def _blocks(cache, dtype):
    """(keys, values) codes as bytes [B, H, nb, 64, D] on the host."""
    B, H, S, _ = cache.k_codes.shape
    k = cache.k_codes.view(torch.uint8).cpu().view(B, H, S // BLOCK, BLOCK, D)
    return k, cache.v_codes.view(torch.uint8).cpu().transpose(3, 4)


def _same_codes(cache, b, k, v, lo, hi, dtype):
    """Blocks [lo, hi) of sequence b are the quantised bf16 history k, v [H, n, D]."""
    kc, vc = _blocks(cache, dtype)
    for x, codes, scales in ((k, kc, cache.k_scale), (v, vc, cache.v_scale)):
        x = x[:, lo * BLOCK:hi * BLOCK].reshape(x.shape[0], hi - lo, BLOCK, D)
        s, m = orc.block_scale(x, dtype)
        assert torch.equal(codes[b, :, lo:hi], orc.block_codes(x, m, dtype).view(torch.uint8))
        torch.testing.assert_close(scales[b, :, lo:hi].cpu(), s, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B,Hkv,S,Smax,lens", [
    (1, 1, 1, 64, [1]), (2, 3, 200, 256, [200, 0]), (3, 2, 128, 128, [128, 64, 63]), (2, 2, 321, 320, [321, 65]),
    (2, 1, 100, 192, [-1, 77])])
def test_load_codes_and_tail(device, dtype, B, Hkv, S, Smax, lens):
    k, v = random_kv(B, Hkv, S, seed=S + B)
    cache, _ = loaded(device, k, v, lens, Smax, dtype)
    kc, vc = _blocks(cache, dtype)
    for b, n in enumerate(min(x, Smax) for x in lens):
        n = max(n, 0)
        _same_codes(cache, b, k[b], v[b], 0, n // BLOCK, dtype)
        assert tail_holds(cache, b, k[b], v[b], max(n // BLOCK - 1, 0) * BLOCK, n)
        # nothing else is touched
        assert (kc[b, :, n // BLOCK:] == 0xA5).all() and (vc[b, :, n // BLOCK:] == 0xA5).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantiser_at_its_edges(device, dtype):
    """Blocks of zeros, of the smallest and largest bf16, with ties, with one
    value at each border of the scale, and with a NaN or an infinity."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(16, BLOCK, D, generator=g)
    x[0] = 0
    x[1] *= 2.0 ** -133   # bf16 subnormals
    x[2] *= 2.0 ** -104
    x[3] *= 2.0 ** 120
    x[3, 0, 0] = 3.3895313892515355e38  # the largest bf16
    x[4] = torch.round(x[4] * 8) / 16   # ties
    x[4, 0, 0] = 127 / 16 * 8
    x[5, 5, 7] = 448.0
    x[6, 5, 7] = 450.0
    x[7, 5, 7] = -7.0     # 1.75 * 4
    x[8, 5, 7] = 7.03125
    x[9, 63, 127] = float("nan")
    x[10, 0, 0] = float("inf")
    x[11, 31, 64] = float("-inf")
    k = x.bfloat16().view(1, 1, -1, D)
    v = k.flip(2).contiguous()
    S = k.shape[2]
    cache, lens = loaded(device, k, v, [S], S, dtype)
    _same_codes(cache, 0, k[0], v[0], 0, S // BLOCK, dtype)
    import dflash_mlx as dm

    got_k, got_v = dm.kv_read_q8(cache, torch.tensor([S + 0], dtype=torch.int32, device=device), S)
    for got, want in ((got_k, k), (got_v, v)):
        torch.testing.assert_close(got[0].cpu(), expected_read(want[0], S, 0, S, dtype), rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lens,start,count", [
    ([300, 129, 64], 0, 384), ([300, 129, 64], 63, 2), ([300, 1, 0], -5, 77), ([65, 80, 81], 1, 200),
    ([300, 200, 100], [236, 130, 99], 65), ([-3, 383, 384], [0, 320, -200], 150), ([128, 144, 145], 60, 1)])
def test_read_back(device, dtype, lens, start, count):
    import dflash_mlx as dm

    k, v = random_kv(3, 2, 384, seed=7)
    cache, lens_d = loaded(device, k, v, lens, 384, dtype)
    st = torch.tensor(start, dtype=torch.int32, device=device) if isinstance(start, list) else start
    before = raw(cache)
    got = dm.kv_read_q8(cache, lens_d, count, start=st)
    for x, y in ((k, got[0]), (v, got[1])):
        for b in range(3):
            want = expected_read(x[b], max(lens[b], 0), start[b] if isinstance(start, list) else start, count, dtype)
            assert torch.equal(y[b].cpu(), want), b
    assert all(torch.equal(a, c) for a, c in zip(before, raw(cache)))  # reading writes nothing


@pytest.mark.parametrize("dtype", DTYPES)
def test_load_takes_strided_keys(device, dtype):
    """Keys [B, S, H, D] seen as [B, H, S, D], and a slice that is not 16-byte aligned."""
    import dflash_mlx as dm

    k, v = random_kv(2, 3, 150, seed=5)
    lens = [150, 130]
    want = raw(loaded(device, k, v, lens, 192, dtype)[0])
    kt = k.transpose(1, 2).contiguous().to(device).transpose(1, 2)
    wide = torch.zeros(2, 3, 150, D + 4, dtype=torch.bfloat16, device=device)
    wide[..., 4:] = v.to(device)
    cache = dm.QuantizedKVCache.zeros(2, 3, 192, dtype, device)
    for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, cache.tail_k, cache.tail_vt):
        t.view(torch.uint8).fill_(0xA5)
    dm.kv_load_q8(kt, wide[..., 4:], torch.tensor(lens, dtype=torch.int32, device=device), cache)
    assert all(torch.equal(a, b) for a, b in zip(want, raw(cache)))


def _append(device, cache, proj, lens, Hq, Hkv, wq, wk, rot, prompt, overflow=None):
    import dflash_mlx as dm

    return dm.attn_prep_q8(proj, wq, wk, lens, cache, num_heads=Hq, rot_dims=rot, rope_base=THETA, eps=EPS,
                           prompt=prompt, overflow=overflow)


def _queries_right(q, proj, lens, Hq, w, rot):
    B, T = proj.shape[:2]
    pos = torch.tensor(lens)[:, None] + torch.arange(T)
    rows = proj[..., :2 * Hq * D].reshape(B, T, Hq, 2, D)[:, :, :, 0]
    assert rounded_right(q.cpu(), *norm_rotated(rows.cpu(), w.cpu(), pos, rot))


@pytest.mark.parametrize("rot", [0, 16, 32, 64, 128])
def test_queries_and_keys_against_their_formula(device, rot):
    """At positions from 0 to over 10^5, in both forms, with rows of every size: the
    formula in 64 bits rounded once, and the bf16 cache's append within its own rounding."""
    import dflash_mlx as dm
    from dflash_mlx import _lib

    B, T, Hq, Hkv, Smax = 5, 16, 6, 2, 131072
    lens = [0, 1000, 40961, 99999, Smax - T]
    proj = proj_rows(B, T, Hq, Hkv, seed=rot)
    proj *= torch.tensor([1.0, 1e-4, 30.0, 0.0, 1e4]).bfloat16()[:, None, None]
    g = torch.Generator().manual_seed(rot)
    w = (1 + 0.2 * torch.randn(D, generator=g)).bfloat16().to(device)
    proj, lens_d = proj.to(device), torch.tensor(lens, dtype=torch.int32, device=device)
    cache = dm.QuantizedKVCache.zeros(B, Hkv, 64, torch.int8, device)  # positions past it are not written
    q = _append(device, cache, proj, lens_d, Hq, Hkv, w, w, rot, False)
    assert torch.equal(q, _append(device, cache, proj, lens_d, Hq, Hkv, w, w, rot, True))
    _queries_right(q, proj, lens, Hq, w, rot)
    keys = appended_keys(device, proj, lens_d, Hq, Hkv, w, rot, 64, torch.int8)
    rows = proj[..., 2 * Hq * D:(2 * Hq + Hkv) * D].reshape(B, T, Hkv, D).cpu()
    want, slack = norm_rotated(rows, w.cpu(), torch.tensor(lens)[:, None] + torch.arange(T), rot)
    assert rounded_right(keys.cpu(), want, slack)
    # the bf16 cache's append: an fp32 angle of up to 2 pi is off by 2.4e-7, so 2^-16 of the pair
    kc = torch.zeros(1, Hkv, Smax, D, dtype=torch.bfloat16, device=device)
    vt = torch.zeros(1, Hkv, D, Smax, dtype=torch.bfloat16, device=device)
    for b, L in enumerate(lens):
        qb = torch.empty(1, T, Hq, D, dtype=torch.bfloat16, device=device)
        _lib.call("dflash_attn_prep", proj[b].data_ptr(), proj.stride(1), w.data_ptr(), w.data_ptr(),
                  lens_d[b:].data_ptr(), kc.data_ptr(), vt.data_ptr(), qb.data_ptr(), None, 1, T, Hq, Hkv, D, Smax, rot,
                  THETA, EPS, _lib.stream_handle(device))
        got = kc[0, :, L:L + T].transpose(0, 1).cpu()
        assert rounded_right(got, want[b], 4 * slack[b])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,Hkv,rot,lens", [
    (1, 4, 1, 32, [0, 63, 64, 80, 81]), (16, 16, 4, 32, [0, 48, 60, 64, 70]), (7, 8, 8, 128, [1, 121, 128, 144, 200]),
    (5, 6, 2, 0, [300, 5, 127, 129, 192]), (3, 3, 3, 16, [17, 62, 63, 66, 319]), (2, 2, 1, 64, [62, 63, 64, 65, 80])])
def test_draft_append(device, dtype, T, Hq, Hkv, rot, lens):
    B, Smax = len(lens), 384
    k, v = random_kv(B, Hkv, Smax, seed=T)
    cache, lens_d = loaded(device, k, v, lens, Smax, dtype)
    # the waiting block's codes are not there yet
    for b, L in enumerate(lens):
        if L >= BLOCK and L % BLOCK <= 16:
            j = L // BLOCK - 1
            cache.k_codes[b, :, j * BLOCK:(j + 1) * BLOCK].view(torch.uint8).fill_(0x11)
            cache.v_codes[b, :, j].view(torch.uint8).fill_(0x11)
            cache.k_scale[b, :, j] = 9.0
            cache.v_scale[b, :, j] = 9.0
    before = raw(cache)
    proj = proj_rows(B, T, Hq, Hkv, seed=T + 1, pad=8).to(device)
    g = torch.Generator().manual_seed(9)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).bfloat16().to(device) for _ in range(2))
    q = _append(device, cache, proj, lens_d, Hq, Hkv, wq, wk, rot, False)
    _queries_right(q, proj, lens, Hq, wq, rot)
    ks, vs = appended(device, k, v, proj, lens, Hq, Hkv, wk, rot, Smax, dtype)
    for b, L in enumerate(lens):
        kk, vv = ks[b], vs[b]
        _same_codes(cache, b, kk, vv, 0, L // BLOCK, dtype)
        lo = max(L // BLOCK - (L % BLOCK + T <= BLOCK), 0) * BLOCK
        assert tail_holds(cache, b, kk, vv, lo, L + T)
    # codes of no other block are touched
    after = raw(cache)
    for i in (0, 1):
        for b, L in enumerate(lens):
            a, c = before[i][b], after[i][b]
            if i == 0:
                a, c = (x.view(Hkv, -1, BLOCK, D) for x in (a, c))
            assert torch.equal(a[:, L // BLOCK:], c[:, L // BLOCK:])


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("T,Hq,Hkv,rot,lens", [
    (1, 4, 1, 32, [0, 63, 64]), (17, 16, 4, 32, [0, 48, 70]), (64, 8, 8, 128, [1, 64, 127]),
    (65, 6, 2, 0, [0, 63, 100]), (200, 4, 2, 32, [0, 70, 130]), (333, 2, 1, 64, [15, 31, 17]), (128, 4, 4, 16, [0, 65, 80])])
def test_prompt_append(device, dtype, T, Hq, Hkv, rot, lens):
    B, Smax = len(lens), 384
    k, v = random_kv(B, Hkv, Smax, seed=T)
    cache, lens_d = loaded(device, k, v, lens, Smax, dtype)
    for b, L in enumerate(lens):
        if L >= BLOCK and L % BLOCK <= 16:
            j = L // BLOCK - 1
            cache.k_codes[b, :, j * BLOCK:(j + 1) * BLOCK].view(torch.uint8).fill_(0x11)
            cache.v_scale[b, :, j] = 9.0
    proj = proj_rows(B, T, Hq, Hkv, seed=T + 1).to(device)
    g = torch.Generator().manual_seed(9)
    wq, wk = ((1 + 0.2 * torch.randn(D, generator=g)).bfloat16().to(device) for _ in range(2))
    flags = torch.zeros(B, dtype=torch.int32, device=device)
    q = _append(device, cache, proj, lens_d, Hq, Hkv, wq, wk, rot, True, flags)
    _queries_right(q, proj, lens, Hq, wq, rot)
    assert flags.cpu().tolist() == [int(L + T > Smax) for L in lens]
    ks, vs = appended(device, k, v, proj, lens, Hq, Hkv, wk, rot, Smax, dtype)
    for b, L in enumerate(lens):
        kk, vv, end = ks[b], vs[b], min(L + T, Smax)
        _same_codes(cache, b, kk, vv, 0, end // BLOCK, dtype)
        assert tail_holds(cache, b, kk, vv, max(end // BLOCK - 1, 0) * BLOCK, end)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("prompt", [False, True])
def test_sequences_that_take_no_part_or_run_over(device, dtype, prompt):
    """A negative length writes nothing; positions past the cache are not written
    and flagged; a length past the cache's end writes nothing."""
    B, Hq, Hkv, Smax, T = 4, 4, 2, 128, 10
    lens = [-1, 120, 128, 500]
    k, v = random_kv(B, Hkv, Smax, seed=2)
    cache, _ = loaded(device, k, v, [100, 120, 128, 100], Smax, dtype)
    before = raw(cache)
    proj = proj_rows(B, T, Hq, Hkv, seed=4).to(device)
    w = torch.ones(D, dtype=torch.bfloat16, device=device)
    flags = torch.zeros(B, dtype=torch.int32, device=device)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=device)
    _append(device, cache, proj, lens_d, Hq, Hkv, w, w, 32, prompt, flags)
    assert flags.cpu().tolist() == [1, 1, 1, 1]
    after = raw(cache)
    for i in range(6):
        for b in (0, 3):
            assert torch.equal(before[i][b], after[i][b]), (i, b)
    ks, vs = appended(device, k, v, proj, [-1, 120, -1, -1], Hq, Hkv, w, 32, Smax, dtype)
    assert tail_holds(cache, 1, ks[1], vs[1], 64, 128)
    _same_codes(cache, 2, k[2], v[2], 0, 2, dtype)
    assert tail_holds(cache, 2, k[2], v[2], 64, 128)  # of a load: the last two blocks, 1 and (empty) 2


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_do_not_depend_on_rejected_drafts(device, dtype):
    """Blocks of draft tokens of which some are rejected, huge ones among them,
    against the kept tokens appended as one prompt: the same codes and reads."""
    import dflash_mlx as dm

    Hq, Hkv, Smax = 4, 2, 320
    g = torch.Generator().manual_seed(21)
    w = torch.ones(D, dtype=torch.bfloat16, device=device)
    cache = dm.QuantizedKVCache.zeros(1, Hkv, Smax, dtype, device)
    kept, L = [], 0
    while L < 250:
        T = int(torch.randint(1, 17, (1,), generator=g))
        keep = int(torch.randint(1, T + 1, (1,), generator=g))
        rows = proj_rows(1, T, Hq, Hkv, seed=1000 + L)
        rows[:, keep:, (2 * Hq + Hkv) * D:] *= 1000.0
        if L % 3 == 0:
            rows[:, keep:, (2 * Hq + Hkv) * D:] = float("nan")
        _append(device, cache, rows.to(device), torch.tensor([L], dtype=torch.int32, device=device), Hq, Hkv, w, w, 32,
                False)
        kept.append(rows[:, :keep])
        L += keep
    lens = torch.tensor([L], dtype=torch.int32, device=device)
    whole = dm.QuantizedKVCache.zeros(1, Hkv, Smax, dtype, device)
    _append(device, whole, torch.cat(kept, 1).to(device), torch.zeros(1, dtype=torch.int32, device=device), Hq, Hkv, w, w,
            32, True)
    for a, b in zip(dm.kv_read_q8(cache, lens, L), dm.kv_read_q8(whole, lens, L)):
        assert torch.equal(a, b) and torch.isfinite(a.float()).all()
    n = (L - 17) // BLOCK  # blocks whose codes are certainly there
    for a, b in zip(raw(cache)[:2], raw(whole)[:2]):
        a, b = (x.view(Hkv, -1, BLOCK * D) for x in (a, b))
        assert torch.equal(a[:, :n], b[:, :n])
