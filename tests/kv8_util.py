"""Helpers of the 8-bit key/value cache's tests: a cache beside its bf16 history."""
from __future__ import annotations

import torch

from oracle import kv8_oracle as orc

D, BLOCK, SLOTS = 128, 64, 128
DTYPES = [torch.int8, torch.float8_e4m3fn]
THETA, EPS = 100000.0, 1e-6


def random_kv(B, Hkv, S, seed, spread=True):
    """bf16 keys and values [B, Hkv, S, D]; spread: magnitudes that change by block."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        x = torch.randn(B, Hkv, S, D, generator=g)
        if spread:
            x *= torch.exp2(torch.randint(-6, 7, (B, Hkv, -(-S // BLOCK)), generator=g).float()).repeat_interleave(
                BLOCK, 2)[:, :, :S, None]
        out.append(x.bfloat16())
    return out


def loaded(device, k, v, lens, Smax, dtype, fill=0xA5):
    """A cache with k, v loaded up to lens; every byte it does not hold is `fill`."""
    import dflash_mlx as dm

    B, Hkv = k.shape[:2]
    cache = dm.QuantizedKVCache.zeros(B, Hkv, Smax, dtype, device)
    for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale, cache.tail_k, cache.tail_vt):
        t.view(torch.uint8).fill_(fill)
    lens_d = torch.tensor(lens, dtype=torch.int32, device=device)
    dm.kv_load_q8(k.to(device), v.to(device), lens_d, cache)
    return cache, lens_d


def raw(cache):
    """Every tensor of the cache as bytes on the host."""
    return [t.view(torch.uint8).cpu().clone() for t in (cache.k_codes, cache.v_codes, cache.k_scale, cache.v_scale,
                                                        cache.tail_k, cache.tail_vt)]


def expected_read(x, L, start, count, dtype):
    """bf16 [H, count, D] of history x [H, n, D] read at committed length L."""
    vals = orc.held(x[:, :L], L // BLOCK, dtype).float()  # one fp32 product: exact, or rounded as the kernel's
    out = torch.zeros(x.shape[0], count, D)
    lo, hi = max(start, 0), min(start + count, L)
    if hi > lo:
        out[:, lo - start:hi - start] = vals[:, lo:hi]
    return out.bfloat16()


def tail_holds(cache, b, k, v, lo, hi):
    """The tail's slots of positions [lo, hi) hold the bf16 history k, v [H, n, D]."""
    p = torch.arange(lo, hi)
    tk, tv = cache.tail_k[b].cpu(), cache.tail_vt[b].cpu()
    return torch.equal(tk[:, p % SLOTS], k[:, p]) and torch.equal(tv[:, :, p % SLOTS].transpose(1, 2), v[:, p])


def proj_rows(B, T, Hq, Hkv, seed, pad=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(B, T, (2 * Hq + 2 * Hkv) * D + pad, generator=g).bfloat16()


def bf16_append(device, proj, lens, Smax, Hq, Hkv, wq, wk, rot):
    """dflash_attn_prep of the same rows: (q, keys, values [B, Hkv, Smax, D])."""
    from dflash_mlx import _lib

    B, T = proj.shape[:2]
    kc = torch.zeros(B, Hkv, Smax, D, dtype=torch.bfloat16, device=device)
    vt = torch.zeros(B, Hkv, D, Smax, dtype=torch.bfloat16, device=device)
    q = torch.empty(B, T, Hq, D, dtype=torch.bfloat16, device=device)
    _lib.call("dflash_attn_prep", proj.data_ptr(), proj.stride(1), wq.data_ptr(), wk.data_ptr(), lens.data_ptr(),
              kc.data_ptr(), vt.data_ptr(), q.data_ptr(), None, B, T, Hq, Hkv, D, Smax, rot, THETA, EPS,
              _lib.stream_handle(device))
    return q, kc, vt.transpose(2, 3)


def attention_error(got, q, k, v, proj, lens, ends, dtype, scale):
    """Largest error of got [B, T, Hq * D] in units of its bound.

    A weight is rounded to bf16 (half a step: 2^-8 of it) and so is the output; the
    scores' fp32 sums, the exponentials and the queries' integer digits move a weight by
    less than 2^-10 of it.  So |error| <= 2^-8 (spread + |out|) + 2^-10 spread, with
    spread the weighted mean of |v| times the gate."""
    B, T, Hq, _ = q.shape
    gate = proj[:, :, :2 * Hq * D].view(B, T, Hq, 2, D)[:, :, :, 1]
    worst = 0.0
    for b in range(B):
        ref, spread = orc.attention(q[b], k[b][:, :ends[b][0]], v[b][:, :ends[b][0]], gate[b], lens[b], ends[b][1],
                                    dtype, scale)
        bound = 2.0 ** -8 * (spread + ref.abs()) + 2.0 ** -10 * spread + 1e-30
        err = (got[b].view(T, Hq, D).double() - ref).abs() / bound
        worst = max(worst, float(err.max()) if not bool(err.isnan().any()) else float("inf"))
    return worst
