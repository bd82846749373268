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


def norm_rotated(x, w, pos, rot):
    """(values, slack) fp64 of RMSNorm(x) * w rotated at pos: x [B, T, H, D] bf16, pos
    [B, T].  slack: what the kernels' fp32 may be off by before rounding, 2^-18 of the
    pair that the rotation mixes (a sum of 128 squares, a square root, a division, two
    products and the cosines' and sines' own 7e-8 each lose less than 2^-20)."""
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
    mag = x.abs()
    if rot:
        inv = THETA ** (-2.0 * torch.arange(rot // 2, dtype=torch.float64) / rot)
        ang = pos.double()[:, :, None, None] * inv
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        both = a.abs() + b.abs()
        x = torch.cat((a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), x[..., rot:]), -1)
        mag = torch.cat((both, both, mag[..., rot:]), -1)
    return x, mag * 2.0 ** -18


def rounded_right(got, want, slack):
    """got (bf16) is want rounded to bf16, half a step (2^-8) of what was rounded."""
    return bool(((got.double() - want).abs() <= 2.0 ** -8 * (want.abs() + slack) + slack).all())


def appended_keys(device, proj, lens, Hq, Hkv, wk, rot, Smax, dtype):
    """The keys [B, T, Hkv, D] that an append of these rows stores, taken from the same
    kernel with the key rows in the queries' place (of a scratch cache)."""
    import dflash_mlx as dm

    B, T = proj.shape[:2]
    rows = torch.zeros(B, T, 4 * Hkv * D, dtype=torch.bfloat16, device=device)
    rows[..., :2 * Hkv * D].view(B, T, Hkv, 2, D)[:, :, :, 0] = \
        proj[..., 2 * Hq * D:(2 * Hq + Hkv) * D].view(B, T, Hkv, D)
    scratch = dm.QuantizedKVCache.zeros(B, Hkv, Smax, dtype, device)
    return dm.attn_prep_q8(rows, wk, wk, lens, scratch, num_heads=Hkv, rot_dims=rot, rope_base=THETA, eps=EPS,
                           prompt=True)


def appended(device, k, v, proj, lens, Hq, Hkv, wk, rot, Smax, dtype):
    """Histories k, v [B, Hkv, Smax, D] with the rows' keys and values at lens[b] + t."""
    keys = appended_keys(device, proj, torch.tensor(lens, dtype=torch.int32, device=device), Hq, Hkv, wk, rot, Smax,
                         dtype).cpu()
    vals = proj[..., (2 * Hq + Hkv) * D:(2 * Hq + 2 * Hkv) * D].view(*proj.shape[:2], Hkv, D).cpu()
    k, v = k.clone(), v.clone()
    for b, L in enumerate(lens):
        n = max(0, min(L + proj.shape[1], Smax) - L) if L >= 0 else 0
        if n:
            k[b, :, L:L + n], v[b, :, L:L + n] = keys[b, :n].transpose(0, 1), vals[b, :n].transpose(0, 1)
    return k, v


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
