"""The 8-bit key/value cache and its attention in plain torch on the CPU.

Written from the definitions (a block's scale and codes, which positions are
read from codes, gated softmax attention), in 64 bits but for the quantiser,
whose fp32 operations are the definition.
"""
from __future__ import annotations

import torch

BLOCK, SLOTS, D = 64, 128, 128
F64 = torch.float64


def block_scale(x: torch.Tensor, dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """(scale, multiplier) fp32 [...] of bf16 blocks [..., 64, 128] (either order)."""
    a = x.float().abs().amax((-2, -1))
    bad = ~torch.isfinite(x.float()).flatten(-2).all(-1)
    a = torch.where(bad, torch.ones_like(a), a).clamp_min(2.0 ** -100)
    if dtype is torch.int8:
        c = torch.full_like(a, 127.0)
        s, m = a / c, c / a  # tensor by tensor: one rounding each
    else:
        e = torch.floor(torch.log2(a.double())) - 9  # at most two below the answer
        s = torch.pow(2.0, e)
        for _ in range(3):
            s = torch.where(a.double() > 448 * s, 2 * s, s)
        s, m = s.float(), (1 / s).float()
    return torch.where(bad, float("nan"), s), torch.where(bad, 0.0, m)


def block_codes(x: torch.Tensor, mul: torch.Tensor, dtype) -> torch.Tensor:
    # a block with a NaN or an infinity: codes 0
    y = torch.where(mul[..., None, None] == 0, 0.0, x.float() * mul[..., None, None])
    if dtype is torch.int8:
        return torch.round(y).to(torch.int8)
    return y.to(torch.float8_e4m3fn)


def quantised(x: torch.Tensor, dtype) -> torch.Tensor:
    """The fp64 values that blocks [..., 64, 128] stand for once quantised."""
    s, m = block_scale(x, dtype)
    return block_codes(x, m, dtype).float().double() * s.double()[..., None, None]


def held(x: torch.Tensor, done: int, dtype) -> torch.Tensor:
    """fp64 values of bf16 positions [H, n, D] with the blocks below `done` quantised."""
    out = x.double()
    cut = min(done * BLOCK, x.shape[1] // BLOCK * BLOCK)
    if cut:
        out[:, :cut] = quantised(x[:, :cut].reshape(x.shape[0], -1, BLOCK, D), dtype).view(x.shape[0], cut, D)
    return out


def attention(q, k, v, gate, base: int, done: int, dtype, scale: float):
    """q [T, Hq, D], gate [T, Hq, D], k, v [Hkv, n, D] bf16 -> (out, spread) fp64
    [T, Hq, D]: row t over positions 0 .. base + t, and sigmoid(gate) times the
    weighted mean of |v|."""
    T, Hq, _ = q.shape
    rep = Hq // k.shape[0]
    n = k.shape[1]
    k, v = held(k, done, dtype), held(v, done, dtype)
    out, spread = torch.empty(T, Hq, D, dtype=F64), torch.empty(T, Hq, D, dtype=F64)
    for h in range(Hq):
        for t in range(T):
            m = min(base + t + 1, n)
            w = torch.softmax(k[h // rep, :m] @ q[t, h].double() * scale, 0)
            out[t, h] = w @ v[h // rep, :m]
            spread[t, h] = w @ v[h // rep, :m].abs()
    s = torch.sigmoid(gate.double())
    return out * s, spread * s
