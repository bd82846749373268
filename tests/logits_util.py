"""Logits processing from its definition, and inputs for its tests."""
from __future__ import annotations

import torch


def counts_of(prompt, generated, V):
    """(times generated [B, V], in the prompt [B, V]) of lists of token lists."""
    made, seen = torch.zeros(len(generated), V, dtype=torch.int64), torch.zeros(len(prompt), V, dtype=torch.bool)
    for b, tokens in enumerate(generated):
        for t in tokens:
            if 0 <= t < V:
                made[b, t] += 1
    for b, tokens in enumerate(prompt):
        for t in tokens:
            if 0 <= t < V:
                seen[b, t] = True
    return made, seen


def processed(logits, made, prompt, bias, penalties, draft, allowed, dtype=torch.float64):
    """[B, N, V] by the definition in `dtype`, on the CPU; magnitude of the terms besides.
    allowed: bool [B, N, V] or None; draft: lists or None."""
    B, N, V = logits.shape
    out, size = torch.empty(B, N, V, dtype=dtype), torch.empty(B, N, V, dtype=dtype)
    for b in range(B):
        rep, pres, freq = penalties[b].to(dtype)
        c = made[b].clone()
        for i in range(N):
            if i and draft is not None and i <= len(draft[b]) and 0 <= draft[b][i - 1] < V:
                c[draft[b][i - 1]] += 1
            l = logits[b, i].to(dtype)
            seen = prompt[b] | (c > 0)
            l = torch.where(seen, torch.where(l > 0, l / rep, l * rep), l)
            size[b, i] = l.abs() + (freq * c).abs() + pres.abs() + bias[b].to(dtype).abs()
            f = torch.where(c > 0, freq * c.to(dtype), torch.zeros((), dtype=dtype))
            p = torch.where(c > 0, pres, torch.zeros((), dtype=dtype))
            l = l - f - p
            l = torch.where(seen | (bias[b] != 0), l + bias[b].to(dtype), l)
            if allowed is not None:
                l = torch.where(allowed[b, i], l, torch.full_like(l, -torch.inf))
            out[b, i] = l
    return out, size


def words(allowed):
    """bool [..., V] -> int32 words [..., ceil(V / 32)], the bits past V as given by chance."""
    V = allowed.shape[-1]
    W = -(-V // 32)
    a = torch.ones(*allowed.shape[:-1], 32 * W, dtype=torch.int64)
    a[..., :V] = allowed.long()
    w = (a.view(*allowed.shape[:-1], W, 32) << torch.arange(32)).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def argmax_lowest(x):
    """argmax with NaN above all and the lowest index on ties."""
    nan = torch.isnan(x)
    y = torch.where(nan, torch.full_like(x, torch.inf), x)
    key = torch.stack((nan.any(-1, keepdim=True).expand_as(x), ), 0)[0]
    best = torch.where(key, nan, y == y.amax(-1, keepdim=True))
    return best.int().argmax(-1)


def accept(posterior, draft):
    """(matched, bonus) lists of posterior [B, N] and draft lists."""
    matched, bonus = [], []
    for post, d in zip(posterior.tolist(), draft):
        n = 0
        while n < min(len(d), len(post)) and d[n] == post[n]:
            n += 1
        matched.append(n)
        bonus.append(post[n] if n < len(post) else -1)
    return matched, bonus
