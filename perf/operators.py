"""Performance cases of the 8-bit key/value cache's operators.

A cache holds, per sequence and key/value head, complete blocks of 64 tokens
in 8 bits (int8 or e4m3) with one fp32 scale a block for the keys and one for
the values, and the latest two blocks of positions in bf16 (the tail, position
p in slot p % 128).  With L committed tokens the blocks below L // 64 are read
from their codes and the rest from the tail; an append quantises a block from
the tail once every token of it is committed.

* ``append``: query/key RMSNorm, rotary and the append of T draft tokens, or of
  a prompt; the positions around it are read back as the values they stand for;
* ``read``: positions of the cache back in bf16;
* ``verify``: gated attention of 1 to 16 new tokens a sequence;
* ``prompt``: gated attention of a prompt's rows.

``listed`` / ``draw`` give cases, ``prepare`` what a program holds before the
call, ``run`` one pass, ``work`` the bytes and operations it cannot do
without and ``exact`` the outputs in 64 bits.  Head counts, head width and
rotary are the package's own configuration (16 query and 4 key/value heads of
128) and generic ones around it.
"""
import sys
from pathlib import Path

import torch

own = False

BF, F32, F64, I32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
D, BLOCK, SLOTS = 128, 64, 128
ROT, THETA, EPS = 32, 100000.0, 1e-6
DTYPES = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one chat, one token a step, a short history: launch latency
        {"name": "verify-1-short", "kind": "verify", "type": "e4m3", "B": 1, "T": 1, "Hq": 16, "Hkv": 4, "past": 500},
        # a 16-token draft block of one chat after a 4k history: the hybrid target's verify step
        {"name": "verify-16-4k", "kind": "verify", "type": "e4m3", "B": 1, "T": 16, "Hq": 16, "Hkv": 4, "past": 4096},
        # a served batch of 32 chats of different lengths, one token each
        {"name": "verify-1-b32", "kind": "verify", "type": "int8", "B": 32, "T": 1, "Hq": 16, "Hkv": 4, "past": 8191},
        # a draft block at the end of a book-length history: the cache's bytes
        {"name": "verify-16-128k", "kind": "verify", "type": "int8", "B": 1, "T": 16, "Hq": 16, "Hkv": 4, "past": 131000},
        # short draft blocks of a dozen sequences, as many key/value heads as query heads
        {"name": "verify-5-b12", "kind": "verify", "type": "e4m3", "B": 12, "T": 5, "Hq": 8, "Hkv": 8, "past": 3001},
        # a chat turn's prompt after an earlier conversation, of odd length
        {"name": "prompt-600", "kind": "prompt", "type": "int8", "T": 600, "Hq": 16, "Hkv": 4, "past": 1000},
        # a document's prompt
        {"name": "prompt-4k", "kind": "prompt", "type": "e4m3", "T": 4096, "Hq": 16, "Hkv": 4, "past": 0},
        # a prompt that goes on after a long cached prefix
        {"name": "prompt-2k-after-14k", "kind": "prompt", "type": "e4m3", "T": 2048, "Hq": 16, "Hkv": 4, "past": 14336},
        # a served batch's new tokens into their caches, the last blocks read back
        {"name": "append-1-b32", "kind": "append", "type": "int8", "B": 32, "T": 1, "Hq": 16, "Hkv": 4, "past": 8191},
        # a document's keys and values into the cache, all of it read back
        {"name": "append-prompt-4k", "kind": "append", "type": "e4m3", "B": 1, "T": 4096, "Hq": 16, "Hkv": 4, "past": 0},
        # the caches of four chats handed on to another engine in bf16
        {"name": "read-b4-8k", "kind": "read", "type": "int8", "B": 4, "Hkv": 4, "past": 8190, "start": 0, "count": 8190},
        # a stretch of one conversation, cut out of the middle
        {"name": "read-odd", "kind": "read", "type": "e4m3", "B": 1, "Hkv": 4, "past": 1000, "start": 77, "count": 901},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "prompt", "append", "read"])
    case = {"kind": kind, "type": rng.choice(["int8", "e4m3"])}
    hq, hkv = rng.choice([(16, 4), (16, 4), (8, 2), (16, 8), (8, 8), (12, 4), (4, 1)])
    if kind == "verify":
        b = _log(rng, 1, 32)
        return {**case, "B": b, "T": rng.choice([1, rng.randint(2, 15), 16]), "Hq": hq, "Hkv": hkv,
                "past": _log(rng, 1, 131000 // b)}
    if kind == "prompt":
        past = rng.choice([0, _log(rng, 1, 8192)])
        return {**case, "T": _log(rng, 17, 4096 if past < 2048 else 2048), "Hq": hq, "Hkv": hkv, "past": past}
    if kind == "append":
        if rng.random() < 0.5:
            return {**case, "B": _log(rng, 1, 32), "T": rng.choice([1, rng.randint(2, 15), 16]), "Hq": hq, "Hkv": hkv,
                    "past": _log(rng, 1, 8192)}
        b = rng.choice([1, 1, 2])
        return {**case, "B": b, "T": _log(rng, 17, 4096 // b), "Hq": hq, "Hkv": hkv, "past": 0}
    b = rng.randint(1, 4)
    past = _log(rng, 2, 8190)
    start = rng.randint(0, past // 2)
    return {**case, "B": b, "Hkv": hkv, "past": past, "start": start, "count": rng.randint(1, past - start)}


# -------------------------------------------------------------------- the data

def _scale(x, kind):
    """(scale, codes' multiplier) of blocks by their largest magnitude, over the last two axes."""
    a = x.abs().amax((-2, -1)).clamp_min(2.0 ** -100)
    if kind == "int8":
        return a / 127, 127 / a
    m, e = torch.frexp(a)  # a = m 2^e, m in [1/2, 1): 448 = 0.875 * 2^9
    s = torch.ldexp(torch.ones_like(a), e - 9 + (m > 0.875).int())
    return s, 1 / s


def _codes(x, mul, kind):
    """uint8 codes of x (32 bits) under its blocks' multipliers."""
    y = x * mul[..., None, None]
    if kind == "int8":
        return y.round().clamp(-127, 127).to(torch.int8).view(torch.uint8)
    return y.to(torch.float8_e4m3fn).view(torch.uint8)


def _values(codes, scale, kind):
    """The values that blocks of uint8 codes stand for, in the scale's type."""
    return codes.view(DTYPES[kind]).to(F32).to(scale.dtype) * scale[..., None, None]


def _gated(out, proj, Hq):
    """out [B, T, Hq, D] times the sigmoid of the gates in the projection rows."""
    B, T = out.shape[:2]
    gate = proj[:, :, :2 * Hq * D].view(B, T, Hq, 2, D)[:, :, :, 1].to(out.dtype)
    return (out * (1 / (1 + torch.exp(-gate)))).reshape(B, T, Hq * D)


def _lens(case, gen, dev):
    """Committed lengths: the first sequence's is `past`, the others' between half of it and all."""
    past, B = case["past"], case.get("B", 1)
    less = torch.randint(0, past // 2 + 1, (B,), generator=gen, device=dev)
    less[0] = 0
    return (past - less).to(I32)


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    kind, B, T, Hkv = case["kind"], case.get("B", 1), case.get("T", 0), case["Hkv"]
    Hq = case.get("Hq", Hkv)
    cap = -(-(case["past"] + max(T, 16)) // BLOCK) * BLOCK
    nb = cap // BLOCK
    rand = lambda *s: torch.randn(*s, generator=gen, device=dev)  # noqa: E731
    lens = _lens(case, gen, dev)
    # what the cache holds: keys after their norm, values; a sequence's own spread of magnitudes
    k = (rand(B, Hkv, nb, BLOCK, D) * (0.5 + torch.rand(B, Hkv, nb, 1, 1, generator=gen, device=dev))).to(BF)
    v = (rand(B, Hkv, nb, BLOCK, D) * (0.5 + torch.rand(B, Hkv, nb, 1, 1, generator=gen, device=dev))).to(BF)
    ends = lens.long() + (T if kind == "prompt" else 0)  # a prompt's rows are in the cache before its attention
    held = ends + (T if kind == "verify" else 0)         # so are a draft block's
    state = {"lens": lens, "k_codes": None, "v_codes": None}
    slot_at = torch.arange(SLOTS, device=dev)[None]
    for name, x in (("k", k), ("v", v)):
        s, mul = _scale(x.float(), case["type"])
        c = _codes(x.float(), mul, case["type"])
        # the tail: slot j holds the latest position p = j mod 128 below the held length
        pos = held[:, None] - 1 - (held[:, None] - 1 - slot_at) % SLOTS
        rows = x.view(B, Hkv, cap, D)[torch.arange(B, device=dev)[:, None], :, pos.clamp_min(0)]  # [B, slot, Hkv, D]
        rows = rows.masked_fill((pos < 0)[..., None, None], 0).transpose(1, 2)
        live = (torch.arange(nb, device=dev)[None] < (ends // BLOCK)[:, None])[:, None]
        state[name + "_scale"] = torch.where(live, s, 0).contiguous()
        c = torch.where(live[..., None, None], c, 0)
        c = c.view(B, Hkv, cap, D) if name == "k" else c.transpose(-2, -1)
        state[name + "_codes"] = c.contiguous().view(DTYPES[case["type"]])
        state["tail_k" if name == "k" else "tail_vt"] = (rows if name == "k" else rows.transpose(2, 3)).contiguous()
    state |= {"kind": kind, "type": case["type"], "T": T, "Hq": Hq, "prompt": kind == "append" and T > 16}
    if kind == "read":
        state |= {"start": case["start"], "count": case["count"]}
    else:
        state["proj"] = rand(B, T, (2 * Hq + 2 * Hkv) * D).to(BF)
    if kind in ("verify", "prompt"):
        state["q"] = (1.5 * rand(B, T, Hq, D)).to(BF)
    if kind == "append":
        state["q_norm"] = (1 + 0.1 * rand(D)).to(BF)
        state["k_norm"] = (1 + 0.1 * rand(D)).to(BF)
        # the positions read back: from the block before the first new token on
        state["start"] = ((lens // BLOCK - 1).clamp_min(0) * BLOCK).to(I32)
        state["count"] = T + 2 * BLOCK
        state["after"] = lens + T if state["prompt"] else lens
    if own:  # the handle that a program keeps for its cache
        state["cache"] = _package().QuantizedKVCache(state["k_codes"], state["v_codes"], state["k_scale"],
                                                     state["v_scale"], state["tail_k"], state["tail_vt"])
    return state


def _package():
    root = str(Path(__file__).resolve().parent.parent / "dflash-mlx_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import dflash_mlx

    return dflash_mlx


# -------------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind == "read":
        return _plain_read(state, state["lens"], state["start"], state["count"])
    if kind == "append":
        return (_plain_append(state), state["tail_k"], state["tail_vt"],
                *_plain_read(state, state["after"], state["start"], state["count"]))
    return _plain_attention(state)


def _run_own(s):
    pkg, cache = _package(), s["cache"]
    if s["kind"] == "read":
        return pkg.kv_read_q8(cache, s["lens"], s["count"], start=s["start"])
    if s["kind"] == "append":
        q = pkg.attn_prep_q8(s["proj"], s["q_norm"], s["k_norm"], s["lens"], cache, num_heads=s["Hq"], rot_dims=ROT,
                             rope_base=THETA, eps=EPS, prompt=s["prompt"])
        return (q, cache.tail_k, cache.tail_vt,
                *pkg.kv_read_q8(cache, s["after"], s["count"], start=s["start"]))
    attend = pkg.attn_verify_q8 if s["kind"] == "verify" else pkg.attn_prefill_q8
    return attend(s["q"], cache, s["lens"], s["proj"])


# -------------------------------------------------------------- the plain forms

def _held(s, done):
    """All keys and values in 32 bits, [B, Hkv, positions, D]: codes below
    `done` blocks [B], the tail's slots from there on."""
    B, Hkv, cap, _ = s["k_codes"].shape
    k = _values(s["k_codes"].view(B, Hkv, -1, BLOCK, D), s["k_scale"], s["type"]).view(B, Hkv, cap, D)
    v = _values(s["v_codes"], s["v_scale"], s["type"]).transpose(-2, -1).reshape(B, Hkv, cap, D)
    # positions from block `done` on: 128 of them, all in the tail
    pos = done.long()[:, None] * BLOCK + torch.arange(SLOTS, device=k.device)[None]
    b = torch.arange(B, device=k.device)[:, None].expand_as(pos)[pos < cap]
    p = pos[pos < cap]
    k[b, :, p] = s["tail_k"][b, :, p % SLOTS].float()
    v[b, :, p] = s["tail_vt"][b, :, :, p % SLOTS].float()
    return k, v


def _plain_read(s, lens, start, count):
    Hkv, cap = s["k_codes"].shape[1:3]
    at = (start[:, None] if torch.is_tensor(start) else start) + torch.arange(count, device=lens.device)[None]
    at = at.expand(len(lens), count).long()
    b, p = torch.arange(len(lens), device=lens.device)[:, None], at.clamp_max(cap - 1)
    k = s["k_codes"].view(torch.uint8)[b, :, p].view(DTYPES[s["type"]]).float() * s["k_scale"][b, :, p // BLOCK, None]
    v = (s["v_codes"].view(torch.uint8)[b, :, p // BLOCK, :, p % BLOCK].view(DTYPES[s["type"]]).float()
         * s["v_scale"][b, :, p // BLOCK, None])  # [B, count, Hkv, D]
    tail = (p // BLOCK >= (lens // BLOCK)[:, None])[..., None, None]
    live = (at < lens[:, None])[..., None, None]
    k = torch.where(tail, s["tail_k"][b, :, p % SLOTS].float(), k)
    v = torch.where(tail, s["tail_vt"][b, :, :, p % SLOTS].float(), v)
    return tuple(torch.where(live, x, 0).to(BF).transpose(1, 2).contiguous() for x in (k, v))


def _plain_attention(s):
    q, T, Hq, lens = s["q"].float(), s["T"], s["Hq"], s["lens"].long()
    done = (lens + (T if s["kind"] == "prompt" else 0)) // BLOCK
    k, v = _held(s, done)
    B, Hkv, cap, _ = k.shape
    q = q.view(B, T, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4)
    score = torch.matmul(q, k[:, :, None].transpose(-2, -1)) * D ** -0.5  # [B, Hkv, rep, T, positions]
    last = lens[:, None] + torch.arange(T, device=q.device)[None]
    seen = (torch.arange(cap, device=q.device) <= last[..., None])[:, None, None]
    score = score.masked_fill_(~seen, float("-inf"))
    w = torch.exp(score.sub_(score.amax(-1, keepdim=True)))
    out = torch.matmul(w, v[:, :, None]) / w.sum(-1, keepdim=True)
    return _gated(out.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, D), s["proj"], Hq).to(BF)


def _norm_rotate(x, weight, pos):
    """RMSNorm over the head's features, then rotary of the first ROT at positions pos [B, T]."""
    x = x.float()
    x = x * (1 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS)) * weight.float()
    inv = THETA ** (-torch.arange(0, ROT, 2, device=x.device, dtype=F64) / ROT)
    ang = pos.double()[:, :, None, None] * inv
    c, s = torch.cos(ang).float(), torch.sin(ang).float()
    a, b = x[..., :ROT // 2], x[..., ROT // 2:ROT]
    return torch.cat((a * c - b * s, b * c + a * s, x[..., ROT:]), -1).to(BF)


def _plain_append(s):
    """Queries; the cache's tensors are updated in place."""
    proj, Hq, T = s["proj"], s["Hq"], s["T"]
    Hkv, dev = s["k_codes"].shape[1], proj.device
    B, lens = proj.shape[0], s["lens"].long()
    pos = lens[:, None] + torch.arange(T, device=dev)[None]
    q = _norm_rotate(proj[..., :2 * Hq * D].view(B, T, Hq, 2, D)[:, :, :, 0], s["q_norm"], pos)
    k = _norm_rotate(proj[..., 2 * Hq * D:(2 * Hq + Hkv) * D].view(B, T, Hkv, D), s["k_norm"], pos)
    v = proj[..., (2 * Hq + Hkv) * D:].view(B, T, Hkv, D)
    # the blocks that this append may complete: from the one before the first new token on
    first = (lens // BLOCK - 1).clamp_min(0)
    n = T // BLOCK + 3
    blocks = first[:, None] + torch.arange(n, device=dev)[None]
    at = (blocks[:, :, None] * BLOCK + torch.arange(BLOCK, device=dev)).view(B, -1)  # [B, n * BLOCK]
    b = torch.arange(B, device=dev)[:, None]
    end = lens + T if s["prompt"] else lens
    total = s["k_scale"].shape[2]
    write = ((blocks < (end // BLOCK)[:, None]) & (blocks < total)
             & ((blocks >= (lens // BLOCK)[:, None]) | (lens % BLOCK <= 16)[:, None]))
    bw = b.expand_as(blocks)[write]
    fresh = (at >= lens[:, None]) & (at < lens[:, None] + T)
    new_at = (at - lens[:, None]).clamp(0, T - 1)
    k_rows = torch.where(fresh[..., None, None], k[b, new_at], s["tail_k"][b, :, at % SLOTS])  # [B, at, Hkv, D]
    v_rows = torch.where(fresh[..., None, None], v[b, new_at], s["tail_vt"][b, :, :, at % SLOTS])
    k_rows = k_rows.view(B, n, BLOCK, Hkv, D).transpose(2, 3).float()
    v_rows = v_rows.view(B, n, BLOCK, Hkv, D).permute(0, 1, 3, 4, 2).float()
    k_codes = s["k_codes"].view(torch.uint8).view(B, Hkv, total, BLOCK, D)
    v_codes = s["v_codes"].view(torch.uint8)
    ks, kmul = _scale(k_rows, s["type"])
    vs, vmul = _scale(v_rows, s["type"])
    k_codes[bw, :, blocks[write]] = _codes(k_rows, kmul, s["type"])[write]
    v_codes[bw, :, blocks[write]] = _codes(v_rows, vmul, s["type"])[write]
    s["k_scale"][bw, :, blocks[write]] = ks[write]
    s["v_scale"][bw, :, blocks[write]] = vs[write]
    # the tail keeps the latest two blocks' new tokens
    keep = (pos >= (((lens + T) // BLOCK - 1) * BLOCK)[:, None]) if s["prompt"] else torch.ones_like(pos, dtype=torch.bool)
    bt = b.expand_as(pos)[keep]
    s["tail_k"][bt, :, pos[keep] % SLOTS] = k[keep]
    s["tail_vt"][bt, :, :, pos[keep] % SLOTS] = v[keep]
    return q


# ------------------------------------------------------------------- what it takes

def work(case):
    kind, B, T, Hkv = case["kind"], case.get("B", 1), case.get("T", 0), case["Hkv"]
    Hq, past = case.get("Hq", Hkv), case["past"]
    tokens = past + (B - 1) * 0.75 * past  # committed, over the batch
    rows = B * T
    if kind == "read":
        n = B * case["count"] * Hkv * 2 * D
        return {"bytes": 3 * n, "flops": n}
    if kind == "append":
        back = (B * (BLOCK if T <= 16 else T)) * Hkv * 2 * D  # read back: codes in, bf16 out
        moved = rows * (2 * Hq + 2 * Hkv) * D * 2 + rows * Hkv * 2 * D
        return {"bytes": moved + 3 * back, "flops": rows * (Hq + Hkv) * D * 8}
    seen = tokens + rows if kind == "verify" else past + T
    pairs = T * tokens + B * T * (T + 1) / 2
    return {"bytes": seen * Hkv * 2 * D + rows * Hq * D * 6, "flops": 4 * pairs * Hq * D}


# ------------------------------------------------------------------- in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    if s["kind"] == "append":
        return _exact_append(s)
    if s["kind"] == "read":
        k, v = zip(*(_exact_read(s, b, int(n), s["start"], s["count"]) for b, n in enumerate(s["lens"].tolist())))
        return torch.stack(k), torch.stack(v)
    T, Hq = s["T"], s["Hq"]
    rep = Hq // case["Hkv"]
    out = torch.empty(len(s["lens"]), T, Hq, D, dtype=F64, device=s["q"].device)
    for b, n in enumerate(s["lens"].tolist()):
        k, v = _exact_held(s, b, (n + (T if s["kind"] == "prompt" else 0)) // BLOCK, n + T)
        later = torch.arange(n + T, device=k.device)[None] > (n + torch.arange(T, device=k.device))[:, None]
        for h in range(Hq):
            p = torch.mm(s["q"][b, :, h].double(), k[h // rep].t()) / D ** 0.5
            p = torch.softmax(p.masked_fill_(later, float("-inf")), -1)
            out[b, :, h] = torch.mm(p, v[h // rep])
    return _gated(out, s["proj"], Hq)


def _exact_held(s, b, done, n):
    """Sequence b's first n keys and values [Hkv, n, D] in 64 bits."""
    cut = min(done * BLOCK, n)
    k = s["k_codes"][b, :, :cut].to(F32).double() * s["k_scale"][b, :, :, None].double().repeat_interleave(BLOCK, 1)[:, :cut]
    v = s["v_codes"][b].to(F32).double() * s["v_scale"][b, :, :, None, None].double()
    v = v.transpose(2, 3).flatten(1, 2)[:, :cut]
    slots = torch.arange(cut, n, device=k.device) % SLOTS
    return (torch.cat((k, s["tail_k"][b, :, slots].double()), 1),
            torch.cat((v, s["tail_vt"][b, :, :, slots].double().transpose(1, 2)), 1))


def _exact_read(s, b, n, start, count):
    k, v = _exact_held(s, b, n // BLOCK, n)
    pad = max(0, start + count - n)
    return tuple(torch.nn.functional.pad(x, (0, 0, 0, pad))[:, start:start + count] for x in (k, v))


def _exact_quantised(x, kind):
    """(codes, scale) of one block [..] of bf16 values."""
    a = max(x.abs().max().item(), 2.0 ** -100)
    if kind == "int8":
        return torch.round(x * 127 / a).to(torch.int8), a / 127
    step = 2.0 ** -120
    while a / step > 448:
        step *= 2
    return (x / step).float().to(torch.float8_e4m3fn), step


def _exact_append(s):
    proj, T, Hq, Hkv = s["proj"], s["T"], s["Hq"], s["k_codes"].shape[1]
    dev = proj.device
    q_all, reads = [], []
    inv = THETA ** (-2 * torch.arange(ROT // 2, device=dev, dtype=F64) / ROT)

    def turned(x, w, n):
        x = x.double()
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * w.double()
        z = torch.complex(x[..., :ROT // 2], x[..., ROT // 2:ROT])
        ang = (n + torch.arange(T, device=dev, dtype=F64))[:, None] * inv
        z = z * torch.polar(torch.ones_like(ang), ang)[:, None]
        return torch.cat((z.real, z.imag, x[..., ROT:]), -1)

    for b, n in enumerate(s["lens"].tolist()):
        row = proj[b].view(T, -1, D)
        q_all.append(turned(row[:, 0:2 * Hq:2], s["q_norm"], n))
        k = turned(row[:, 2 * Hq:2 * Hq + Hkv], s["k_norm"], n).to(BF)  # the tail's type
        v = row[:, 2 * Hq + Hkv:]
        old = max(0, n // BLOCK - 1) * BLOCK  # the first position that the tail still holds
        slots = torch.arange(old, n, device=dev) % SLOTS
        k = torch.cat((s["tail_k"][b][:, slots], k.transpose(0, 1)), 1)  # positions old .. n + T
        v = torch.cat((s["tail_vt"][b][:, :, slots].transpose(1, 2), v.transpose(0, 1)), 1)
        end = n + T if s["prompt"] else n
        for j in range(old // BLOCK, end // BLOCK):
            if j < n // BLOCK and n % BLOCK > 16:
                continue
            at = slice(j * BLOCK - old, (j + 1) * BLOCK - old)
            for h in range(Hkv):
                c, s["k_scale"][b, h, j] = _exact_quantised(k[h, at].double(), s["type"])
                s["k_codes"].view(torch.uint8)[b, h, j * BLOCK:(j + 1) * BLOCK] = c.view(torch.uint8)
                c, s["v_scale"][b, h, j] = _exact_quantised(v[h, at].double(), s["type"])
                s["v_codes"].view(torch.uint8)[b, h, j] = c.view(torch.uint8).t()
        kept = max(n, ((n + T) // BLOCK - 1) * BLOCK) if s["prompt"] else n
        slots = torch.arange(kept, n + T, device=dev) % SLOTS
        s["tail_k"][b, :, slots] = k[:, kept - old:]
        s["tail_vt"][b, :, :, slots] = v[:, kept - old:].transpose(1, 2)
        reads.append(_exact_read(s, b, int(s["after"][b]), int(s["start"][b]), s["count"]))
    return (torch.stack(q_all), s["tail_k"].double(), s["tail_vt"].double(),
            torch.stack([r[0] for r in reads]), torch.stack([r[1] for r in reads]))
