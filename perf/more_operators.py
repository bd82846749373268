"""Performance cases of the 8-bit integer projections and of logits processing.

* ``linear``: rows x in 16 bits against a weight held in 8-bit integers.  Each
  row is quantised (a = max(max |x|, 2^-100), scale a / 127, code rint(127 x / a)),
  the product of codes is an integer, and out = sum * row scale * channel scale,
  rounded once.  ``gated``: the weight is [gate; up], out = silu(gate) * up.
* ``product``: the same with the rows' codes and scales in hand.
* ``logits``: penalties for repeated tokens, biases and grammar masks on the
  logits [B, N, V] of draft blocks.  Row i of a block knows the tokens committed
  so far and the block's drafts 0 .. i-1.  With c(v) how often v was generated:
  a token of the prompt or with c > 0 has its logit divided (if positive) or
  multiplied by the repetition penalty; then frequency * c is subtracted,
  presence where c > 0, the bias is added, and where the mask's bit is 0 the
  result is -inf.
* ``accept``: the greedy token of every row of those, how many drafts agree with
  them from the first on, and the token after these (-1 if all rows agree).
* ``count``: a batch's requests begin: nothing is known, then the prompts' and the
  generated tokens are counted.  A count is an int32, its sign bit set for tokens
  of the prompt.

``listed`` / ``draw`` give cases, ``prepare`` what a program holds before the
call, ``run`` one pass, ``work`` the bytes and operations it cannot do without
and ``exact`` the outputs in 64 bits.  Projection shapes and the vocabulary are
the package's own configuration (hidden 2560, MLP 9216, vocabulary 151936) and
generic ones around it.
"""
import sys
from pathlib import Path

import torch

own = False

BF, F16, F32, F64, I32 = torch.bfloat16, torch.float16, torch.float32, torch.float64, torch.int32
TYPES = {"bf16": BF, "fp16": F16, "fp32": F32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
PROMPT = -2 ** 31  # a count's sign bit


# ------------------------------------------------------------------ the cases

def listed():
    return [
        # one token of one chat through the stacked query|key|value projection: launch latency
        {"name": "linear-1-qkv", "kind": "linear", "x": "bf16", "out": "bf16", "M": 1, "N": 5120, "K": 2560, "gated": False},
        # a draft block through the MLP's down projection
        {"name": "linear-16-down", "kind": "linear", "x": "bf16", "out": "bf16", "M": 16, "N": 2560, "K": 9216, "gated": False},
        # a chat turn through an adapter of odd sizes
        {"name": "linear-700-odd", "kind": "linear", "x": "fp16", "out": "fp16", "M": 700, "N": 5003, "K": 1001, "gated": False},
        # a document's prompt through the MLP's gate|up projection: the matrix unit's rate
        {"name": "linear-4k-gate-up", "kind": "linear", "x": "bf16", "out": "bf16", "M": 4096, "N": 18432, "K": 2560, "gated": True},
        # a short prompt, or several draft blocks, through gate|up
        {"name": "product-120-gate-up", "kind": "product", "out": "bf16", "M": 120, "N": 18432, "K": 2560, "gated": True},
        # four draft blocks through the LM head: the weight's bytes
        {"name": "product-64-head", "kind": "product", "out": "fp32", "M": 64, "N": 151936, "K": 2560, "gated": False},
        # a draft block's logits before sampling, under a grammar
        {"name": "logits-16-grammar", "kind": "logits", "type": "fp32", "B": 1, "N": 16, "V": 151936, "mask": True, "history": 4000},
        # a served batch, one token each, a vocabulary of odd size, penalties and biases only
        {"name": "logits-b32-odd", "kind": "logits", "type": "bf16", "B": 32, "N": 1, "V": 50257, "mask": False, "history": 700},
        # a draft block of one chat with penalties: latency
        {"name": "accept-16", "kind": "accept", "type": "fp32", "B": 1, "N": 16, "V": 151936, "mask": False, "history": 900},
        # draft blocks of a served batch, all under grammars
        {"name": "accept-b32-16-grammar", "kind": "accept", "type": "bf16", "B": 32, "N": 16, "V": 151936, "mask": True, "history": 4000},
        # one chat begins
        {"name": "count-1", "kind": "count", "B": 1, "V": 151936, "prompt": 500, "generated": 16},
        # a served batch of long conversations is taken over from another engine
        {"name": "count-b32", "kind": "count", "B": 32, "V": 151936, "prompt": 16000, "generated": 2500},
    ]


def _log(rng, lo, hi):
    """A whole number spread evenly over the logarithm of [lo, hi]."""
    return min(hi, max(lo, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(["linear", "linear", "product", "logits", "accept", "count"])
    if kind in ("linear", "product"):
        while True:
            case = {"M": rng.choice([_log(rng, 1, 64), _log(rng, 1, 4096)]), "N": _log(rng, 16, 18432), "K": _log(rng, 16, 18432)}
            if rng.random() < 0.6:  # most projections are of round sizes
                case["N"], case["K"] = max(16, case["N"] // 16 * 16), max(64, case["K"] // 64 * 64)
            if case["M"] * case["N"] * case["K"] <= 4096 * 18432 * 2560:
                break
        gated = case["N"] % 2 == 0 and rng.random() < 0.3
        case |= {"kind": kind, "gated": gated, "out": rng.choice(["bf16", "bf16", "fp32", "fp16"])}
        return case | ({"x": rng.choice(["bf16", "bf16", "fp16"])} if kind == "linear" else {})
    V = rng.choice([151936, 151936, 50257, _log(rng, 100, 262144)])
    if kind == "count":
        return {"kind": kind, "B": _log(rng, 1, 32), "V": V, "prompt": _log(rng, 1, 16000), "generated": _log(rng, 1, 2500)}
    N = rng.choice([1, rng.randint(2, 15), 16])
    B = _log(rng, 1, max(1, min(64, 32 * 16 * 151936 // (2 * V * N))))
    return {"kind": kind, "type": rng.choice(["bf16", "fp32", "fp16"]), "B": B, "N": N, "V": V, "mask": rng.random() < 0.5,
            "history": _log(rng, 1, 8000)}


# -------------------------------------------------------------------- the data

def _package():
    root = str(Path(__file__).resolve().parent.parent / "dflash-mlx_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import dflash_mlx

    return dflash_mlx


def _tokens(gen, dev, B, n, V):
    """Token ids of which a few are frequent and most rare, as in text."""
    return (V * torch.rand(B, n, generator=gen, device=dev) ** 4).to(I32).clamp_max_(V - 1)


def prepare(case, seed):
    dev = torch.device("cuda", 0)
    gen = torch.Generator(device=dev).manual_seed(seed)
    pkg = _package() if own else None
    state = {"kind": case["kind"], "pkg": pkg}
    if case["kind"] in ("linear", "product"):
        M, N, K = case["M"], case["N"], case["K"]
        # hidden states: rows of different size, a few features larger than the rest
        feature = 1 + 9 * (torch.rand(K, generator=gen, device=dev) < 0.01)
        size = 0.5 + torch.rand(M, 1, generator=gen, device=dev)
        x = torch.randn(M, K, generator=gen, device=dev) * size * feature
        w = torch.randn(N, K, generator=gen, device=dev) * (0.5 + torch.rand(N, 1, generator=gen, device=dev)) * K ** -0.5
        state["w_codes"], state["w_scale"] = _quantised(w.to(BF))
        state |= {"out": TYPES[case["out"]], "gated": case["gated"]}
        if case["kind"] == "linear":
            state["x"] = x.to(TYPES[case["x"]])
        else:
            state["x_codes"], state["x_scale"] = _quantised(x.to(BF))
        if own:  # a program lays its weights out once
            state["weight"] = pkg.pack_weight_i8(state["w_codes"], state["w_scale"], gated=case["gated"])
        return state
    B, V = case["B"], case["V"]
    if case["kind"] == "count":
        state |= {"V": V, "prompt": _tokens(gen, dev, B, case["prompt"], V), "generated": _tokens(gen, dev, B, case["generated"], V)}
        for name in ("prompt", "generated"):
            n = case[name]
            less = torch.randint(0, n // 2 + 1, (B,), generator=gen, device=dev)
            state[name + "_len"] = (n - less).to(I32)
        if own:
            state["state"] = pkg.LogitsState.zeros(B, V, dev)
        return state
    N, n = case["N"], case["history"]
    logits = (3 * torch.randn(B, N, V, generator=gen, device=dev)).to(TYPES[case["type"]])
    # the drafts: the target's own choice for about half of the rows, else likely tokens
    draft = _tokens(gen, dev, B, max(N - 1, 1), V)[:, :N - 1]
    same = torch.rand(B, N - 1, generator=gen, device=dev) < 0.7
    draft = torch.where(same, logits[:, :N - 1].argmax(-1).to(I32), draft).contiguous()
    prompt, generated = _tokens(gen, dev, B, n - n // 3, V), _tokens(gen, dev, B, n // 3, V)
    # penalties of each request: some have none
    r = torch.rand(B, 3, generator=gen, device=dev)
    on = torch.rand(B, 3, generator=gen, device=dev) < 0.8
    pen = torch.where(on, torch.stack((1 + 0.4 * r[:, 0], 1.5 * r[:, 1], r[:, 2] - 0.2), 1),
                      torch.tensor([1.0, 0.0, 0.0], device=dev))
    nb = min(64, V)
    ids = torch.rand(B, V, generator=gen, device=dev).topk(nb, 1).indices.to(I32)
    values = 10 * torch.rand(B, nb, generator=gen, device=dev) - 5
    state |= {"logits": logits, "draft": draft, "mask": None}
    if case["mask"]:
        W = -(-V // 32)
        words = [torch.randint(-2 ** 31, 2 ** 31, (B, N, W), generator=gen, device=dev) for _ in range(3)]
        # a string's rows allow half of the vocabulary, a keyword's few tokens, free text everything
        form = torch.randint(0, 3, (B, N, 1), generator=gen, device=dev)
        mask = torch.where(form == 0, words[0], torch.where(form == 1, words[0] & words[1] & words[2], -1))
        if B * N > 8:  # a grammar that has no way on
            mask[-1, -1] = 0
        state["mask"] = mask.to(I32)
    if own:
        s = state["state"] = pkg.LogitsState.zeros(B, V, dev)
        s.set_penalties(repetition=pen[:, 0], presence=pen[:, 1], frequency=pen[:, 2])
        s.set_bias(ids, values)
        s.add(prompt, prompt=True)
        s.add(generated)
    else:
        state["counts"] = _counts(prompt, None, generated, None, V)
        state["pen"] = pen
        state["bias"] = torch.zeros(B, V, device=dev).scatter_(1, ids.long(), values)
    return state


def _quantised(x):
    """(int8 codes, scales) of rows."""
    x = x.float()
    a = x.abs().amax(-1).clamp_min(2.0 ** -100)
    return (127 * x / a[:, None]).round().to(torch.int8), a / 127


# -------------------------------------------------------------------- one pass

def run(state):
    if own:
        return _run_own(state)
    kind = state["kind"]
    if kind in ("linear", "product"):
        codes, scale = _quantised(state["x"]) if kind == "linear" else (state["x_codes"], state["x_scale"])
        y = (codes.float() @ state["w_codes"].float().T) * scale[:, None] * state["w_scale"]
        if state["gated"]:
            gate, up = y.chunk(2, -1)
            y = gate / (1 + torch.exp(-gate)) * up
        return y.to(state["out"])
    if kind == "count":
        return _counts(state["prompt"], state["prompt_len"], state["generated"], state["generated_len"], state["V"])
    y = _processed(state)
    if kind == "logits":
        return y.to(state["logits"].dtype)
    return _accepted(y, state["draft"])


def _run_own(s):
    pkg, kind = s["pkg"], s["kind"]
    if kind == "linear":
        return pkg.linear_i8(s["x"], s["weight"], out_dtype=s["out"])
    if kind == "product":
        return pkg.matmul_i8(s["x_codes"], s["x_scale"], s["weight"], out_dtype=s["out"])
    if kind == "count":
        s["state"].reset()
        s["state"].add(s["prompt"], s["prompt_len"], prompt=True)
        s["state"].add(s["generated"], s["generated_len"])
        return s["state"].counts
    if kind == "logits":
        return pkg.process_logits(s["logits"], s["state"], s["draft"], mask=s["mask"])
    return pkg.greedy_accept(s["logits"], s["draft"], state=s["state"], mask=s["mask"])


# -------------------------------------------------------------- the plain forms

def _counts(prompt, prompt_len, generated, generated_len, V):
    """int32 [B, V]: how often a token was generated, the sign bit set where the prompt has it."""
    def occurrences(tokens, lens):
        at = torch.arange(tokens.shape[1], device=tokens.device)
        live = torch.ones_like(tokens) if lens is None else (at < lens[:, None]).to(I32)
        return torch.zeros(len(tokens), V, dtype=I32, device=tokens.device).scatter_add_(1, tokens.long(), live)

    return occurrences(generated, generated_len) + torch.where(occurrences(prompt, prompt_len) > 0, PROMPT, 0).to(I32)


def _processed(s):
    """The processed logits in 32 bits."""
    y, counts, draft = s["logits"].float(), s["counts"], s["draft"]
    B, N, V = y.shape
    rep, pres, freq = (p[:, None, None] for p in s["pen"].unbind(1))
    made = (counts & (2 ** 31 - 1))[:, None].expand(B, N, V).contiguous()
    for i in range(1, N):  # draft i - 1 is known to the rows from i on
        b = torch.arange(B, device=y.device)
        made[b, i:, draft[:, i - 1].long()] += 1
    seen = (made > 0) | (counts < 0)[:, None]
    y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
    y = y - freq * made - torch.where(made > 0, pres, 0) + s["bias"][:, None]
    if s["mask"] is not None:
        v = torch.arange(V, device=y.device)
        y = y.masked_fill((s["mask"][:, :, v // 32] >> (v % 32)) & 1 == 0, -torch.inf)
    return y


def _accepted(y, draft):
    """(greedy tokens, lowest index on ties, agreeing drafts, the token after them)."""
    B, N, V = y.shape
    best = y.amax(-1, keepdim=True)
    post = torch.where(y == best, torch.arange(V, device=y.device), V).amin(-1)
    agree = (draft[:, :N] == post[:, :draft.shape[1]]).to(I32).cumprod(1).sum(1)
    padded = torch.cat((post, torch.full_like(post[:, :1], -1)), 1)
    return post.to(I32), agree.to(I32), padded.gather(1, agree[:, None].long())[:, 0].to(I32)


# ------------------------------------------------------------------------ work

def work(case):
    if case["kind"] in ("linear", "product"):
        M, N, K = case["M"], case["N"], case["K"]
        cols = N // 2 if case["gated"] else N
        rows = M * K * SIZE[case["x"]] if case["kind"] == "linear" else M * (K + 4)
        return {"bytes": rows + N * (K + 4) + M * cols * SIZE[case["out"]], "flops": 2 * M * N * K}
    B, V = case["B"], case["V"]
    if case["kind"] == "count":  # the tokens, a read and a write of each one's count, which of them are known
        tokens = B * (case["prompt"] + case["generated"]) * 3 // 4
        return {"bytes": 12 * tokens + B * V // 8, "flops": tokens}
    N = case["N"]
    logits = B * N * V * SIZE[case["type"]]
    known = B * V // 8 + 8 * B * (case["history"] + 64)  # which tokens are known; their counts and biases
    mask = B * N * V // 8 if case["mask"] else 0
    return {"bytes": logits * (2 if case["kind"] == "logits" else 1) + known + mask, "flops": B * N * V}


# ----------------------------------------------------------------------- exact

def exact(case, seed):
    """run's outputs from the definitions in 64 bits."""
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if s["kind"] in ("linear", "product"):
        if s["kind"] == "linear":
            x = s["x"].to(F64)
            largest = x.abs().max(1, keepdim=True).values.clamp(min=2.0 ** -100)
            rows = torch.round(x * 127 / largest) * (largest / 127)
        else:
            rows = s["x_codes"].to(F64) * s["x_scale"].to(F64).unsqueeze(1)
        out = []
        for part in range(0, len(s["w_codes"]), 16384):  # some channels at a time
            channels = s["w_codes"][part:part + 16384].to(F64) * s["w_scale"][part:part + 16384].to(F64).unsqueeze(1)
            out.append(torch.matmul(rows, channels.t()))
        y = torch.cat(out, 1)
        if s["gated"]:
            half = y.shape[1] // 2
            y = y[:, :half] * torch.sigmoid(y[:, :half]) * y[:, half:]
        return y
    if s["kind"] == "count":
        B, V = len(s["prompt"]), s["V"]
        rows = []
        for b in range(B):
            p = s["prompt"][b, :int(s["prompt_len"][b])]
            g = s["generated"][b, :int(s["generated_len"][b])]
            row = torch.bincount(g, minlength=V)
            row[p.unique().long()] += PROMPT
            rows.append(row)
        return torch.stack(rows).to(I32)
    logits, draft = s["logits"], s["draft"]
    B, N, V = logits.shape
    bit = torch.arange(V, device=logits.device) % 32
    word = torch.arange(V, device=logits.device).div(32, rounding_mode="floor")
    values, tokens = [], torch.zeros(B, N, dtype=I32, device=logits.device)
    for b in range(B):
        repetition, presence, frequency = s["pen"][b].to(F64).unbind()
        in_prompt = s["counts"][b] < 0
        made = torch.where(in_prompt, s["counts"][b].long() - PROMPT, s["counts"][b].long()).to(F64)
        for i in range(N):
            if i:
                made[draft[b, i - 1].long()] += 1
            row = logits[b, i].to(F64)
            factor = torch.where(row > 0, 1 / repetition, repetition)
            row = torch.where(in_prompt | (made > 0), row * factor, row)
            row = row - made * frequency - (made > 0) * presence + s["bias"][b].to(F64)
            if s["mask"] is not None:
                allowed = (s["mask"][b, i][word].long() >> bit) & 1
                row = torch.where(allowed == 1, row, torch.full_like(row, -torch.inf))
            tokens[b, i] = torch.nonzero(row == row.max())[0, 0]
            if s["kind"] == "logits":
                values.append(row)
    if s["kind"] == "logits":
        return torch.stack(values).view(B, N, V)
    matched, bonus = [], []
    for b in range(B):
        post, block = tokens[b].tolist(), draft[b].tolist()
        n = 0
        while n < len(block) and block[n] == post[n]:
            n += 1
        matched.append(n)
        bonus.append(post[n] if n < N else -1)
    as_tensor = lambda v: torch.tensor(v, dtype=I32, device=logits.device)  # noqa: E731
    return tokens, as_tensor(matched), as_tensor(bonus)
