"""Measured cases of serving from a paged cache (micro_engram_fork_b200.ops.paged).

The cache of a layer is two tensors of pages [P, Hk, page, D]; position p of sequence b lies in row p % page of page
block_table[b, p // page]. A call brings the new tokens of a batch, packed: sequence b has the tokens
cu_seqlens[b] .. cu_seqlens[b + 1], its last ones, and seq_lens[b] tokens in all.

  append   the fused q/k/v projection of the new tokens: RMS norm of each head, rotation of q and k by the
           position, k and v into their pages, q out
  attend   attention of the new tokens over all that their sequence has in the cache (causal, with a
           sliding window where the layer has one): output and log-sum-exp of each row

`run` computes an operator in its plain form, in 32 bits, where `own` is false, and through the
framework's entry points where it is true. `exact` computes it from the definition in 64 bits.
"""
import math
import random

import torch

own = False

EPS = 1e-6
# the layers of the benchmark's decoder and of the tests' small one, and shapes between them
SLIDING = {"hq": 32, "hk": 16, "d": 256, "window": 1024}
GLOBAL = {"hq": 32, "hk": 4, "d": 512, "window": 0}
SMALL_SLIDING = {"hq": 4, "hk": 2, "d": 64, "window": 64}
SMALL_GLOBAL = {"hq": 4, "hk": 1, "d": 128, "window": 0}
OTHERS = [
    {"hq": 8, "hk": 8, "d": 128, "window": 0},
    {"hq": 15, "hk": 3, "d": 128, "window": 512},
    {"hq": 24, "hk": 4, "d": 256, "window": 0},
    {"hq": 16, "hk": 1, "d": 64, "window": 0},
]


def listed():
    """A case has `seqs` sequences; each has between ctx[0] and ctx[1] tokens in the cache before the call and brings
    between new[0] and new[1] tokens (`mix` seeds the lengths)."""
    return [
        # one request being answered: the next token of a sliding layer, bound by latency
        _case("append one token", "append", SLIDING, 1, (1000, 1000), (1, 1), 64),
        # a server's batch of answers in a global layer, whose values are its keys before their norm
        _case("append batch of answers", "append", GLOBAL, 96, (200, 9000), (1, 1), 64),
        # prompts of several requests, ragged, in the small decoder, on short pages
        _case("append ragged prompts", "append", SMALL_SLIDING, 23, (0, 300), (1, 401), 16),
        # a chunk of a long prompt
        _case("append chunk", "append", SLIDING, 1, (4096, 4096), (8192, 8192), 64),
        # one request: its next token in a sliding layer, and in a global layer over a long document
        _case("answer one, sliding", "attend", SLIDING, 1, (5000, 5000), (1, 1), 64),
        _case("answer one, long document", "attend", GLOBAL, 1, (131071, 131071), (1, 1), 64),
        # a server's batch of answers of any length
        _case("answers, sliding", "attend", SLIDING, 128, (30, 9000), (1, 1), 64),
        _case("answers, global", "attend", GLOBAL, 64, (100, 16000), (1, 1), 64),
        # a few tokens a sequence: drafts that are checked at once
        _case("drafts, global", "attend", GLOBAL, 16, (500, 6000), (3, 6), 32),
        # chunks of prompts and answers in one batch, five heads a key head, short pages
        _case("mixed batch, odd", "attend", OTHERS[1], 19, (0, 3000), (1, 333), 16),
        # a chunk of a long prompt
        _case("chunk, sliding", "attend", SLIDING, 1, (6000, 6000), (4096, 4096), 64),
        _case("chunk, global", "attend", GLOBAL, 1, (14000, 14000), (2048, 2048), 128),
    ]


def _case(name, op, layer, seqs, ctx, new, page, mix=1):
    return {"name": name, "op": op, **layer, "seqs": seqs, "ctx_lo": ctx[0], "ctx_hi": ctx[1], "new_lo": new[0], "new_hi": new[1],
            "page": page, "mix": mix}


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend"])
    layer = rng.choice([SLIDING, GLOBAL, SLIDING, GLOBAL, SMALL_SLIDING, SMALL_GLOBAL, *OTHERS])
    seqs = _log(rng, 1, 128)
    kind = rng.choice(["answers", "drafts", "chunks"])
    new_hi = {"answers": 1, "drafts": rng.randint(2, 8), "chunks": _log(rng, 9, max(10, 4096 // seqs))}[kind]
    new_lo = 1 if kind != "chunks" else rng.randint(1, new_hi)
    ctx_hi = _log(rng, 1, 131072 if op == "attend" else 16384)
    # the cache of a call and its products stay below those of the largest listed cases
    row = 4 * layer["hk"] * layer["d"]
    ctx_hi = max(1, min(ctx_hi, (3 << 29) // (row * seqs)))
    if op == "attend":
        pairs = 2048 * 15000 * 512 * 32
        ctx_hi = max(1, min(ctx_hi, pairs // (seqs * new_hi * layer["d"] * layer["hq"])))
    case = _case("", op, layer, seqs, (rng.randint(0, ctx_hi), ctx_hi), (new_lo, new_hi), rng.choice([16, 32, 64, 64, 128]), rng.randint(2, 1 << 30))
    del case["name"]
    return case


def _lengths(case):
    """[(tokens in the cache before the call, new tokens)] of the sequences."""
    r = random.Random(case["mix"])
    return [(r.randint(case["ctx_lo"], case["ctx_hi"]), r.randint(case["new_lo"], case["new_hi"])) for _ in range(case["seqs"])]


def _first_key(case, ctx):
    """The first position that any of the new tokens sees."""
    return max(0, ctx - case["window"] + 1) if case["window"] else 0


# ------------------------------------------------------------------------------- inputs
def _kv_eq(case):
    """Global layers of the decoder take their values from the raw keys."""
    return case["window"] == 0


def _inv_freq(case):
    d = case["d"]
    if case["window"]:
        return 10000.0 ** (-torch.arange(0, d, 2).float() / d)
    rot = d // 8  # a quarter of the dimensions rotates
    f = 1000000.0 ** (-torch.arange(0, 2 * rot, 2).float() / d)
    return torch.cat([f, torch.zeros(d // 2 - rot)])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, device="cuda", generator=gen)  # noqa: E731
    r = random.Random(seed)
    hq, hk, d, page = case["hq"], case["hk"], case["d"], case["page"]
    lens = _lengths(case)
    cu = [0]
    for _, new in lens:
        cu.append(cu[-1] + new)
    width = max((ctx + new + page - 1) // page for ctx, new in lens)
    # pages of a sequence that lie before its window are given back: no page for them
    first = [_first_key(case, ctx) // page for ctx, _ in lens]
    used = [(ctx + new + page - 1) // page - a for (ctx, new), a in zip(lens, first)]
    pages = sum(used) + 3
    order = list(range(pages))
    r.shuffle(order)
    rows, at = [], 0
    for a, n in zip(first, used):
        rows.append([-1] * a + order[at:at + n] + [-1] * (width - a - n))
        at += n
    int32 = dict(dtype=torch.int32, device="cuda")
    state = {"case": case, "table": torch.tensor(rows, **int32), "cu": torch.tensor(cu, **int32),
             "lens": torch.tensor([ctx + new for ctx, new in lens], **int32), "max_q": max(new for _, new in lens)}
    tokens = cu[-1]
    for name in ("k", "v"):
        state[name] = torch.empty(pages, hk, page, d, dtype=torch.bfloat16, device="cuda")
        step = max(1, (1 << 27) // (hk * page * d))
        for a in range(0, pages, step):
            state[name][a:a + step] = rand(min(step, pages - a), hk, page, d)
    if case["op"] == "append":
        heads = hq + (1 if _kv_eq(case) else 2) * hk
        state["qkv"] = torch.empty(tokens, heads * d, dtype=torch.bfloat16, device="cuda")
        for a in range(0, tokens, 2048):
            part = state["qkv"][a:a + 2048]
            part.copy_(rand(*part.shape).mul_(1.5))
        state["q_w"] = 1 + 0.2 * rand(d)
        state["k_w"] = 1 + 0.2 * rand(d)
        state["inv_freq"] = _inv_freq(case).cuda()
    else:
        # scores of a spread of 2.5, as trained norm weights leave them, and some rows that single out a key
        q = rand(tokens, hq, d).mul_(2.5 / math.sqrt(d))
        at = torch.randint(0, pages, (tokens,), device="cuda", generator=gen)
        on = torch.randint(0, page, (tokens,), device="cuda", generator=gen)
        liked = state["k"][at, :, on].float().repeat_interleave(hq // hk, 1)
        some = (torch.rand(tokens, hq, 1, device="cuda", generator=gen) < 0.2).float()
        state["q"] = (q + liked * some * (8.0 / d)).to(torch.bfloat16)
    return state


# ------------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    from micro_engram_fork_b200.ops import paged

    c = s["case"]
    if c["op"] == "append":
        q = paged.qkv_norm_rope_append(s["qkv"], s["q_w"], s["k_w"], s["inv_freq"], s["k"], s["v"], s["table"], s["cu"], s["lens"],
                                       c["hq"], kv_shared=_kv_eq(c), eps=EPS)
        return {"q": q, "k": s["k"], "v": s["v"]}
    o, lse = paged.paged_attention(s["q"], s["k"], s["v"], s["table"], s["cu"], s["lens"], window=c["window"] or None, scale=1.0,
                                   max_q=s["max_q"])
    return {"o": o, "lse": lse}


# ------------------------------------------------------------------------------- the plain forms
def _token_places(s, tokens):
    """(position, page, row of the page) of each new token."""
    cu, lens, page = s["cu"].long(), s["lens"].long(), s["case"]["page"]
    t = torch.arange(tokens, device=cu.device)
    b = (t.unsqueeze(1) >= cu[1:].unsqueeze(0)).sum(1)
    pos = lens[b] - (cu[b + 1] - t)
    return pos, s["table"].long()[b, pos // page], pos % page


def _plain_append(s):
    c = s["case"]
    hq, hk, d = c["hq"], c["hk"], c["d"]
    tokens = s["qkv"].shape[0]
    x = s["qkv"].float().view(tokens, -1, d)
    n = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS)
    pos, page, row = _token_places(s, tokens)
    # the angle of a far position loses its fraction in 32 bits
    angle = torch.remainder(pos.double().unsqueeze(1) * s["inv_freq"].double(), 2 * math.pi).float().unsqueeze(1)
    cos, sin = torch.cos(angle), torch.sin(angle)

    def rotate(y):
        a, b = y[..., :d // 2], y[..., d // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin], 2).to(torch.bfloat16)

    s["k"][page, :, row] = rotate(n[:, hq:hq + hk] * s["k_w"])
    s["v"][page, :, row] = n[:, -hk:].to(torch.bfloat16)
    return {"q": rotate(n[:, :hq] * s["q_w"]), "k": s["k"], "v": s["v"]}


def _plain_attend(s):
    c = s["case"]
    hq, hk, d, page, window = c["hq"], c["hk"], c["d"], c["page"], c["window"]
    out, lses = [], []
    at = 0
    for b, (ctx, new) in enumerate(_lengths(c)):
        first = _first_key(c, ctx) // page
        pages = s["table"][b, first:(ctx + new + page - 1) // page].long()
        k = s["k"][pages].float().transpose(0, 1).reshape(hk, -1, d)[:, :ctx + new - first * page]
        v = s["v"][pages].float().transpose(0, 1).reshape(hk, -1, d)[:, :ctx + new - first * page]
        q = s["q"][at:at + new].float().view(new, hk, hq // hk, d).permute(1, 2, 0, 3).reshape(hk, -1, d)
        x = torch.matmul(q, k.transpose(1, 2)).view(hk, hq // hk, new, -1)
        pos = torch.arange(ctx, ctx + new, device=x.device).unsqueeze(1)
        key = torch.arange(first * page, ctx + new, device=x.device).unsqueeze(0)
        hidden = key > pos
        if window:
            hidden = hidden | (key <= pos - window)
        x.masked_fill_(hidden, -math.inf)
        m = x.amax(3, keepdim=True)
        p = x.sub_(m).exp_()
        z = p.sum(3, keepdim=True)
        o = torch.matmul(p.view(hk, -1, p.shape[3]), v).view(hk, hq // hk, new, d) / z
        out.append(o.permute(2, 0, 1, 3).reshape(new, hq, d).to(torch.bfloat16))
        lses.append((m + torch.log(z)).view(hq, new))
        at += new
    return {"o": torch.cat(out), "lse": torch.cat(lses, 1)}


def run(state):
    if own:
        return _run_own(state)
    return _plain_append(state) if state["case"]["op"] == "append" else _plain_attend(state)


# ------------------------------------------------------------------------------- the definitions in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    hq, hk, d, page, window = case["hq"], case["hk"], case["d"], case["page"], case["window"]
    table = s["table"].cpu()
    lens = _lengths(case)
    if case["op"] == "append":
        k, v = s["k"].double(), s["v"].double()
        q = torch.empty(s["qkv"].shape[0], hq, d, dtype=torch.float64, device="cuda")
        at = 0
        for b, (ctx, new) in enumerate(lens):
            for first in range(0, new, 1024):
                n = min(1024, new - first)
                x = s["qkv"][at + first:at + first + n].double().view(n, -1, d)
                x = x / torch.sqrt((x * x).sum(2, keepdim=True) / d + EPS)
                p = torch.arange(ctx + first, ctx + first + n, device="cuda", dtype=torch.float64)
                turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), p[:, None, None] * s["inv_freq"].double())

                def rotated(y):
                    z = torch.complex(y[..., :d // 2].contiguous(), y[..., d // 2:].contiguous()) * turn
                    return torch.cat([z.real, z.imag], 2)

                q[at + first:at + first + n] = rotated(x[:, :hq] * s["q_w"].double())
                p = p.long()
                where = table[b][(p // page).cpu()].long().cuda()
                k[where, :, p % page] = rotated(x[:, hq:hq + hk] * s["k_w"].double())
                v[where, :, p % page] = x[:, x.shape[1] - hk:]
            at += new
        return {"q": q, "k": k, "v": v}
    if work(case)["flops"] > 1e13:
        return None
    o = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    lse = torch.empty(hq, s["q"].shape[0], dtype=torch.float64, device="cuda")
    at = 0
    for b, (ctx, new) in enumerate(lens):
        lo, end = _first_key(case, ctx), ctx + new
        p = torch.arange(lo, end)
        where, row = table[b][p // page].long().cuda(), (p % page).cuda()
        pos, key = torch.arange(ctx, end, device="cuda"), torch.arange(lo, end, device="cuda")
        seen = key[None, :] <= pos[:, None]
        if window:
            seen &= pos[:, None] - key[None, :] < window
        for g in range(hk):
            k, v = s["k"][where, g, row].double(), s["v"][where, g, row].double()
            for h in range(g * (hq // hk), (g + 1) * (hq // hk)):
                x = s["q"][at:at + new, h].double() @ k.T
                x = torch.where(seen, x, -math.inf)
                e = torch.logsumexp(x, 1)
                lse[h, at:at + new] = e
                o[at:at + new, h] = torch.exp(x - e[:, None]) @ v
        at += new
    return {"o": o, "lse": lse}


def work(case):
    hq, hk, d, window = case["hq"], case["hk"], case["d"], case["window"]
    lens = _lengths(case)
    tokens = sum(new for _, new in lens)
    if case["op"] == "append":
        heads = hq + (1 if _kv_eq(case) else 2) * hk
        elements = tokens * (heads + hq + 2 * hk) * d
        return {"bytes": 2 * elements, "flops": 8 * tokens * (hq + 2 * hk) * d}
    keys = sum(ctx + new - _first_key(case, ctx) for ctx, new in lens)
    pairs = 0
    for ctx, new in lens:
        full = sum(range(ctx + 1, ctx + new + 1))
        if window:
            full -= sum(p + 1 - window for p in range(ctx, ctx + new) if p + 1 > window)
        pairs += full
    return {"bytes": 4 * keys * hk * d + 4 * tokens * hq * d + 4 * tokens * hq, "flops": 4 * pairs * hq * d}
