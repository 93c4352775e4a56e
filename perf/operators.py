"""Measured cases of the training objectives over a vocabulary (micro_engram_fork_b200.ops.objectives).

The operators work on rows of next-token logits x [N, V] (one row a token, V the vocabulary),
softcapped to z = c tanh(x / c) where the model has a final softcap c:

  top_logits        the k largest z of each row with their ids, and the row's log-sum-exp: what a
                    teacher records for its student
  token_logprobs    log softmax(z)[target] of each row, and its gradient in x
  distill           KL(teacher || student) from a teacher's recorded top logits, and its gradient in x
  preference        paired log-ratio loss over packed chosen / rejected sequences, and its gradient

`run` computes an operator in its plain form, in 32 bits, where `own` is false, and through the
framework's entry points where it is true. `exact` computes it from the definition in 64 bits.
"""
import math
import random

import torch

own = False

IGNORE = -100
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
FULL = 2048 * 262144  # logits of the largest case: one loss chunk of the trainer at the benchmark's vocabulary


def listed():
    return [
        # the teacher's side: one token of a served answer, as a server that returns top logprobs does
        {"name": "top one token", "op": "top", "n": 1, "v": 262144, "k": 20, "dtype": "bf16", "cap": 30.0, "temp": 1.0},
        # recording a data set: one chunk of the trainer's head
        {"name": "top chunk", "op": "top", "n": 2048, "v": 262144, "k": 64, "dtype": "bf16", "cap": 30.0, "temp": 1.0},
        # a model of another vocabulary, odd, without a softcap, logits kept in 32 bits, at a raised temperature
        {"name": "top odd fp32", "op": "top", "n": 333, "v": 50001, "k": 100, "dtype": "fp32", "cap": 0.0, "temp": 2.0},
        # scoring a few tokens of one answer
        {"name": "logprobs few tokens", "op": "logprobs", "n": 5, "v": 262144, "dtype": "bf16", "cap": 30.0},
        # the reference policy's log-probabilities of a chunk (no gradient)
        {"name": "logprobs chunk", "op": "logprobs", "n": 2048, "v": 262144, "dtype": "bf16", "cap": 30.0},
        # log-probabilities with a gradient, for a loss that the user writes on top of them
        {"name": "logprobs train odd fp32", "op": "logprobs_train", "n": 777, "v": 32003, "dtype": "fp32", "cap": 0.0},
        # distilling a short row of tokens at a toy vocabulary: bound by launches
        {"name": "distill small", "op": "distill", "n": 16, "v": 4096, "k": 8, "dtype": "bf16", "cap": 30.0, "temp": 1.0, "tail": False},
        # the trainer's chunk: loss and gradient at once
        {"name": "distill chunk", "op": "distill", "n": 2048, "v": 262144, "k": 64, "dtype": "bf16", "cap": 30.0, "temp": 1.0, "tail": False},
        # the autograd form, odd sizes, the rest of the vocabulary as one class of its own
        {"name": "distill autograd odd tail", "op": "distill_train", "n": 515, "v": 100003, "k": 33, "dtype": "bf16", "cap": 0.0, "temp": 2.0, "tail": True},
        # the pair loss on log-probabilities that are there already (the trainer's head gives them)
        {"name": "pairs on logprobs", "op": "pairs", "n": 6000, "pairs": 4, "kind": "sigmoid"},
        # a preference step from the logits of a packed micro-batch, prompts untrained
        {"name": "preference chunk", "op": "preference", "n": 2048, "v": 262144, "pairs": 4, "dtype": "bf16", "cap": 30.0, "kind": "sigmoid"},
        # the same with short answers and an odd vocabulary in fp16
        {"name": "preference odd fp16", "op": "preference", "n": 301, "v": 50001, "pairs": 5, "dtype": "fp16", "cap": 0.0, "kind": "ipo"},
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["top", "logprobs", "logprobs_train", "distill", "distill_train", "pairs", "preference"])
    if op == "pairs":
        pairs = _log(rng, 1, 64)
        return {"op": op, "n": _log(rng, 2 * pairs, 60000), "pairs": pairs, "kind": rng.choice(["sigmoid", "hinge", "ipo"])}
    v = _log(rng, 1000, 262144)
    if rng.random() < 0.4:
        v -= v % 8  # most models' vocabularies are padded to a multiple of 8
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    case = {"op": op, "n": _log(rng, 1, 2048), "v": v, "dtype": dtype, "cap": rng.choice([0.0, 30.0, 30.0])}
    if dtype == "fp32":
        case["n"] = max(1, min(case["n"], FULL // 2 // v))
    if op in ("top", "distill", "distill_train"):
        case |= {"k": _log(rng, 1, 128), "temp": rng.choice([1.0, 1.0, 2.0])}
    if op in ("distill", "distill_train"):
        case["tail"] = rng.random() < 0.5
    if op == "preference":
        case |= {"pairs": max(1, min(case["n"] // 2, _log(rng, 1, 16))), "kind": rng.choice(["sigmoid", "hinge", "ipo"])}
    return case


# ------------------------------------------------------------------------------- inputs
def _logits(n, v, dtype, gen, like=None):
    """Raw logits as a language model has them: a broad body (-5 +- 2.5) and a few tokens far above
    it. With `like`, a second model's view of the same rows. The last columns of an odd vocabulary
    are masked out (-inf), as a padded vocabulary's are."""
    x = torch.empty(n, v, dtype=dtype, device="cuda")
    step = max(1, (1 << 26) // v)
    for a in range(0, n, step):
        b = min(n, a + step)
        if like is None:
            t = torch.randn(b - a, v, device="cuda", generator=gen).mul_(2.5).sub_(5.0)
            part = v // 12  # distinct columns: what a scatter does with equal ones is not settled
            hot = torch.arange(12, device="cuda") * part + torch.randint(0, part, (b - a, 12), device="cuda", generator=gen)
            t.scatter_(1, hot, torch.randn(b - a, 12, device="cuda", generator=gen).mul_(3.0).add_(10.0))
        else:
            t = like[a:b].float()
            t = t + torch.randn(t.shape, device="cuda", generator=gen).mul_(0.7)
        if v % 2:
            t[:, v - 3:] = -math.inf
        x[a:b] = t
    return x


def _weights(n, gen):
    """Per-token loss weights: a third of the tokens untrained, the others share one sum."""
    w = (torch.rand(n, device="cuda", generator=gen) > 1 / 3).float()
    w[0] = 1.0
    return w / w.sum()


def _packed(n, pairs, seed):
    """Cumulative lengths of 2 * pairs packed sequences over n tokens (ragged, some may be empty)."""
    r = random.Random(seed)
    cuts = sorted(r.randint(0, n) for _ in range(2 * pairs - 1))
    return [0] + cuts + [n]


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, n = case["op"], case["n"]
    state = {"case": case}
    if op in ("pairs", "preference"):
        cu = _packed(n, case["pairs"], seed)
        state["cu"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    if op == "pairs":
        state["logp"] = -torch.rand(n, device="cuda", generator=gen).mul_(4.0).square()
        state["ref"] = state["logp"] + torch.randn(n, device="cuda", generator=gen).mul_(0.1)
        return state
    v, dtype = case["v"], DTYPES[case["dtype"]]
    x = _logits(n, v, dtype, gen)
    state["x"] = x
    if op in ("logprobs_train", "distill_train"):
        state["leaf"] = x.requires_grad_()
    if op in ("logprobs", "logprobs_train", "preference"):
        t = torch.randint(0, v - 3, (n,), device="cuda", generator=gen)
        if op == "preference":  # the first half of each sequence is its prompt
            for a, b in zip(cu[:-1], cu[1:]):
                t[a:(a + b) // 2] = IGNORE
            state["ref"] = torch.randn(n, device="cuda", generator=gen).mul_(1.5).sub_(14.0)
        else:
            t[torch.rand(n, device="cuda", generator=gen) < 0.1] = IGNORE
            t[0] = 1
        state["t"] = t
    if op == "logprobs_train":
        state["g"] = torch.randn(n, device="cuda", generator=gen) / n
    if op in ("distill", "distill_train"):
        k, temp = case["k"], case["temp"]
        ids, top, lse = [], [], []
        step = max(1, (1 << 27) // v)
        for a in range(0, n, step):
            y = _logits(min(n, a + step) - a, v, torch.float32, gen, like=x.detach()[a:a + step])
            y = case["cap"] * torch.tanh(y / case["cap"]) if case["cap"] else y
            values, at = torch.topk(y, k, dim=1)
            ids.append(at)
            top.append(values)
            lse.append(torch.logsumexp(y / temp, dim=1))
        state |= {"ids": torch.cat(ids), "top": torch.cat(top), "lse": torch.cat(lse) if case["tail"] else None,
                  "w": _weights(n, gen)}
    return state


# ------------------------------------------------------------------------------- the framework's calls
def _run_own(s):
    from micro_engram_fork_b200.ops import objectives as O

    c = s["case"]
    op = c["op"]
    cap = c.get("cap") or None
    smooth = 0.05 if c.get("kind") == "sigmoid" else 0.0
    if op == "top":
        values, ids, lse = O.top_logits(s["x"], c["k"], softcap=cap, temperature=c["temp"])
        return {"values": values, "ids": ids, "lse": lse}
    if op == "logprobs":
        return {"logp": O.token_logprobs(s["x"], s["t"], softcap=cap)}
    if op == "logprobs_train":
        logp = O.token_logprobs(s["leaf"], s["t"], softcap=cap)
        return {"logp": logp.detach(), "grad": torch.autograd.grad(logp, s["leaf"], s["g"])[0]}
    if op == "distill":
        loss, grad = O.distill_loss_grad(s["x"], s["ids"], s["top"], teacher_lse=s["lse"], weights=s["w"], softcap=cap,
                                         temperature=c["temp"])
        return {"loss": loss, "grad": grad}
    if op == "distill_train":
        loss = O.distill_loss(s["leaf"], s["ids"], s["top"], teacher_lse=s["lse"], weights=s["w"], softcap=cap,
                              temperature=c["temp"])
        return {"loss": loss.detach(), "grad": torch.autograd.grad(loss.sum(), s["leaf"])[0]}
    if op == "pairs":
        loss, rewards, grad = O.preference_loss_grad(s["logp"], s["ref"], s["cu"], beta=0.1, label_smoothing=smooth,
                                                     kind=c["kind"])
        return {"loss": loss, "rewards": rewards, "grad": grad}
    loss, rewards, logp, grad = O.preference_logits_grad(s["x"], s["t"], s["ref"], s["cu"], beta=0.1, label_smoothing=smooth,
                                                         kind=c["kind"], softcap=cap)
    return {"loss": loss, "rewards": rewards, "logp": logp, "grad": grad}


# ------------------------------------------------------------------------------- the plain forms
def _capped(x, cap):
    """(z, dz/dx) in 32 bits."""
    x = x.detach().float()
    if not cap:
        return x, None
    t = torch.tanh(x / cap)
    return t * cap, 1 - t * t


def _softmax(y):
    """(softmax, log-sum-exp) of rows."""
    m = y.amax(1, keepdim=True)
    e = torch.exp(y - m)
    s = e.sum(1, keepdim=True)
    return e / s, m + torch.log(s)


def _plain_logprobs(x, t, cap):
    """(log-probabilities, 0 where untrained; a function that gives the gradient for coefficients)."""
    z, dz = _capped(x, cap)
    p, lse = _softmax(z)
    keep = t != IGNORE
    col = t.clamp_min(0).unsqueeze(1)
    logp = torch.where(keep, (z.gather(1, col) - lse).squeeze(1), 0.0)

    def grad(g):
        g = torch.where(keep, g, 0.0).unsqueeze(1)
        d = p * -g
        d.scatter_add_(1, col, g)
        if dz is not None:
            d *= dz
        return d.to(x.dtype)

    return logp, grad


def _plain_distill(s):
    c = s["case"]
    x, temp, ids, w = s["x"], c["temp"], s["ids"], s["w"].unsqueeze(1)
    z, dz = _capped(x, c["cap"])
    y = z / temp
    p, lse = _softmax(y)
    t = s["top"] / temp
    log_p = y.gather(1, ids) - lse
    if s["lse"] is None:
        q, t_lse = _softmax(t)
        kl = (q * (t - t_lse - log_p)).sum(1, keepdim=True)
        d = p.clone()
    else:
        log_q = t - s["lse"].unsqueeze(1)
        q = torch.exp(log_q)
        q_rest = (1 - q.sum(1, keepdim=True)).clamp_min(0)
        rest = p.scatter(1, ids, 0.0)
        p_rest = rest.sum(1, keepdim=True)
        kl = (q * (log_q - log_p)).sum(1, keepdim=True)
        kl = kl + torch.where(q_rest > 0, q_rest * (torch.log(q_rest) - torch.log(p_rest)), 0.0)
        d = p - rest * (q_rest / p_rest)
    d.scatter_add_(1, ids, -q)
    d = d * (w * temp)
    if dz is not None:
        d *= dz
    return {"loss": (kl * w * temp * temp).squeeze(1), "grad": d.to(x.dtype)}


def _plain_pairs(logp, ref, cu, kind, beta=0.1, smooth=0.05):
    """(loss of each pair, rewards, gradient of their mean in each token's log-probability); `smooth` of the sigmoid loss."""
    n, seqs = logp.numel(), cu.numel() - 1
    at = torch.arange(n, device=logp.device)
    seq = (at.unsqueeze(1) >= cu[1:].unsqueeze(0)).sum(1)  # the sequence of each token
    member = (seq.unsqueeze(0) == torch.arange(seqs, device=logp.device).unsqueeze(1)).float()
    ratio = (member * (logp - ref)).sum(1).view(-1, 2)
    h = ratio[:, 0] - ratio[:, 1]
    if kind == "sigmoid":
        u = beta * h
        soft = lambda v: v.clamp_min(0) + torch.log1p(torch.exp(-v.abs()))  # noqa: E731  log(1 + e^v)
        loss = (1 - smooth) * soft(-u) + smooth * soft(u)
        d = beta * (smooth - 1 / (1 + torch.exp(u)))
    elif kind == "hinge":
        loss = (1 - beta * h).clamp_min(0)
        d = torch.where(beta * h < 1, -beta, 0.0)
    else:
        loss = (h - 1 / (2 * beta)).square()
        d = 2 * (h - 1 / (2 * beta))
    d = torch.stack([d, -d], 1).reshape(-1) / (seqs // 2)
    return loss, beta * ratio, d[seq]


def _run_plain(s):
    c = s["case"]
    op = c["op"]
    if op == "top":
        z, _ = _capped(s["x"], c["cap"])
        _, lse = _softmax(z / c["temp"])
        ids = torch.sort(s["x"].float(), dim=1, descending=True, stable=True)[1][:, :c["k"]].contiguous()
        return {"values": z.gather(1, ids), "ids": ids, "lse": lse.squeeze(1)}
    if op == "logprobs":
        return {"logp": _plain_logprobs(s["x"], s["t"], c["cap"])[0]}
    if op == "logprobs_train":
        logp, grad = _plain_logprobs(s["x"], s["t"], c["cap"])
        return {"logp": logp, "grad": grad(s["g"])}
    if op in ("distill", "distill_train"):
        return _plain_distill(s)
    if op == "pairs":
        loss, rewards, grad = _plain_pairs(s["logp"], s["ref"], s["cu"], c["kind"])
        return {"loss": loss, "rewards": rewards, "grad": grad}
    logp, grad = _plain_logprobs(s["x"], s["t"], c["cap"])
    ref = torch.where(s["t"] != IGNORE, s["ref"], 0.0)
    loss, rewards, g = _plain_pairs(logp, ref, s["cu"], c["kind"])
    return {"loss": loss, "rewards": rewards, "logp": logp, "grad": grad(g)}


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ------------------------------------------------------------------------------- the definitions in 64 bits
def _rows(n, v):
    step = max(1, (1 << 26) // v)
    return [(a, min(n, a + step)) for a in range(0, n, step)]


def _z64(x, cap):
    x = x.detach().double()
    return cap * torch.tanh(x / cap) if cap else x


def _top64(s):
    c = s["case"]
    x, k, v = s["x"], c["k"], c["v"]
    values, ids, lse = [], [], []
    for a, b in _rows(c["n"], v):
        r = x[a:b].float() + 0.0
        bits = r.view(torch.int32).long()
        rank = torch.where(bits >= 0, bits, -(bits & 0x7FFFFFFF))  # ordered as the values are
        at = torch.topk(rank * (1 << 20) + (v - 1 - torch.arange(v, device=x.device)), k, dim=1)[1]
        z = _z64(x[a:b], c["cap"])
        values.append(z.gather(1, at))
        ids.append(at)
        lse.append(torch.logsumexp(z / c["temp"], 1))
    return {"values": torch.cat(values), "ids": torch.cat(ids), "lse": torch.cat(lse)}


def _chain64(x, g, cap):
    """dL/dx from dL/dz."""
    return g / torch.cosh(x.detach().double() / cap).square() if cap else g


def _logp64(s, coef):
    """Log-probabilities, and with `coef` (one a token) the gradient of sum(coef * logp) in the logits."""
    c = s["case"]
    x, t = s["x"], s["t"]
    logp = torch.zeros(c["n"], dtype=torch.float64, device=x.device)
    grad = None if coef is None else torch.zeros(c["n"], c["v"], dtype=torch.float64, device=x.device)
    for a, b in _rows(c["n"], c["v"]):
        at = (t[a:b] >= 0).nonzero().squeeze(1)
        z = torch.log_softmax(_z64(x[a:b], c["cap"]), 1)[at]
        col = t[a:b][at]
        logp[a + at] = z[torch.arange(at.numel(), device=x.device), col]
        if grad is not None:
            g = -torch.exp(z)
            g[torch.arange(at.numel(), device=x.device), col] += 1
            grad[a + at] = _chain64(x[a:b][at], g * coef[a:b][at].double().unsqueeze(1), c["cap"])
    return logp, grad


def _distill64(s):
    c = s["case"]
    x, n, temp = s["x"], c["n"], c["temp"]
    loss = torch.zeros(n, dtype=torch.float64, device=x.device)
    grad = torch.zeros(n, c["v"], dtype=torch.float64, device=x.device)
    for a, b in _rows(n, c["v"]):
        lp = torch.log_softmax(_z64(x[a:b], c["cap"]) / temp, 1)
        ids = s["ids"][a:b]
        t = s["top"][a:b].double() / temp
        w = s["w"][a:b].double()
        top_lp = lp.gather(1, ids)
        g = torch.exp(lp)
        if s["lse"] is None:
            lq = torch.log_softmax(t, 1)
            loss[a:b] = w * temp ** 2 * (lq.exp() * (lq - top_lp)).sum(1)
        else:
            lq = t - s["lse"][a:b].double().unsqueeze(1)
            q_rest = 1 - lq.exp().sum(1)
            hidden = lp.scatter(1, ids, -math.inf)
            lp_rest = torch.logsumexp(hidden, 1)
            loss[a:b] = w * temp ** 2 * ((lq.exp() * (lq - top_lp)).sum(1)
                                         + torch.special.xlogy(q_rest.clamp_min(0), q_rest.clamp_min(1e-300)) - q_rest.clamp_min(0) * lp_rest)
            g -= torch.exp(hidden) * (q_rest.clamp_min(0) / lp_rest.exp()).unsqueeze(1)
        g.scatter_add_(1, ids, -lq.exp())
        grad[a:b] = _chain64(x[a:b], g * (w * temp).unsqueeze(1), c["cap"])
    return {"loss": loss, "grad": grad}


def _pairs64(logp, ref, cu, kind, beta=0.1, smooth=0.05):
    cu = cu.tolist()
    pairs = (len(cu) - 1) // 2
    ratio = torch.stack([(logp[a:b].double() - ref[a:b].double()).sum() for a, b in zip(cu[:-1], cu[1:])]).view(pairs, 2)
    ratio = ratio.clone().requires_grad_()
    h = ratio[:, 0] - ratio[:, 1]
    if kind == "sigmoid":
        loss = -(1 - smooth) * torch.nn.functional.logsigmoid(beta * h) - smooth * torch.nn.functional.logsigmoid(-beta * h)
    elif kind == "hinge":
        loss = torch.relu(1 - beta * h)
    else:
        loss = (h - 0.5 / beta) ** 2
    d, = torch.autograd.grad(loss.mean(), ratio)
    grad = torch.zeros_like(logp, dtype=torch.float64)
    for i, (a, b) in enumerate(zip(cu[:-1], cu[1:])):
        grad[a:b] = d.view(-1)[i]
    return loss.detach(), beta * ratio.detach(), grad


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "top":
        return _top64(s)
    if op == "logprobs":
        return {"logp": _logp64(s, None)[0]}
    if op == "logprobs_train":
        logp, grad = _logp64(s, s["g"])
        return {"logp": logp, "grad": grad}
    if op in ("distill", "distill_train"):
        return _distill64(s)
    if op == "pairs":
        loss, rewards, grad = _pairs64(s["logp"], s["ref"], s["cu"], case["kind"])
        return {"loss": loss, "rewards": rewards, "grad": grad}
    logp, _ = _logp64(s, None)
    loss, rewards, coef = _pairs64(logp, s["ref"] * (s["t"] != IGNORE), s["cu"], case["kind"])
    return {"loss": loss, "rewards": rewards, "logp": logp, "grad": _logp64(s, coef)[1]}


# ------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Bytes: the logits of the rows that count once, the gradient of every row once, and the small
    tensors. Operations: about 4 a logit for a softmax, 4 more for its gradient, 8 more for a softcap."""
    op, n = case["op"], case["n"]
    if op == "pairs":
        return {"bytes": 4 * 3 * n + 4 * (2 * case["pairs"] + 1) + 12 * case["pairs"], "flops": 4 * n}
    x = n * case["v"]
    size = x * BYTES[case["dtype"]]
    flops = x * (4 + (8 if case["cap"] else 0))
    if op == "top":
        return {"bytes": size + n * (case["k"] * 12 + 4), "flops": flops + x}
    if op == "logprobs":
        return {"bytes": 0.9 * size + n * 12, "flops": 0.9 * flops}
    if op == "logprobs_train":
        return {"bytes": 1.9 * size + n * 16, "flops": 0.9 * (flops + 4 * x)}
    if op == "preference":
        return {"bytes": 1.5 * size + n * 16, "flops": 0.5 * (flops + 4 * x)}
    return {"bytes": (1 + 2 / 3) * size + n * (case["k"] * 12 + 12), "flops": 2 / 3 * (flops + 4 * x)}
