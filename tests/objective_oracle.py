"""64-bit definitions of the vocabulary objectives for their tests, by autograd over log_softmax: written
apart from micro_engram_fork_b200.ops.objectives, and shared by the CPU and the GPU tests."""
import torch

IGNORE = -100
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}
TINY = {torch.bfloat16: 1e-38, torch.float16: 2.0 ** -24, torch.float32: 1e-38, torch.float64: 1e-300}


def z64(x, cap):
    x = x.double()
    return cap * torch.tanh(x / cap) if cap else x


def logprobs(x, targets, cap, g):
    """(logp, gradient for coefficients g, probabilities + the target's 1) in fp64; valid targets."""
    leaf = x.detach().double().requires_grad_()
    lp = torch.log_softmax(z64(leaf, cap), 1)
    trained = targets != IGNORE
    logp = torch.where(trained, lp.gather(1, targets.clamp_min(0).unsqueeze(1)).squeeze(1), 0.0)
    (logp * g.double()).sum().backward()
    mass = lp.detach().exp().scatter_add(1, targets.clamp_min(0).unsqueeze(1), torch.ones_like(logp.detach()).unsqueeze(1))
    return logp.detach(), torch.where(trained.unsqueeze(1), leaf.grad, 0.0), mass


def distill(x, ids, top, lse, w, cap, temp):
    """(loss, gradient of its sum, probabilities + the teacher's). ids: valid and distinct, or negative."""
    leaf = x.detach().double().requires_grad_()
    lp = torch.log_softmax(z64(leaf, cap) / temp, 1)
    N, V = x.shape
    loss = []
    mass = lp.detach().exp()
    for r in range(N):
        used = ids[r] >= 0
        at, t = ids[r][used].long(), top[r][used].double() / temp
        if float(w[r]) == 0 or (lse is None and not bool((t > -float("inf")).any())):  # nothing to match
            loss.append(leaf.new_zeros(()))
            mass[r] = 0
            continue
        lq = torch.log_softmax(t, 0) if lse is None else t - lse[r].double()
        q = lq.exp()
        kl = torch.special.xlogy(q, q).sum() - (q * lp[r, at]).sum()
        if lse is not None and at.numel() < V:
            q_rest = (1 - q.sum()).clamp_min(0)
            if q_rest > 0:
                out = torch.ones(V, dtype=torch.bool, device=x.device)
                out[at] = False
                kl = kl + q_rest * (q_rest.log() - torch.logsumexp(lp[r, out], 0))
        mass[r, at] += q
        loss.append(w[r].double() * temp ** 2 * kl)
    loss = torch.stack(loss) if loss else leaf.new_zeros(0)
    if N:
        loss.sum().backward()
    grad = leaf.grad if leaf.grad is not None else torch.zeros_like(leaf)
    return loss.detach(), torch.where((w != 0).unsqueeze(1), grad, 0.0), mass


def pairs(logp, ref, cu, kind, beta, smooth, scale):
    """(loss, rewards, scale * gradient of sum(loss)) in fp64."""
    leaf = logp.detach().double().requires_grad_()
    ratio = leaf if ref is None else leaf - ref.double()
    sums = torch.stack([ratio[a:b].sum() for a, b in zip(cu[:-1], cu[1:])]).view(-1, 2)
    h = sums[:, 0] - sums[:, 1]
    log_sigmoid = torch.nn.functional.logsigmoid
    loss = {"sigmoid": lambda: -(1 - smooth) * log_sigmoid(beta * h) - smooth * log_sigmoid(-beta * h),
            "hinge": lambda: torch.relu(1 - beta * h), "ipo": lambda: (h - 0.5 / beta) ** 2}[kind]()
    (loss.sum() * scale).backward()
    return loss.detach(), beta * sums.detach(), leaf.grad


def close_logp(got, want, x, cap, temp=1.0, factor=1.0):
    """Absolute error of a log-probability: 32 rounding units of fp32 at the size of the logits it
    is formed from (their maximum, the target's, and the log of the sum)."""
    finite = x.detach().double()
    finite = torch.where(finite.isfinite(), finite, 0.0)
    big = finite.abs().amax(1).clamp(max=cap or float("inf")) / temp
    tol = factor * 32 * 2.0 ** -24 * (2 * big + 16)
    assert torch.equal(got.isnan(), want.isnan()), (got, want)
    bad = torch.where(got.double() == want, 0.0, (got.double() - want).abs() - tol)
    bad = torch.where(want.isnan(), 0.0, bad)
    assert bool((bad <= 0).all()), (got.double() - want).abs().max()


def close_grad(got, want, coef, mass, dtype):
    """Elementwise: one rounding to the output's type, plus fp32 error of the probabilities: their
    exponent's argument is rounded at up to about 2^7 (2^-17 relative), and so is the softcap."""
    tol = 1.01 * UNIT[dtype] * want.abs() + 2.0 ** -16 * coef.abs().unsqueeze(1) * mass + TINY[dtype]
    err = (got.double() - want).abs()
    assert torch.equal(got.isnan(), want.isnan())
    assert bool(((err <= tol) | want.isnan()).all()), float((err - tol).max())


def merged(ids, top, temp):
    """The same teacher with one entry an id: the first one has the sum of the probabilities, the others are unused."""
    ids, top = ids.clone(), top.double() / temp
    for r in range(ids.shape[0]):
        for j in ids[r].unique().tolist():
            at = (ids[r] == j).nonzero().squeeze(1)
            top[r, at[0]] = torch.logsumexp(top[r, at], 0)
            ids[r, at[1:]] = -1
    return ids, top * temp


def rest_mass(x, ids, top, lse, cap, temp):
    """What the teacher's rest puts on each column that is no entry (its probability times the column's share of the
    student's rest): with the probabilities and the entries' own, all that a gradient with a rest is a sum of."""
    lp = torch.log_softmax(z64(x, cap) / temp, 1)
    out = torch.zeros_like(lp)
    for r in range(x.shape[0] if lse is not None else 0):
        used = ids[r] >= 0
        keep = torch.ones(x.shape[1], dtype=torch.bool, device=x.device)
        keep[ids[r][used]] = False
        q_rest = (1 - (top[r][used].double() / temp - lse[r].double()).exp().sum()).clamp_min(0)
        if bool(keep.any()):
            out[r, keep] = q_rest * (lp[r, keep] - torch.logsumexp(lp[r, keep], 0)).exp()
    return out


def repeated_cases(dev):
    """(V, ids, top, lse or None): repeated ids, among them rows whose entries are the whole vocabulary only if repeats
    are counted, or are it with repeats."""
    g = torch.Generator(device=dev).manual_seed(11)
    for V, k, N in ((2, 2, 3), (2, 3, 4), (4, 4, 6), (37, 12, 8), (5003, 256, 5), (9001, 40, 6)):
        ids = torch.randint(0, min(V, max(2, k // 3)), (N, k), device=dev, generator=g)
        ids[0] = ids[0, 0]                      # one token, k times
        ids[1] = torch.arange(k, device=dev) % V  # every token as long as there are some
        if k > 3:
            ids[2, k // 2:] = -1
        top = torch.randn(N, k, device=dev, generator=g) * 3
        top[N - 1, 0] = -float("inf")
        for lse in (None, torch.logsumexp(top / 1.5, 1) + 0.3, torch.logsumexp(top / 1.5, 1)):
            yield V, ids, top, lse
