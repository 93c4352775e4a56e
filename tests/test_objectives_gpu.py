"""Vocabulary objectives on the sm_100a kernels: against the 64-bit definitions at the sizes, types,
strides and masks where they can go wrong; edge rules as on the CPU; streams, repeatability, refusals."""
import math

import pytest
import torch

import objective_oracle as oracle
from micro_engram_fork_b200.ops import objectives as O
from test_objectives import impossible_answers, nothing_to_match, overwritten, refusals

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _x(N, V, dtype, seed=0, pitch=0, shift=0):
    """Rows of logits `pitch` elements longer than V apart, `shift` elements into their storage."""
    g = _gen(seed)
    whole = torch.zeros(shift + N * (V + pitch), dtype=dtype, device=DEV)
    x = whole[shift:].view(N, V + pitch)[:, :V]
    x.copy_(torch.randn(N, V, device=DEV, generator=g) * 4)
    if V > 4:
        hot = torch.randint(0, V, (N, 3), device=DEV, generator=g)
        x.scatter_(1, hot, torch.full((N, 3), 14.0, device=DEV, dtype=dtype))
    return x


def _teacher(N, V, k, seed=0):
    g = _gen(seed)
    ids = torch.rand(N, V, device=DEV, generator=g).topk(k, dim=1)[1]
    return ids, torch.randn(N, k, device=DEV, generator=g) * 3


# vocabularies around the vector, block and slice sizes; row pitches and offsets off 16 bytes
SHAPES = [(1, 1, 0, 0), (3, 2, 0, 0), (2, 7, 1, 0), (5, 8, 0, 0), (4, 9, 0, 3), (3, 255, 2, 1), (6, 4096, 0, 0),
          (37, 5003, 0, 0), (9, 5003, 5, 1), (2, 32768, 8, 0), (3, 65537, 0, 0), (301, 12345, 3, 0), (2, 262144, 0, 0),
          (2, 300001, 0, 0), (1, 600008, 0, 0)]


@pytest.mark.parametrize("cap", [None, 30.0])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
@pytest.mark.parametrize("N,V,pitch,shift", SHAPES)
def test_token_logprobs(N, V, pitch, shift, dtype, cap):
    x = _x(N, V, dtype, N + V, pitch, shift)
    g = _gen(1)
    t = torch.randint(0, V, (N,), device=DEV, generator=g)
    if N > 2:
        t[1] = -100
    t[-1] = V - 1
    coef = torch.randn(N, device=DEV, generator=g)
    leaf = x.detach().requires_grad_()
    logp = O.token_logprobs(leaf, t, softcap=cap)
    dx, = torch.autograd.grad(logp, leaf, coef)
    want, grad, mass = oracle.logprobs(x, t, cap, coef)
    oracle.close_logp(logp.detach(), want, x, cap)
    oracle.close_grad(dx, grad, coef, mass, dtype)
    if N > 2:
        assert bool((dx[1] == 0).all()) and logp[1] == 0


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("dtype,cap,temp", [(BF, 30.0, 1.0), (BF, None, 2.0), (HF, 30.0, 2.0), (FP, None, 1.0),
                                            (FP, 30.0, 0.7)])
@pytest.mark.parametrize("N,V,pitch,shift", SHAPES)
def test_distill(N, V, pitch, shift, dtype, cap, temp, tail):
    x = _x(N, V, dtype, N + V, pitch, shift)
    k = min(V, {0: 33, 1: 256, 2: 1}[V % 3])
    ids, top = _teacher(N, V, k, 5)
    lse = torch.logsumexp(top / temp, 1) + 0.4 if tail else None
    w = torch.rand(N, device=DEV, generator=_gen(6)) + 0.2
    if N > 2:
        w[1] = 0.0
        ids[2, k // 2:] = -1
    if N > 4:
        ids[3] = -1
        top[4, 0] = -float("inf")
    args = (x, ids, top, lse, w)
    n = min(N, 40)  # the oracle walks the rows
    want, grad, mass = oracle.distill(x[:n], ids[:n], top[:n], None if lse is None else lse[:n], w[:n], cap, temp)
    scale = float(temp) ** 2 * 8
    loss, dx = O.distill_loss_grad(*args, softcap=cap, temperature=temp)
    oracle.close_logp(loss[:n], want, x[:n], cap, temp, factor=scale)
    oracle.close_grad(dx[:n], grad, w[:n] * temp, mass, dtype)
    leaf = x.detach().requires_grad_()
    loss2 = O.distill_loss(leaf, *args[1:], softcap=cap, temperature=temp)
    oracle.close_logp(loss2.detach()[:n], want, x[:n], cap, temp, factor=scale)
    g = torch.randn(N, device=DEV, generator=_gen(7))
    dx2, = torch.autograd.grad(loss2, leaf, g)
    oracle.close_grad(dx2[:n], grad * g[:n, None].double(), w[:n] * temp * g[:n], mass, dtype)
    if N > n:  # the rest against the plain form
        ref = O.distill_ref(x[n:], ids[n:], top[n:], None if lse is None else lse[n:], w[n:], cap or 0.0, temp)
        assert torch.allclose(loss[n:], ref[0], rtol=1e-4, atol=1e-4)
        assert torch.allclose(dx[n:].float(), ref[1].float(), rtol=2.0 ** -7, atol=1e-6)
    inplace = _x(N, V, dtype, N + V, pitch, shift)  # the same alignment: the same order of sums
    loss3, dx3 = O.distill_loss_grad(inplace, *args[1:], softcap=cap, temperature=temp, out=inplace)
    assert dx3 is inplace and torch.equal(dx3, dx) and torch.equal(loss3, loss)


@pytest.mark.parametrize("dtype,cap", [(BF, 30.0), (HF, 12.0), (FP, 30.0), (BF, 1e-3), (FP, 1000.0)])
def test_beyond_the_cap(dtype, cap):
    """Logits on both sides of the cap in the same vectors, and caps for which there is no polynomial."""
    N, V = 9, 20011
    x = (torch.randn(N, V, device=DEV, generator=_gen(1)) * 25).to(dtype)
    x[:, 5] = float("inf")
    x[:, 6] = -float("inf")
    t = torch.randint(0, V, (N,), device=DEV, generator=_gen(2))
    t[0] = 5
    coef = torch.randn(N, device=DEV, generator=_gen(3))
    logp, dx = O.token_logprobs_grad(x, t, coef, softcap=cap)
    finite = x.clamp(-3e4, 3e4)  # the same z, and derivatives that the oracle can take
    want, grad, mass = oracle.logprobs(finite, t, cap, coef)
    oracle.close_logp(logp, want, finite, cap)
    oracle.close_grad(dx, grad, coef, mass, dtype)
    leaf = x.detach().requires_grad_()
    logp2 = O.token_logprobs(leaf, t, softcap=cap)
    assert torch.equal(logp2.detach(), logp)
    assert torch.equal(torch.autograd.grad(logp2, leaf, coef)[0], dx)


def test_rows_longer_than_the_masks():
    """More vectors in a block's slice than there are bytes for the teacher's entries (they are shared then)."""
    N, V, k = 2, 2300011, 200
    x = _x(N, V, BF, 5)
    ids, top = _teacher(N, V, k, 6)
    ids[0, :3] = torch.tensor([17, 17 + 32768 * 8, V - 1], device=DEV)
    lse = torch.logsumexp(top, 1) + 0.5
    w = torch.ones(N, device=DEV)
    loss, dx = O.distill_loss_grad(x, ids, top, lse, w, softcap=30.0)
    want, grad, mass = oracle.distill(x, ids, top, lse, w, 30.0, 1.0)
    oracle.close_logp(loss, want, x, 30.0, factor=8)
    oracle.close_grad(dx, grad, w, mass, BF)
    _check_top(x, 100, 30.0, 1.0)


def test_padded_rows_keep_their_pitch():
    x = _x(40, 5003, BF, 3, pitch=5)
    t = torch.randint(0, 5003, (40,), device=DEV, generator=_gen(1))
    leaf = x.detach().requires_grad_()
    dx, = torch.autograd.grad(O.token_logprobs(leaf, t, softcap=30.0).sum(), leaf)
    _, same = O.token_logprobs_grad(x.contiguous(), t, None, softcap=30.0)
    assert dx.shape == x.shape and torch.allclose(dx.float(), same.float(), rtol=2.0 ** -7, atol=1e-9)
    _, wide = O.token_logprobs_grad(x, t, None, softcap=30.0, out=torch.empty(40, 5003, dtype=BF, device=DEV))
    assert torch.equal(wide, dx)


def test_gradients_are_not_differentiated():
    x = _x(3, 64, FP).requires_grad_()
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(O.token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=DEV)).sum(), x, create_graph=True)


def test_distill_repeated_and_foreign_ids():
    x = _x(3, 4097, BF, 3)
    ids = torch.tensor([[5, 5, 9, -1], [4096, 0, 4097, 1 << 40], [7, 7, 7, 7]], device=DEV)
    top = torch.tensor([[1.0, 2.0, 3.0, 9.0], [0.0, 1.0, 50.0, 60.0], [1.0, 1.0, 1.0, 1.0]], device=DEV)
    for lse in (None, torch.full((3,), 5.0, device=DEV)):
        loss, dx = O.distill_loss_grad(x, ids, top, lse, softcap=30.0)
        ref, dref = O.distill_ref(x.double(), ids, top.double(), lse, None, 30.0, 1.0)
        assert torch.allclose(loss.double(), ref, rtol=1e-5, atol=1e-5)
        assert torch.allclose(dx.double(), dref, rtol=2.0 ** -7, atol=1e-6)


def test_distill_whole_vocabulary():
    x = _x(4, 200, FP, 8)
    ids = torch.arange(200, device=DEV).expand(4, 200)
    top = torch.randn(4, 200, device=DEV, generator=_gen(2))
    lse = torch.logsumexp(top, 1)
    a, b = (O.distill_loss_grad(x, ids, top, t) for t in (None, lse))
    assert torch.allclose(a[0], b[0], rtol=1e-5, atol=1e-5) and torch.allclose(a[1], b[1], rtol=1e-4, atol=1e-6)


TOP = [(1, 1, 1), (2, 9, 9), (5, 300, 256), (3, 4096, 8), (2, 5003, 100), (300, 3001, 20), (1, 262144, 20), (4, 262144, 256),
       (700, 20000, 64), (2, 600007, 33)]


def _check_top(x, k, cap, temp):
    values, ids, lse = O.top_logits(x, k, softcap=cap, temperature=temp)
    want = torch.sort(x.double(), dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(ids, want)
    z = oracle.z64(x, cap)
    zt = z.gather(1, want)
    assert torch.allclose(values.double(), zt, rtol=2.0 ** -20, atol=2.0 ** -20)
    oracle.close_logp(lse, torch.logsumexp(z / temp, 1), x, cap, temp)


@pytest.mark.parametrize("dtype,cap,temp", [(BF, 30.0, 1.0), (HF, None, 2.0), (FP, 30.0, 0.5)])
@pytest.mark.parametrize("N,V,k", TOP)
def test_top_logits(N, V, k, dtype, cap, temp):
    _check_top(_x(N, V, dtype, N + V, V % 3, V % 2), k, cap, temp)


@pytest.mark.parametrize("dtype", [BF, FP])
def test_top_logits_orders(dtype):
    """Rows that a filter by block maxima handles worst: equal values, sorted both ways, one block of
    large ones, few finite ones, zeros of both signs, infinities."""
    V, k = 70001, 200
    j = torch.arange(V, device=DEV, dtype=torch.float32)
    inf = float("inf")
    rows = [torch.zeros(V, device=DEV), j / V, -j / V, torch.where(j < 5000, 1.0 + (j % 7), -1.0),
            torch.where(j % 1000 == 999, j / V, -inf), torch.where(j % 2 == 0, 0.0, -0.0), torch.where(j > V - 300, inf, j % 3),
            torch.full((V,), -inf, device=DEV), torch.where((j >= 33000) & (j < 34000), 2.0, 1.0), (j * 7919 % V) % 50]
    x = torch.stack(rows).to(dtype)
    values, ids, lse = O.top_logits(x, k)
    want = torch.sort(x.double(), dim=1, descending=True, stable=True)[1][:, :k]
    assert torch.equal(ids, want)
    assert torch.equal(values.double(), x.double().gather(1, want))
    lse64 = torch.logsumexp(x.double(), 1)
    keep = [0, 1, 2, 3, 4, 5, 8, 9]
    oracle.close_logp(lse[keep], lse64[keep], x[keep], None)
    assert bool(lse[6].isnan()) and lse[7] == -inf


def test_top_logits_nan():
    x = _x(3, 9001, BF, 4)
    x[1, [70, 8000]] = float("nan")
    values, ids, lse = O.top_logits(x, 5)
    assert ids[1, :2].tolist() == [70, 8000] and bool(values[1, :2].isnan().all()) and bool(lse[1].isnan())
    keep = x[1].float().clone()
    keep[[70, 8000]] = -float("inf")
    assert torch.equal(ids[1, 2:], torch.sort(keep, descending=True, stable=True)[1][:3])
    assert bool(lse[[0, 2]].isfinite().all())


@pytest.mark.parametrize("cap", [None, 5.0])
@pytest.mark.parametrize("dtype,V", [(BF, 4096), (FP, 5003), (BF, 262144), (HF, 12345)])
def test_non_finite(dtype, V, cap):
    nan, inf = float("nan"), float("inf")
    x = _x(7, V, dtype, 1)
    low = torch.finfo(dtype).min
    x[0] = nan                                  # untrained: not read
    x[1, V // 2] = nan
    x[2, V - 1] = inf
    x[3] = -inf
    x[4, 10:] = -inf                            # ten tokens left
    x[5, : V - 1] = low                         # one token left, the others at the type's lowest value
    t = torch.tensor([-100, 0, 0, 0, 3, V - 1, V], device=DEV)
    leaf = x.detach().requires_grad_()
    logp = O.token_logprobs(leaf, t, softcap=cap)
    dx, = torch.autograd.grad(logp.sum(), leaf)
    ref, grad = O.token_logprobs_ref(x.double(), t, cap or 0.0)
    assert torch.equal(logp.isnan(), ref.isnan()) and torch.equal(dx.isnan(), grad(torch.ones(7, device=DEV)).isnan())
    ok = ~ref.isnan()
    assert torch.allclose(logp[ok].double(), ref[ok], rtol=1e-5, atol=1e-5)
    assert logp[0] == 0 and bool((dx[0] == 0).all()) and bool(logp[6].isnan()) and bool(dx[6].isnan().all())
    ids, top = _teacher(7, V, 8, 3)
    ids[4] = torch.arange(8, device=DEV)
    ids[5, 0] = V - 1
    ids[5, 1:] = -1
    w = torch.tensor([0.0, 1, 1, 1, 1, 1, 1], device=DEV)
    for lse in (None, torch.logsumexp(top, 1) + 0.3):
        loss, dx = O.distill_loss_grad(x, ids, top, lse, w, softcap=cap)
        ref, dref = O.distill_ref(x.double(), ids, top.double(), None if lse is None else lse.double(), w, cap or 0.0, 1.0)
        assert torch.equal(loss.isnan(), ref.isnan()) and loss[0] == 0 and bool((dx[0] == 0).all())
        finite = ref.isfinite()
        assert torch.equal(loss.isfinite(), finite)
        assert torch.allclose(loss[finite].double(), ref[finite], rtol=1e-4, atol=1e-5)
        assert torch.equal(dx[finite].isnan(), dref[finite].isnan())


@pytest.mark.parametrize("low", [-float("inf"), None])
@pytest.mark.parametrize("dtype", [BF, HF, FP])
def test_masked_columns(dtype, low):
    """Most columns masked (-inf, or the type's lowest value), ahead of the others or between them."""
    N, V, k = 6, 30011, 16
    x = _x(N, V, dtype, 3)
    low = torch.finfo(dtype).min if low is None else low
    x[:3, : V - 700] = low
    x[3:, (torch.arange(V, device=DEV) % 50) != 7] = low
    x[2] -= 900 if dtype != HF else 200
    keep = [torch.arange(V - 700, V, device=DEV)] * 3 + [torch.arange(7, V, 50, device=DEV)] * 3
    g = _gen(5)
    t = torch.stack([c[torch.randint(0, c.numel(), (1,), device=DEV, generator=g)][0] for c in keep])
    ids = torch.stack([c[torch.randperm(c.numel(), device=DEV, generator=g)[:k]] for c in keep])
    top = torch.randn(N, k, device=DEV, generator=g) * 3
    coef = torch.randn(N, device=DEV, generator=g)
    logp, dx = O.token_logprobs_grad(x, t, coef)
    z = torch.where(x.double() <= torch.finfo(dtype).min, -float("inf"), x.double())  # the lowest value has p = 0 too
    want, grad, mass = oracle.logprobs(z, t, None, coef)
    oracle.close_logp(logp, want, torch.where(z.isinf(), 0.0, z), None)
    oracle.close_grad(dx, torch.where(z.isinf(), 0.0, grad), coef, mass, dtype)
    w = torch.ones(N, device=DEV)
    for lse in (None, torch.logsumexp(top, 1) + 0.5):
        loss, dx = O.distill_loss_grad(x, ids, top, lse, w)
        for r in range(N):  # the kept columns alone are the same problem
            at = torch.searchsorted(keep[r], ids[r])[None]
            want, grad, mass = oracle.distill(x[r:r + 1, keep[r]], at, top[r:r + 1], None if lse is None else lse[r:r + 1],
                                              w[:1], None, 1.0)
            oracle.close_logp(loss[r:r + 1], want, x[r:r + 1, keep[r]], None, factor=8)
            oracle.close_grad(dx[r:r + 1, keep[r]], grad, w[:1], mass, dtype)
        assert int((dx != 0).sum()) <= sum(c.numel() for c in keep)
    values, at, lse = O.top_logits(x, k)
    assert torch.equal(at, torch.sort(x.double(), dim=1, descending=True, stable=True)[1][:, :k])
    oracle.close_logp(lse, torch.logsumexp(z, 1), torch.where(z.isinf(), 0.0, z), None)


@pytest.mark.parametrize("kind", O.KINDS)
@pytest.mark.parametrize("cu_type", [torch.int32, torch.int64])
def test_pairs(kind, cu_type):
    T = 7001
    cu = [0, 1, 1, 900, 2900, 2901, 2901, 6000, 6998]
    g = _gen(2)
    lp, ref = (-torch.rand(T, device=DEV, generator=g) * 3 for _ in range(2))
    cut = torch.tensor(cu, dtype=cu_type, device=DEV)
    smooth = 0.05 if kind == "sigmoid" else 0.0
    for r in (ref, None):
        loss, rewards, grad = O.preference_loss_grad(lp, r, cut, beta=0.02, label_smoothing=smooth, kind=kind)
        want = oracle.pairs(lp, r, cu, kind, 0.02, smooth, 0.25)
        # the sums run over up to 3,100 values of 3 at most: 2^-24 * 9300 * a few, times beta
        size = float(want[1].abs().max()) / 0.02
        assert torch.allclose(rewards.double(), want[1], rtol=1e-5, atol=1e-2 * 0.02)
        if kind == "ipo":  # a square of a sum
            assert torch.allclose(loss.double(), want[0], rtol=1e-4, atol=1e-5 * size * size)
        else:
            assert torch.allclose(loss.double(), want[0], rtol=1e-4, atol=2e-4)
        assert torch.allclose(grad.double(), want[2], rtol=1e-3, atol=1e-5)
        assert bool((grad[6998:] == 0).all())
        leaf = lp.clone().requires_grad_()
        l2, r2 = O.preference_loss(leaf, r, cut, 0.02, smooth, kind)
        c = torch.rand(4, device=DEV, generator=g)
        (l2 * c).sum().backward()
        seq = torch.tensor(cu).diff().to(DEV)
        per = torch.nn.functional.pad((c * 4).repeat_interleave(2).repeat_interleave(seq), (0, T - 6998))
        assert torch.equal(l2.detach(), loss) and torch.allclose(leaf.grad, grad * per, rtol=1e-5, atol=1e-9)


def test_pairs_many_and_malformed():
    g = _gen(9)
    P = 700
    lens = torch.randint(0, 9, (2 * P,), generator=torch.Generator().manual_seed(1))
    cu = [0] + lens.cumsum(0).tolist()
    lp = torch.randn(cu[-1], device=DEV, generator=g)
    loss, rewards, grad = O.preference_loss_grad(lp, None, torch.tensor(cu, device=DEV), beta=0.5)
    want = oracle.pairs(lp, None, cu, "sigmoid", 0.5, 0.0, 1 / P)
    for a, b in zip((loss, rewards, grad), want):
        assert torch.allclose(a.double(), b, rtol=1e-5, atol=1e-5)
    bad = torch.tensor([5, 3, 40, 20, 1 << 30, -7, 9], device=DEV)  # read as 5, 5, 40, 40, T, T, T
    a = O.preference_loss_grad(lp, None, bad)
    b = O.preference_ref(lp.cpu(), None, bad.cpu(), 0, 0.1, 0.0, 1 / 3)
    for u, v in zip(a, b):
        assert torch.allclose(u.cpu(), v, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("T,V,dtype,kind", [(1, 4096, BF, "sigmoid"), (60, 5003, HF, "ipo"), (200, 32768, BF, "hinge"),
                                            (64, 262144, BF, "sigmoid")])
def test_preference_from_logits(T, V, dtype, kind):
    x = _x(T, V, dtype, T)
    g = _gen(4)
    t = torch.randint(0, V, (T,), device=DEV, generator=g)
    cu = [0, T // 5, T // 2, T // 2, T - T // 6]
    t[: T // 9] = -100
    ref = -torch.rand(T, device=DEV, generator=g) * 20
    ref[: T // 9] = float("nan")
    loss, rewards, logps, dx = O.preference_logits_grad(x, t, ref, torch.tensor(cu, device=DEV), kind=kind, softcap=30.0)
    lp64, _, _ = oracle.logprobs(x, t, 30.0, torch.zeros(T, device=DEV))
    oracle.close_logp(logps, lp64, x, 30.0)
    l64, r64, g64 = oracle.pairs(lp64, torch.where(t == -100, 0.0, ref), cu, kind, 0.1, 0.0, 0.5)
    _, grad, mass = oracle.logprobs(x, t, 30.0, g64)
    assert torch.allclose(rewards.double(), r64, rtol=1e-4, atol=1e-4)
    assert torch.allclose(loss.double(), l64, rtol=1e-3, atol=1e-3)
    # the pair's coefficient itself carries up to 1e-4 of relative error
    tol = (1.01 * oracle.UNIT[dtype] + 1e-4) * grad.abs() + (2.0 ** -16) * g64.abs()[:, None] * mass + oracle.TINY[dtype]
    assert bool(((dx.double() - grad).abs() <= tol).all())
    assert bool((dx[: T // 9] == 0).all()) and bool((dx[cu[-1]:] == 0).all())


def test_expanded_rows_and_empty():
    row = _x(1, 5003, BF, 2)
    x = row.expand(6, 5003)
    t = torch.arange(6, device=DEV)
    leaf = x.detach().requires_grad_()
    logp = O.token_logprobs(leaf, t)
    dx, = torch.autograd.grad(logp.sum(), leaf)
    want, grad, mass = oracle.logprobs(x, t, None, torch.ones(6, device=DEV))
    oracle.close_logp(logp.detach(), want, x, None)
    oracle.close_grad(dx, grad, torch.ones(6, device=DEV), mass, BF)
    none = x[:0]
    assert O.token_logprobs(none, t[:0]).shape == (0,)
    v, i, lse = O.top_logits(none, 4)
    assert v.shape == (0, 4) and lse.shape == (0,)
    loss, d = O.distill_loss_grad(none, t[:0, None], torch.zeros(0, 1, device=DEV))
    assert loss.shape == (0,) and d.shape == (0, 5003)
    loss, _, grad = O.preference_loss_grad(torch.ones(3, device=DEV), None, torch.zeros(1, dtype=torch.int64, device=DEV))
    assert loss.shape == (0,) and grad.tolist() == [0, 0, 0]


def test_offsets_past_32_bits():
    """More than 2^31 logits: the last rows, against the same rows alone."""
    N, V = 8240, 262144
    if torch.cuda.mem_get_info()[0] < 14 << 30:
        pytest.skip("needs 14 GB of free memory")
    x = torch.empty(N, V, dtype=BF, device=DEV)
    x.normal_(generator=_gen(3))
    t = torch.randint(0, V, (N,), device=DEV, generator=_gen(4))
    ids, top = t[:, None], torch.zeros(N, 1, device=DEV)
    values, at, lse = O.top_logits(x, 3)
    logp = O.token_logprobs(x, t)
    tail = x[-9:].clone()
    few = O.top_logits(tail, 3)
    assert torch.equal(values[-9:], few[0]) and torch.equal(at[-9:], few[1])
    # (sums: a row of a small batch is split over more blocks, in another order)
    assert torch.allclose(lse[-9:], few[2], rtol=1e-6, atol=1e-6)
    assert torch.allclose(logp[-9:], O.token_logprobs(tail, t[-9:]), rtol=1e-6, atol=1e-6)
    loss, dx = O.distill_loss_grad(x, ids, top, softcap=30.0, out=x)
    loss2, dx2 = O.distill_loss_grad(tail, ids[-9:], top[-9:], softcap=30.0)
    assert torch.allclose(loss[-9:], loss2, rtol=1e-5, atol=1e-5)
    assert torch.allclose(dx[-9:].float(), dx2.float(), rtol=2.0 ** -7, atol=1e-9)


def _every_call(x, t, ids, top, w, cu):
    out = list(O.top_logits(x, 40, softcap=30.0))
    leaf = x.detach().requires_grad_()
    logp = O.token_logprobs(leaf, t, softcap=30.0)
    out += [logp.detach(), torch.autograd.grad(logp.sum(), leaf)[0]]
    out += list(O.distill_loss_grad(x, ids, top, None, w, softcap=30.0))
    out += list(O.distill_loss_grad(x, ids, top, torch.logsumexp(top, 1), w, softcap=30.0))
    out += list(O.preference_logits_grad(x, t, None, cu, softcap=30.0))
    return out


def test_streams_and_repeats():
    """The same bits on every run, on another stream, and as a CUDA graph."""
    x = _x(500, 50001, BF, 1)
    t = torch.randint(0, 50001, (500,), device=DEV, generator=_gen(1))
    ids, top = _teacher(500, 50001, 30, 2)
    w = torch.rand(500, device=DEV, generator=_gen(3))
    cu = torch.tensor([0, 100, 300, 301, 480], device=DEV)
    first = _every_call(x, t, ids, top, w, cu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        moved = x + 0  # made on this stream: a launch on another one would race with it
        second = _every_call(moved, t, ids, top, w, cu)
        graph = torch.cuda.CUDAGraph()
    s.synchronize()
    for a, b in zip(first, second):
        assert torch.equal(a, b)
    with torch.cuda.graph(graph, stream=s):
        third = _every_call(x, t, ids, top, w, cu)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(first, third):
        assert torch.equal(a, b)


@pytest.mark.parametrize("what", list(refusals("cpu")))
def test_refusals(what):
    with pytest.raises(ValueError):
        refusals(DEV)[what]()


def test_native_refusals():
    x = _x(4, 64, BF)
    t = torch.zeros(4, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="contiguous"):
        O.token_logprobs(_x(64, 4, BF).t(), t)
    with pytest.raises(RuntimeError, match="bfloat16, float16 or float32"):
        O.top_logits(x.double(), 2)
    with pytest.raises(RuntimeError, match="another device"):
        O.token_logprobs(x, t.cpu())
    with pytest.raises(RuntimeError, match="another device"):
        O.distill_loss(x, t[:, None], torch.zeros(4, 1))
    with pytest.raises(RuntimeError, match="device"):
        O.preference_loss(torch.zeros(4, device=DEV), None, torch.tensor([0, 1, 4]))
    with pytest.raises(RuntimeError, match="apart"):
        O.distill_loss_grad(x, t[:, None], torch.zeros(4, 1, device=DEV), out=x[:1].expand(4, 64))


def test_exponential_alone():
    """Rows whose sum is 2^q equal terms e^d with d close to -q ln 2, so that its logarithm is close to 0 and nothing but
    the exponential rounds: a thread's first four vectors are masked (its sum's reference is 0 then), its others hold
    two terms at most in each of two partial sums, and the sums of threads are powers of two times one term."""
    V, per = 8188, 64
    i = torch.arange(1024, device=DEV)
    place = 4096 + 4 * (i % 256) + i // 256 % 2 + 1024 * (i // 512)
    delta = torch.linspace(-0.345, 0.345, per, dtype=torch.float64, device=DEV)
    q = torch.arange(11, device=DEV).repeat_interleave(per)
    d = (delta.repeat(11) - q * math.log(2)).float()
    x = torch.where(i < (1 << q).unsqueeze(1), d.unsqueeze(1), -float("inf"))
    whole = torch.full((q.numel(), V), -float("inf"), device=DEV)
    whole[:, place] = x
    want = d.double() + q * math.log(2)
    # ex2's 2^-22; ln 2 and log2 e in fp32, the roundings of r and of its product: 6e-8; the logarithm's two units
    assert float((O.top_logits(whole, 1)[2].double() - want).abs().max()) <= 3 * 2.0 ** -23


@pytest.mark.parametrize("V", [8200, 12005, 16301])
@pytest.mark.parametrize("dtype", [BF, FP])
def test_two_blocks_a_row(dtype, V):
    """Half a warp merges the shares of two blocks, and each lane by its own branch: shares of masked columns alone, of
    NaN and of numbers side by side; the same bits again and again."""
    inf, nan = float("inf"), float("nan")
    x = _x(9, V, dtype, V)
    x[0, : V // 2 + 64] = -inf      # nothing in the first block
    x[1, V // 2 - 64:] = -inf       # nothing in the second one
    x[2, V - 1000] = nan
    x[3, 1000] = inf
    x[4, (torch.arange(V, device=DEV) // 256) % 2 == 0] = -inf  # nothing for some of the warps
    x[5] = -inf
    x[6, : V - 1] = -inf
    x[7, :2100] = -inf
    t = torch.full((9,), V - 1, device=DEV)
    t[1] = 5
    want, grad = O.token_logprobs_ref(x.double(), t)
    dref = grad(torch.ones(9, device=DEV))
    ids, top = t[:, None], torch.zeros(9, 1, device=DEV)
    loss64, _ = O.distill_ref(x.double(), ids, top.double(), torch.ones(9, device=DEV))
    first = None
    for _ in range(20):
        logp, dx = O.token_logprobs_grad(x, t)
        loss, dd = O.distill_loss_grad(x, ids, top, torch.ones(9, device=DEV))
        lse = O.top_logits(x, 3)[2]
        out = [logp, dx, loss, dd, lse]
        first = first or out
        for a, b in zip(out, first):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0)) and torch.equal(a.isnan(), b.isnan())
    assert torch.equal(logp.isnan(), want.isnan()) and want.isnan().tolist() == [False] * 2 + [True] * 2 + [False, True] + [False] * 3
    ok = ~want.isnan()
    assert torch.allclose(logp[ok].double(), want[ok], rtol=1e-5, atol=1e-5)
    oracle.close_grad(dx[ok], dref[ok], torch.ones(int(ok.sum()), device=DEV), torch.ones_like(dref[ok]), dtype)
    assert torch.equal(loss.isfinite(), loss64.isfinite())
    some = loss64.isfinite()
    assert torch.allclose(loss[some].double(), loss64[some], rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("V", [2 ** 31 - 100, 2 ** 31 - 4096, 2 ** 31 + 5])
def test_too_many_columns(V):
    """Rows whose column numbers would pass 32 bits within a loop are refused (nothing is read: one element, expanded)."""
    x = torch.zeros(1, 1, device=DEV, dtype=BF).expand(2, V)
    t = torch.zeros(2, dtype=torch.int64, device=DEV)
    for call in (lambda: O.top_logits(x, 1), lambda: O.token_logprobs(x, t), lambda: O.token_logprobs_grad(x, t),
                 lambda: O.distill_loss_grad(x, t[:, None], torch.zeros(2, 1, device=DEV)),
                 lambda: O.preference_logits_grad(x, t, None, torch.tensor([0, 1, 2], device=DEV))):
        with pytest.raises(ValueError, match="vocabulary"):
            call()


@pytest.mark.parametrize("dtype,cap", [(BF, 30.0), (HF, None), (FP, None), (FP, 30.0)])
def test_repeated_ids(dtype, cap):
    for V, ids, top, lse in oracle.repeated_cases(DEV):
        x = _x(ids.shape[0], V, dtype, V)
        w = torch.ones(ids.shape[0], device=DEV)
        one = oracle.merged(ids, top, 1.5)
        want, grad, mass = oracle.distill(x, *one, lse, w, cap, 1.5)
        mass = mass + oracle.rest_mass(x, *one, lse, cap, 1.5)
        leaf = x.detach().requires_grad_()
        auto = O.distill_loss(leaf, ids, top, lse, w, softcap=cap, temperature=1.5)
        auto = auto.detach(), torch.autograd.grad(auto.sum(), leaf)[0]
        for loss, dx in (O.distill_loss_grad(x, ids, top, lse, w, softcap=cap, temperature=1.5), auto):
            oracle.close_logp(loss, want, x, cap, 1.5, factor=8)
            oracle.close_grad(dx, grad, 1.5 * w, mass, dtype)


def test_overwritten_logits():
    for y in overwritten(DEV):
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()


def test_overwritten_logits_of_inference():
    with torch.inference_mode():
        x = _x(4, 300, BF, 1)
        t = torch.arange(4, device=DEV)
        logp, dx = O.token_logprobs_grad(x.clone(), t)
        logp2, dx2 = O.token_logprobs_grad(x, t, out=x)
    assert dx2 is x and torch.equal(dx, x) and torch.equal(logp, logp2)


@pytest.mark.parametrize("cap", [None, 40.0])
def test_small_coefficients_far_from_the_reference(cap):
    """Most logits 76 below the largest one, which no thread sees first: the sums are of e^76 then, and a small
    coefficient divided by one has to keep its digits."""
    N, V = 5, 262144
    x = torch.randn(N, V, device=DEV, generator=_gen(1)) * 0.3 - 75.0
    t = torch.arange(N, device=DEV)
    x[:, V - 100] = 75.0 if cap else 1.0
    coef = torch.tensor([1.0, 1e-6, 1e-9, 1e-11, -1e-12], device=DEV)
    logp, dx = O.token_logprobs_grad(x, t, coef, softcap=cap)
    want, grad, mass = oracle.logprobs(x, t, cap, coef)
    oracle.close_logp(logp, want, x, cap)
    oracle.close_grad(dx, grad, coef, mass, FP)
    w = coef.abs()
    ids, top = torch.stack([t, t + 9], 1), torch.zeros(N, 2, device=DEV)
    for lse in (None, torch.full((N,), 2.0, device=DEV)):
        loss, dx = O.distill_loss_grad(x, ids, top, lse, w, softcap=cap)
        want, grad, mass = oracle.distill(x, ids, top, lse, w, cap, 1.0)
        oracle.close_logp(loss, want, x, cap, factor=8)
        oracle.close_grad(dx, grad, w, mass + oracle.rest_mass(x, ids, top, lse, cap, 1.0), FP)


def test_impossible_answers():
    impossible_answers(DEV)


WIDE = [(BF, 50.0, 0.25, None), (BF, 100.0, 1.0, None), (FP, 100.0, 1.0, None), (HF, 200.0, 0.7, None), (BF, None, 1.0, -1e9),
        (FP, None, 1.0, -1e9), (HF, None, 1.0, -3e4), (BF, None, 2.0, -1e4)]


def _wide_row(N, V, dtype, masked, seed=1):
    """An ordinary body with a few peaks; `masked` is the value of all columns but the last 9000."""
    x = torch.randn(N, V, device=DEV, generator=_gen(seed)) * 2.5 - 5.0
    x[:, 5::V // 12] = 12.0
    if masked is not None:
        x[:, : V - 9000] = masked
    return x.to(dtype)


@pytest.mark.parametrize("dtype,cap,temp,masked", WIDE)
def test_wide_caps_and_finite_masks(dtype, cap, temp, masked):
    N, V = 6, 100003
    x = _wide_row(N, V, dtype, masked)
    x[0] = (x[0].float() * 8).to(dtype)  # beyond what one reference can hold
    t = torch.randint(V - 9000, V, (N,), device=DEV, generator=_gen(2))
    coef = torch.randn(N, device=DEV, generator=_gen(3))
    logp, dx = O.token_logprobs_grad(x, t, coef, softcap=cap)
    want, grad, mass = oracle.logprobs(x, t, cap, coef)
    big = torch.where(x < -9000, 0.0, x.float())  # what the sums are formed of
    oracle.close_logp(logp, want, big, cap)
    oracle.close_grad(dx, grad, coef, mass, dtype)
    lse = O.top_logits(x, 4, softcap=cap, temperature=temp)[2]
    oracle.close_logp(lse, torch.logsumexp(oracle.z64(x, cap) / temp, 1), big, cap, temp)
    ids, top, w = t[:, None], torch.zeros(N, 1, device=DEV), torch.ones(N, device=DEV)
    for rest in (None, torch.ones(N, device=DEV)):
        loss, dx = O.distill_loss_grad(x, ids, top, rest, w, softcap=cap, temperature=temp)
        want, grad, mass = oracle.distill(x, ids, top, rest, w, cap, temp)
        oracle.close_logp(loss, want, big, cap, temp, factor=8)
        oracle.close_grad(dx, grad, w * temp, mass + oracle.rest_mass(x, ids, top, rest, cap, temp), dtype)


@pytest.mark.parametrize("dtype,cap,temp", [w[:3] for w in WIDE if w[0] != HF and w[1]])
def test_wide_caps_take_the_fast_sum(dtype, cap, temp):
    """The time of one call against that with cap 30 at temperature 1: the element by element form takes more than four
    times as long."""
    def best(x, cap, temp):
        O.top_logits(x, 20, cap, temp)
        times = []
        for _ in range(7):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            O.top_logits(x, 20, cap, temp)
            b.record()
            b.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    x = _wide_row(1024, 262144, dtype, None)
    assert best(x, cap, temp) < 2.5 * best(x, 30.0, 1.0)


def test_small_probabilities_of_fp32_gradients():
    """Columns far below the largest logit, on a grid on which their differences to it are exact: a gradient's error is
    that of the exponential alone, 2^-22 of ex2 and up to 2^-23 of the reduction (72 times what fp32 leaves out of ln 2)."""
    N, V = 4, 50003
    x = -10.0 - torch.randint(0, 20 << 10, (N, V), device=DEV, generator=_gen(1)) / 1024.0
    x[:, 0] = 20.0
    t = torch.zeros(N, dtype=torch.int64, device=DEV)
    _, dx = O.token_logprobs_grad(x, t)
    want, grad, _ = oracle.logprobs(x, t, None, torch.ones(N, device=DEV))
    assert float((dx.double() / grad - 1)[:, 1:].abs().max()) < 2.0 ** -21
    ids, top = t[:, None], torch.zeros(N, 1, device=DEV)
    _, dx = O.distill_loss_grad(x, ids, top)
    want, grad, _ = oracle.distill(x, ids, top, None, torch.ones(N, device=DEV), None, 1.0)
    assert float((dx.double() / grad - 1)[:, 1:].abs().max()) < 2.0 ** -21


def test_nothing_to_match():
    nothing_to_match(DEV)
