"""Vocabulary objectives on CPU tensors (the plain PyTorch forms): against the 64-bit definitions, the
gradients against finite differences, the edge cases' rules, and every refusal."""
import pytest
import torch

import objective_oracle as oracle
from micro_engram_fork_b200.ops import objectives as O


def _teacher(N, V, k, seed=0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(V, generator=g)[:k] for _ in range(N)])
    return ids, torch.randn(N, k, generator=g) * 3


@pytest.mark.parametrize("cap", [None, 3.0, 30.0])
def test_differences(cap):
    x = (torch.randn(5, 37, dtype=torch.float64) * 5).requires_grad_()
    t = torch.tensor([3, -100, 36, 0, 9])
    assert torch.autograd.gradcheck(lambda x: O.token_logprobs(x, t, softcap=cap), (x,))
    ids, top = _teacher(5, 37, 6)
    ids[1, 4:] = -1
    ids[2] = 40
    w = torch.tensor([1.0, 0.5, 2.0, 0.0, 1.0], dtype=torch.float64)
    for lse in (None, torch.full((5,), 9.0, dtype=torch.float64)):
        assert torch.autograd.gradcheck(
            lambda x: O.distill_loss(x, ids, top.double(), lse, w, softcap=cap, temperature=1.5), (x,))
    lp = torch.randn(12, dtype=torch.float64).requires_grad_()
    cu = torch.tensor([1, 4, 4, 7, 11])
    for kind in O.KINDS:
        assert torch.autograd.gradcheck(lambda v: O.preference_loss(v, torch.ones(12), cu, 0.3, kind=kind)[0], (lp,))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("cap", [None, 30.0])
def test_plain_forms(dtype, cap):
    N, V, k = 7, 301, 9
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(N, V, generator=g) * 4).to(dtype)
    x[3, 17:40] = -float("inf")
    t = torch.randint(0, 17, (N,), generator=g)
    t[2] = -100
    coef = torch.randn(N, generator=g)
    leaf = x.clone().requires_grad_()
    logp = O.token_logprobs(leaf, t, softcap=cap)
    logp.backward(coef)
    want, grad, p = oracle.logprobs(x, t, cap, coef)
    oracle.close_logp(logp.detach(), want, x, cap)
    oracle.close_grad(leaf.grad, grad, coef, p, dtype)

    ids, top = _teacher(N, V, k, 2)
    ids[3] = torch.arange(k)
    w = torch.tensor([1.0, 0.0, 0.3, 2.0, 1.0, 1.0, 1.0])
    for lse in (None, torch.logsumexp(top, 1) + 0.5):
        loss, dx = O.distill_loss_grad(x, ids, top, lse, w, softcap=cap, temperature=2.0)
        want, grad, mass = oracle.distill(x, ids, top, lse, w, cap, 2.0)
        oracle.close_logp(loss, want, x, cap, factor=8)
        oracle.close_grad(dx, grad, 2.0 * w, mass, dtype)

    values, at, lse = O.top_logits(x, 20, softcap=cap, temperature=2.0)
    for r in range(N):
        order = sorted(range(V), key=lambda j: (-float(x[r, j]), j))[:20]
        assert at[r].tolist() == order
    z = oracle.z64(x, cap)
    assert torch.allclose(values.double(), z.gather(1, at), rtol=1e-6, atol=1e-6)
    assert torch.allclose(lse.double(), torch.logsumexp(z / 2.0, 1), rtol=1e-6, atol=1e-6)


@pytest.mark.parametrize("kind", O.KINDS)
def test_pairs(kind):
    cu = [0, 3, 3, 10, 16, 17, 20]
    g = torch.Generator().manual_seed(3)
    lp, ref = torch.randn(22, generator=g), torch.randn(22, generator=g)
    smooth = 0.1 if kind == "sigmoid" else 0.0
    loss, rewards, grad = O.preference_loss_grad(lp, ref, torch.tensor(cu), beta=0.2, label_smoothing=smooth, kind=kind)
    want = oracle.pairs(lp, ref, cu, kind, 0.2, smooth, 1 / 3)
    for a, b in zip((loss, rewards, grad), want):
        assert torch.allclose(a.double(), b, rtol=1e-5, atol=1e-6)
    assert bool((grad[20:] == 0).all())
    leaf = lp.clone().requires_grad_()
    O.preference_loss(leaf, ref, torch.tensor(cu), 0.2, smooth, kind)[0].mean().backward()
    assert torch.allclose(leaf.grad, grad, rtol=1e-6, atol=1e-8)


def test_preference_from_logits():
    cu = torch.tensor([0, 4, 9])
    x = torch.randn(10, 33)
    t = torch.randint(0, 33, (10,))
    t[[0, 4, 5]] = -100
    ref = torch.randn(10)
    ref[0] = float("nan")  # not read at an untrained token
    loss, rewards, logps, dx = O.preference_logits_grad(x, t, ref, cu, softcap=8.0)
    leaf = x.clone().requires_grad_()
    lp = O.token_logprobs(leaf, t, softcap=8.0)
    l2, r2 = O.preference_loss(lp, torch.where(t == -100, 0.0, ref), cu)
    l2.mean().backward()
    assert torch.allclose(loss, l2) and torch.allclose(rewards, r2) and torch.allclose(logps, lp)
    assert torch.allclose(dx, leaf.grad, atol=1e-7) and bool((dx[[0, 4, 5, 9]] == 0).all())


def test_edges():
    nan, inf = float("nan"), float("inf")
    x = torch.randn(6, 11)
    x[0] = nan       # untrained below
    x[1, 3] = nan
    x[2, 4] = inf
    x[3] = -inf
    t = torch.tensor([-100, 0, 0, 0, 11, -7])
    leaf = x.clone().requires_grad_()
    logp = O.token_logprobs(leaf, t)
    assert logp[0] == 0 and bool(logp[1:].isnan().all())
    logp.sum().backward()
    assert bool((leaf.grad[0] == 0).all()) and bool(leaf.grad[[1, 2, 3, 4, 5]].isnan().all())
    assert bool(O.token_logprobs(x[2:4], t[2:4], softcap=5.0).isfinite().all())
    ids, top = _teacher(6, 11, 3)
    loss, dx = O.distill_loss_grad(x, ids, top, weights=torch.tensor([0.0, 1, 1, 1, 1, 1]))
    assert loss[0] == 0 and bool((dx[0] == 0).all()) and bool(loss[1:4].isnan().all()) and bool(loss[4:].isfinite().all())
    _, at, _ = O.top_logits(x, 2)
    assert at[1, 0] == 3 and at[2, 0] == 4 and at[3].tolist() == [0, 1] and at[0].tolist() == [0, 1]


def test_empty():
    x = torch.randn(0, 9, requires_grad=True)
    none = torch.empty(0, dtype=torch.int64)
    logp = O.token_logprobs(x, none)
    logp.sum().backward()
    assert logp.shape == (0,) and x.grad.shape == (0, 9)
    v, i, lse = O.top_logits(x, 3)
    assert v.shape == (0, 3) and i.shape == (0, 3) and lse.shape == (0,)
    loss, rewards, grad = O.preference_loss_grad(torch.randn(4), None, torch.tensor([0]))
    assert loss.shape == (0,) and rewards.shape == (0, 2) and grad.tolist() == [0, 0, 0, 0]


def test_leading_dimensions_and_out():
    x = torch.randn(2, 3, 17)
    t = torch.randint(0, 17, (2, 3))
    assert torch.equal(O.token_logprobs(x, t), O.token_logprobs(x.view(6, 17), t.view(6)).view(2, 3))
    assert O.token_logprobs(x[0, 0], t[0, 0]).shape == ()
    ids, top = _teacher(6, 17, 4)
    loss, dx = O.distill_loss_grad(x, ids.view(2, 3, 4), top.view(2, 3, 4))
    y = x.clone()
    loss2, dx2 = O.distill_loss_grad(y, ids.view(2, 3, 4), top.view(2, 3, 4), out=y)
    assert dx2 is y and torch.equal(dx, y) and torch.equal(loss, loss2) and loss.shape == (2, 3)


def test_one_call_forms():
    x = torch.randn(6, 40)
    t = torch.tensor([0, 39, -100, 5, 6, 7])
    coef = torch.randn(6)
    leaf = x.clone().requires_grad_()
    logp = O.token_logprobs(leaf, t, softcap=4.0)
    logp.backward(coef)
    got, dx = O.token_logprobs_grad(x, t, coef, softcap=4.0)
    assert torch.equal(got, logp.detach()) and torch.equal(dx, leaf.grad)
    got, dx = O.token_logprobs_grad(x.view(2, 3, 40), t.view(2, 3), softcap=4.0)
    assert got.shape == (2, 3) and dx.shape == (2, 3, 40)
    assert torch.equal(dx.view(6, 40), O.token_logprobs_grad(x, t, torch.ones(6), softcap=4.0)[1])


def refusals(dev):
    """(what is refused, the call) on `dev`; shared with the GPU tests."""
    x = torch.randn(4, 9, device=dev)
    t = torch.zeros(4, dtype=torch.int64, device=dev)
    ids, top = torch.zeros(4, 2, dtype=torch.int64, device=dev), torch.zeros(4, 2, device=dev)
    lp, cu = torch.zeros(6, device=dev), torch.tensor([0, 2, 6], device=dev)
    return {
        "k 0": lambda: O.top_logits(x, 0),
        "k above the vocabulary": lambda: O.top_logits(x, 10),
        "k above 256": lambda: O.top_logits(torch.randn(2, 400, device=dev), 257),
        "softcap": lambda: O.token_logprobs(x, t, softcap=-1.0),
        "temperature": lambda: O.top_logits(x, 2, temperature=0.0),
        "integer logits": lambda: O.token_logprobs(t.view(2, 2), t[:2]),
        "empty vocabulary": lambda: O.token_logprobs(x[:, :0], t),
        "targets' shape": lambda: O.token_logprobs(x, t[:3]),
        "targets' type": lambda: O.token_logprobs(x, t.float()),
        "coefficients": lambda: O.token_logprobs_grad(x, t, torch.ones(3, device=dev)),
        "teacher's shapes": lambda: O.distill_loss(x, ids, top[:, :1]),
        "teacher's rows": lambda: O.distill_loss(x, ids[:3], top[:3]),
        "teacher's ids": lambda: O.distill_loss(x, ids.float(), top),
        "teacher's size": lambda: O.distill_loss(x, ids.new_zeros(4, 257), top.new_zeros(4, 257)),
        "no entries": lambda: O.distill_loss(x, ids[:, :0], top[:, :0]),
        "teacher_lse": lambda: O.distill_loss(x, ids, top, teacher_lse=top),
        "weights": lambda: O.distill_loss(x, ids, top, weights=torch.ones(3, device=dev)),
        "out's type": lambda: O.distill_loss_grad(x, ids, top, out=x.half()),
        "out's shape": lambda: O.distill_loss_grad(x, ids, top, out=x[:2]),
        "kind": lambda: O.preference_loss(lp, lp, cu, kind="other"),
        "beta": lambda: O.preference_loss(lp, lp, cu, beta=0.0),
        "label smoothing": lambda: O.preference_loss(lp, lp, cu, label_smoothing=0.6),
        "label smoothing of hinge": lambda: O.preference_loss(lp, lp, cu, label_smoothing=0.1, kind="hinge"),
        "odd sequences": lambda: O.preference_loss(lp, lp, cu[:2]),
        "offsets' type": lambda: O.preference_loss(lp, lp, cu.float()),
        "reference's shape": lambda: O.preference_loss(lp, lp[:5], cu),
        "log-probabilities' shape": lambda: O.preference_loss(lp.view(2, 3), lp, cu),
        "logits' dimensions": lambda: O.preference_logits_grad(x.view(2, 2, 9), t, lp[:4], cu),
    }


@pytest.mark.parametrize("what", list(refusals("cpu")))
def test_refusals(what):
    with pytest.raises(ValueError):
        refusals("cpu")[what]()


@pytest.mark.parametrize("cap", [None, 30.0])
def test_repeated_ids(cap):
    """A repeated id is one entry with the sum of its probabilities: value, gradient, and whether there is a rest."""
    for V, ids, top, lse in oracle.repeated_cases("cpu"):
        N = ids.shape[0]
        x = torch.randn(N, V, generator=torch.Generator().manual_seed(V)) * 4
        w = torch.ones(N)
        one_ids, one_top = oracle.merged(ids, top, 1.5)
        want, grad, mass = oracle.distill(x, one_ids, one_top, lse, w, cap, 1.5)
        mass = mass + oracle.rest_mass(x, one_ids, one_top, lse, cap, 1.5)
        for loss, dx in (O.distill_loss_grad(x, ids, top, lse, w, softcap=cap, temperature=1.5),
                         O.distill_loss_grad(x, one_ids, one_top, lse, w, softcap=cap, temperature=1.5)):
            oracle.close_logp(loss, want, x, cap, 1.5, factor=8)
            oracle.close_grad(dx, grad, 1.5 * w, mass, torch.float32)


def test_repeated_ids_by_hand():
    """A student that is certain of the teacher's only token has nothing to learn, however often that token is named."""
    x = torch.full((1, 9), -200.0)
    x[0, 5] = 0.0
    loss, dx = O.distill_loss_grad(x, torch.tensor([[5, 5]]), torch.zeros(1, 2))
    assert abs(float(loss)) < 1e-6 and float(dx.abs().max()) < 1e-6
    x = torch.tensor([[0.3, -0.2]])
    lse = torch.tensor([1.5])
    a = O.distill_loss_grad(x, torch.tensor([[0, 0]]), torch.tensor([[0.0, 0.0]]), lse)
    b = O.distill_loss_grad(x, torch.tensor([[0]]), torch.tensor([[2.0]]).log(), lse)
    assert torch.allclose(a[0], b[0], atol=1e-6) and torch.allclose(a[1], b[1], atol=1e-6)


def overwritten(dev):
    """An earlier graph on the logits, and a call that overwrites them: the graph's backward has to refuse."""
    cu = torch.tensor([0, 2, 4], device=dev)
    t = torch.tensor([1, 2, 3, 4], device=dev)
    ids, top = t[:, None], torch.zeros(4, 1, device=dev)
    graphs = {"logprobs": lambda x: O.token_logprobs(x, t), "distill": lambda x: O.distill_loss(x, ids, top)}
    writes = {"logprobs": lambda z: O.token_logprobs_grad(z, t, out=z), "distill": lambda z: O.distill_loss_grad(z, ids, top, out=z),
              "preference": lambda z: O.preference_logits_grad(z, t, None, cu, out=z)}
    for graph in graphs.values():
        for write in writes.values():
            x = torch.randn(4, 9, device=dev, requires_grad=True)
            y = graph(x)
            version = x._version
            write(x.detach())
            assert x._version > version
            yield y
    x = torch.randn(2, 2, 9, device=dev, requires_grad=True)  # by way of flattened rows
    y = O.token_logprobs(x, t.view(2, 2))
    z = x.detach()
    O.distill_loss_grad(z, ids.view(2, 2, 1), top.view(2, 2, 1), out=z)
    yield y


def test_overwritten_logits():
    for y in overwritten("cpu"):
        with pytest.raises(RuntimeError, match="inplace"):
            y.sum().backward()


def impossible_answers(dev):
    """Pairs whose rejected / chosen answer has a token of probability 0, per kind: (loss, rewards, gradient) as the
    limits of the formulas have them (a NaN only where a difference of infinities has no limit)."""
    inf = float("inf")
    lp = torch.tensor([-1.0, -inf, -inf, -1.0, -1.0, -1.0], device=dev)
    ref = torch.zeros(6, device=dev)
    cu = torch.tensor([0, 1, 2, 3, 4, 5, 6], device=dev)  # rejected impossible, chosen impossible, neither
    want = {("sigmoid", 0.0): ([0.0, inf, 0.6931472], [0, 0, -0.1, 0.1, -0.05, 0.05]),
            ("sigmoid", 0.25): ([inf, inf, 0.6931472], [0.025, -0.025, -0.075, 0.075, -0.025, 0.025]),
            ("hinge", 0.0): ([0.0, inf, 1.0], [0, 0, -0.1, 0.1, -0.1, 0.1])}
    for (kind, smooth), (loss, grad) in want.items():
        got = O.preference_loss_grad(lp, ref, cu, 0.1, smooth, kind, scale=1.0)
        leaf = lp.clone().requires_grad_()
        auto, _ = O.preference_loss(leaf, ref, cu, 0.1, smooth, kind)
        for value, d in ((got[0], got[2]), (auto.detach(), torch.autograd.grad(auto.sum(), leaf)[0])):
            assert torch.allclose(value.cpu(), torch.tensor(loss)), (kind, smooth, value)
            assert torch.allclose(d.cpu(), torch.tensor(grad, dtype=torch.float32), atol=1e-7), (kind, smooth, d)
        assert torch.allclose(got[1].cpu(), torch.tensor([[-0.1, -inf], [-inf, -0.1], [-0.1, -0.1]]))


def test_impossible_answers():
    impossible_answers("cpu")


def nothing_to_match(dev):
    """Rows without an entry and without a rest: value 0 and gradient 0, whatever their logits hold."""
    nan, inf = float("nan"), float("inf")
    x = torch.randn(5, 40, device=dev)
    x[1, 3], x[2, 4], x[3] = nan, inf, -inf
    ids = torch.tensor([[-1, 40], [-1, -7], [41, -1], [-1, -1], [2, 3]], device=dev)
    top = torch.zeros(5, 2, device=dev)
    top[4] = -inf  # entries of probability 0 are none
    for cap in (None, 30.0):
        loss, dx = O.distill_loss_grad(x, ids, top, softcap=cap)
        leaf = x.clone().requires_grad_()
        auto = O.distill_loss(leaf, ids, top, softcap=cap)
        auto.sum().backward()
        for t in (loss, dx, auto.detach(), leaf.grad):
            assert bool((t == 0).all()), (cap, t)


def test_nothing_to_match():
    nothing_to_match("cpu")
