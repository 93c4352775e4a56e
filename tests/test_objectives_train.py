"""The objectives in the trainer and its head: per-token values and their gradients in the hidden states
against the objectives on the whole logits, the refusal of a split head, and the example (distillation and
preference training of a small random base), on CPU tensors and on the sm_100a kernels."""
import os
import sys

import pytest
import torch

import objective_oracle as oracle
from micro_engram_fork_b200.ops import objectives as O

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _shard(dev, V=1003, d=64, chunk=16, softcap=30.0):
    from micro_engram.train.head import VocabShard

    torch.manual_seed(0)
    W = (torch.randn(V, d) * 0.3).to(torch.bfloat16)
    return VocabShard(W, 0, 1, softcap=softcap, chunk_tokens=chunk, device=dev), W.to(dev)


@pytest.mark.parametrize("dev", DEVICES)
def test_head(dev):
    """Chunks of 16 tokens (the last one short), a vocabulary that is padded for the GEMMs."""
    shard, W = _shard(dev)
    N, k = 53, 12
    h = torch.randn(N, 64, device=dev).to(torch.bfloat16)
    z = (h @ W.t()).detach()  # the same bf16 logits up to one rounding
    z64 = oracle.z64(z, 30.0)
    values, ids, lse = shard.top_logits(h, k, temperature=1.5)
    want = z64.topk(k, dim=1)[0]
    # a bf16 logit of up to 32 is rounded at 2^-4: the two products may differ by a unit
    assert torch.allclose(values.double(), want, atol=0.13) and values.shape == ids.shape == (N, k)
    assert torch.allclose(lse.double(), torch.logsumexp(z64 / 1.5, 1), atol=0.02)
    assert ids.max() < W.shape[0]

    labels = torch.randint(0, W.shape[0], (N,), device=dev)
    labels[::5] = -100
    coef = torch.randn(N, device=dev)
    w = torch.rand(N, device=dev)
    w[3] = 0.0
    teacher = torch.randn(N, k, device=dev) * 3
    t_lse = torch.logsumexp(teacher, 1) + 0.2
    h64 = h.double().requires_grad_()
    x64 = h64 @ W.double().t()
    cases = {
        "logprobs": (lambda v: shard.token_logprobs(v, labels), O.token_logprobs_ref(x64.detach(), labels, 30.0)[0],
                     O.token_logprobs_ref(x64.detach(), labels, 30.0)[1](coef.double())),
        "distill": (lambda v: shard.distill(v, ids, teacher, t_lse, w, 1.5),
                    O.distill_ref(x64.detach(), ids, teacher.double(), t_lse, w, 30.0, 1.5)[0],
                    O.distill_ref(x64.detach(), ids, teacher.double(), t_lse, w, 30.0, 1.5)[1] * coef.double()[:, None]),
    }
    for name, (call, value, dx) in cases.items():
        leaf = h.clone().requires_grad_()
        got = call(leaf)
        assert got.shape == (N,) and got.dtype == torch.float32
        # logits rounded to bf16 (2^-9 of up to 16): a few hundredths in a value
        assert torch.allclose(got.detach().double(), value, atol=0.15), name
        (got * coef).sum().backward()
        dh = dx @ W.double()
        err = (leaf.grad.double() - dh).abs().max().item()
        assert err <= 3e-2 * dh.abs().max().item(), (name, err)
        with torch.no_grad():
            assert torch.allclose(call(h), got.detach(), rtol=1e-5, atol=1e-5), name


@pytest.mark.parametrize("dev", DEVICES)
def test_head_edges(dev):
    shard, W = _shard(dev)
    none = torch.zeros(0, 64, device=dev, dtype=torch.bfloat16)
    assert shard.token_logprobs(none, torch.zeros(0, dtype=torch.int64, device=dev)).shape == (0,)
    assert shard.top_logits(none, 3)[0].shape == (0, 3)
    with pytest.raises(ValueError):
        shard.top_logits(torch.zeros(2, 65, device=dev), 3)


def test_split_head_is_refused():
    from micro_engram.train.head import VocabShard

    shard = VocabShard(torch.randn(64, 8), 0, 2)
    with pytest.raises(ValueError):
        shard.top_logits(torch.randn(3, 8), 2)
    with pytest.raises(ValueError):
        shard.token_logprobs(torch.randn(3, 8), torch.zeros(3, dtype=torch.int64))


@pytest.mark.parametrize("dev", DEVICES)
def test_example(dev, monkeypatch, dist_env):
    if dev == "cpu":
        monkeypatch.setenv("MICRO_ENGRAM_CPU", "1")
    monkeypatch.syspath_prepend(os.path.join(ROOT, "examples"))
    import distill_and_prefer

    out = distill_and_prefer.main(steps=12, seq=96 if dev == "cpu" else 512)
    assert out["device"].startswith(dev)
    first, last = out["distill_loss"]
    assert first > 0 and last < 0.7 * first
    first, last = out["preference_loss"]
    assert abs(first - 0.6931) < 1e-2 and last < 0.5 * first and min(out["margins"]) > 0
    sys.modules.pop("distill_and_prefer", None)


def test_teacher_of_another_temperature():
    """teacher_lse is of one temperature; a batch that says which is refused at another one, where the rest is used."""
    from micro_engram.train.objectives import Distillation, record_teacher

    shard, _ = _shard("cpu", V=40)
    h = torch.randn(6, 64)

    class Teacher:
        vocab = shard

        def hidden(self, batch):
            return batch["h"]

    batch = {"h": h, "labels": torch.arange(6)}
    recorded = record_teacher(Teacher(), batch, 5, temperature=2.0)
    assert float(Distillation(2.0, with_rest=True)(shard, h, recorded)) < 1e-3
    with pytest.raises(ValueError, match="temperature"):
        Distillation(1.0, with_rest=True)(shard, h, recorded)
    with pytest.raises(ValueError, match="temperature"):
        Distillation(2.0, with_rest=True)(shard, h, record_teacher(Teacher(), batch, 5))
    Distillation(1.0)(shard, h, recorded)  # the entries alone are of no temperature
    own = {k: v for k, v in recorded.items() if k != "teacher_temperature"}  # records that do not say
    assert torch.equal(Distillation(2.0, with_rest=True)(shard, h, own), Distillation(2.0, with_rest=True)(shard, h, recorded))


@pytest.mark.parametrize("dev", DEVICES)
def test_trainer_feeds_the_objective(dev, monkeypatch, dist_env, tmp_path):
    """train() and train_step(bins) have the data set's batches only: an objective that needs more is refused before
    anything runs; the step's token count stays that of the trained tokens whatever the objective counts."""
    if dev == "cpu":
        monkeypatch.setenv("MICRO_ENGRAM_CPU", "1")
    monkeypatch.syspath_prepend(os.path.join(ROOT, "examples"))
    import distill_and_prefer as example
    from micro_engram.train.objectives import Distillation, NextToken, Preference, record_reference, record_teacher

    seq, vocab = 96, 4096
    trainer = example.make_trainer(str(tmp_path), seq, vocab)
    micro = trainer.plan.micro_batches(0, 0, 0)
    for objective, field in ((Distillation(), "teacher_ids"), (Distillation(with_rest=True), "teacher_lse"),
                             (Preference(), "cu_seqlens")):
        trainer.objective = objective
        for call in (trainer.train, lambda: trainer.train_step(micro)):
            with pytest.raises(ValueError, match=field):
                call()
    assert trainer.global_step == 0 and not os.path.exists(trainer.cfg.output_dir)
    lengths = [32, 24, 19, 16]
    batch = example.packed(lengths, vocab, seq, torch.Generator().manual_seed(1), trainer.device)
    batch["cu_seqlens"] = torch.tensor([0] + lengths, device=trainer.device).cumsum(0)
    trained = int((batch["labels"] != -100).sum())
    batch = record_reference(trainer, record_teacher(trainer, batch, 8))
    for objective in (NextToken(), Distillation(), Preference()):
        trainer.objective = objective
        logs = trainer.train_step(None, batches=[batch, batch])
        assert logs["tokens"] == 2 * trained
    assert abs(logs["loss"] - 0.6931) < 0.05  # a mean over the pairs
    trainer.objective = NextToken()
    assert trainer.train_step(micro)["tokens"] > 0
    sys.modules.pop("distill_and_prefer", None)


@pytest.mark.parametrize("dev", DEVICES)
def test_head_backward_again(dev):
    """The gradient is kept for a graph that is retained, released with one that is not, and not differentiable itself."""
    shard, W = _shard(dev, V=200)
    h = torch.randn(9, 64, device=dev).to(torch.bfloat16).requires_grad_()
    labels = torch.arange(9, device=dev)
    values = shard.token_logprobs(h, labels)
    first, = torch.autograd.grad(values.sum(), h, retain_graph=True)
    again, = torch.autograd.grad((2 * values).sum(), h)
    assert torch.equal(again, 2 * first)
    with pytest.raises(RuntimeError, match="second time|retain_graph"):
        torch.autograd.grad(values.sum(), h)
    values = shard.distill(h, labels[:, None], torch.zeros(9, 1, device=dev))
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(values.sum(), h, create_graph=True)


@pytest.mark.parametrize("dev", DEVICES)
def test_head_refuses_other_lengths(dev):
    """One value a token: longer or shorter arguments are refused, not cut to the hidden states."""
    shard, _ = _shard(dev, V=200)  # chunks of 16
    h = torch.randn(20, 64, device=dev).to(torch.bfloat16)
    for n in (0, 16, 19, 21, 32, 40):
        labels = torch.zeros(n, dtype=torch.int64, device=dev)
        ids, top, one = labels[:, None], torch.zeros(n, 1, device=dev), torch.ones(n, device=dev)
        good = torch.zeros(20, 1, dtype=torch.int64, device=dev), torch.zeros(20, 1, device=dev)
        for call in (lambda: shard.token_logprobs(h, labels), lambda: shard.distill(h, ids, top),
                     lambda: shard.distill(h, good[0], top), lambda: shard.distill(h, *good, one),
                     lambda: shard.distill(h, *good, None, one), lambda: shard.token_logprobs(h[:0], labels) if n else shard.distill(h, ids, top)):
            with pytest.raises(ValueError):
                call()
    with pytest.raises(ValueError):
        shard.token_logprobs(h, torch.zeros(20, 1, dtype=torch.int64, device=dev))


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_head_of_another_type(dev, dtype):
    """A head that is not bf16 has the other objectives too, as it has the cross entropy."""
    from micro_engram.train.head import VocabShard

    torch.manual_seed(0)
    W = torch.randn(203, 64).to(dtype)
    shard = VocabShard(W * 0.3, 0, 1, softcap=30.0, chunk_tokens=16, device=dev)
    h = torch.randn(21, 64, device=dev).to(dtype).requires_grad_()
    labels = torch.randint(0, 203, (21,), device=dev)
    labels[::4] = -100
    ce, _ = shard.loss_sum(h, labels)
    lp = shard.token_logprobs(h, labels)
    # the logits are one product of `dtype` in both; fp32 sums of up to 21 values of 10
    tol = 1e-3 if dtype == torch.float32 else 3e-2
    assert abs(float(ce.detach()) + float(lp.detach().sum())) < tol
    a, = torch.autograd.grad(ce, h)
    b, = torch.autograd.grad(-lp.sum(), h)
    assert torch.allclose(a, b, rtol=1e-2, atol=tol)
    values, ids, lse = shard.top_logits(h, 5)
    assert bool((values.diff(dim=1) <= 0).all())
    loss = shard.distill(h, ids, values, lse)
    assert float(loss.abs().max()) < tol  # the model is its own teacher
