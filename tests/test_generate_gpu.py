"""Generation with the native decoder on the sm_100a kernels: append, attention over the pages and sampling together, against the
same model in fp32 and beside its whole forward pass."""
import copy

import pytest
import torch

from micro_engram_fork_b200.models.generate import Generator
from test_generate import PROMPTS, small_model, whole_forward

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("page,chunk", [(16, 16), (64, 100)])
def test_extend_against_fp32(page, chunk):
    """Prompts in chunks, then single tokens: as near to the fp32 model (of the same bf16 weights) as the decoder's forward pass over
    whole sequences is, which rounds in more places."""
    model, eng = small_model("cuda", torch.bfloat16)
    eng = eng.to("cuda", torch.bfloat16)
    plain, plain_eng = small_model(engram=True)
    plain.load_state_dict({k: v.float().cpu() for k, v in model.state_dict().items()})
    plain_eng = copy.deepcopy(eng).float().cpu()
    long = [p + [(11 * i + 1) % 256 for i in range(15)] for p in PROMPTS]
    exact = [whole_forward(plain, plain_eng, p) for p in long]
    whole = [whole_forward(model, eng, p) for p in long]
    gen = Generator(model, 3, 100, chunk=chunk, page=page)  # (the engram is nested in layer 1 by now)
    assert model.model.layers[1].micro_engram is eng
    rest, got = [list(p) for p in PROMPTS], [[], [], []]
    steps = []
    while any(rest):
        steps.append([r[:chunk] for r in rest])
        rest = [r[chunk:] for r in rest]
    steps += [[[p[len(q) + i]] for p, q in zip(long, PROMPTS)] for i in range(15)]
    for now in steps:
        h, at = gen.extend(now), 0
        for b, n in enumerate(now):
            got[b].append(h[at:at + len(n)])
            at += len(n)
    for a, w, e in zip(got, whole, exact):
        scale = float(e.abs().max())
        a, w = torch.cat(a).float().cpu(), w.float().cpu()
        err, ref = float((a - e).square().mean().sqrt()), float((w - e).square().mean().sqrt())
        assert err <= 1.5 * ref + 2.0 ** -9 * scale, f"error {err:.3e}, the whole forward pass's {ref:.3e}"


def test_generate():
    """Answers repeat bit for bit, and sequences do not touch each other."""
    model, eng = small_model("cuda", torch.bfloat16)
    model.model.layers[1].add_module("micro_engram", eng.to("cuda", torch.bfloat16))
    gen = Generator(model, 3, 200, chunk=64, page=64)
    a = gen.generate(PROMPTS, 50, eos=-1)
    assert a == gen.generate(PROMPTS, 50, eos=-1) and all(len(x) == 50 for x in a)
    alone = Generator(model, 1, 200, chunk=64, page=64)
    h = [g.extend(n)[-1] for g, n in ((gen, [[], [], PROMPTS[2][:20]]), (alone, [PROMPTS[2][:20]])) for _ in [g.reset()]]
    assert float((h[0] - h[1]).abs().max()) <= 2.0 ** -6 * float(h[1].abs().max())
    drawn = gen.generate(PROMPTS, 30, temperature=1.0, top_p=0.9, eos=-1, generator=torch.Generator("cuda").manual_seed(2))
    assert drawn == gen.generate(PROMPTS, 30, temperature=1.0, top_p=0.9, eos=-1, generator=torch.Generator("cuda").manual_seed(2))
