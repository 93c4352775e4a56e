"""Generation with the native decoder on its paged cache, on CPU: the same hidden states and answers as whole forward passes."""
import json
import math

import pytest
import torch

from micro_engram.module import MicroEngram, attach_engram
from micro_engram_fork_b200.models import gemma as G
from micro_engram_fork_b200.models.generate import Generator


def small_model(device="cpu", dtype=torch.float32, engram=True, seed=0, **kw):
    cfg = G.tiny_config(vocab_size=256, hidden_size=128, intermediate_size=256, sliding_window=20, **kw)
    model = G.GemmaForCausalLM(cfg).to(device)
    G.cast_projections_(model, dtype)
    G.init_random_(model, seed=seed, std=0.08)
    g = torch.Generator().manual_seed(seed)
    for layer in model.model.layers:  # scores as trained norm weights leave them
        layer.self_attn.q_norm.weight.copy_(0.3 + 0.1 * torch.rand(layer.head_dim, generator=g))
        layer.self_attn.k_norm.weight.copy_(0.3 + 0.1 * torch.rand(layer.head_dim, generator=g))
        layer.layer_scalar.fill_(0.8)
    eng = None
    if engram:
        eng = MicroEngram(model_dim=128, vocab_size=256, table_size=97, engram_dim=16, num_heads=2, gate="scalar_sqrt", seed=3)
        with torch.no_grad():
            for p in eng.parameters():
                p.copy_(torch.randn(p.shape, generator=g) * 0.2)
        eng.eval()
    return model, eng


def whole_forward(model, eng, ids, layer=1):
    """Final hidden states of one sequence by the decoder's forward pass over all of it, the engram by its hook."""
    ids = torch.tensor([ids], device=model.model.embed_tokens.weight.device)
    handles = []
    if eng is not None:
        _, handles = attach_engram(model, eng, layer, get_ids=lambda: (ids, None))
    w = model.model.embed_tokens.weight
    x = (w[ids[0]] * torch.tensor(model.model.embed_scale, dtype=w.dtype)).to(w.dtype)
    with torch.no_grad():
        h = model.model(x, torch.arange(ids.shape[1], device=x.device))
    for handle in handles:
        handle.remove()
    return h


PROMPTS = [[(7 * i * i + 3) % 256 for i in range(n)] for n in (70, 1, 33)]


@pytest.mark.parametrize("engram", [False, True])
@pytest.mark.parametrize("chunk", [16, 100])
def test_extend_matches_whole_forward(chunk, engram):
    model, eng = small_model(engram=engram)
    want = [whole_forward(model, eng, p) for p in PROMPTS]
    gen = Generator(model, 3, 90, chunk=chunk, page=16)
    rest, got = [list(p) for p in PROMPTS], [[], [], []]
    while any(rest):
        now = [r[:chunk - 3 * b] for b, r in enumerate(rest)]
        h, at = gen.extend(now), 0
        for b, n in enumerate(now):
            got[b].append(h[at:at + len(n)])
            at += len(n)
        rest = [r[len(n):] for r, n in zip(rest, now)]
    for a, b in zip(got, want):
        a = torch.cat(a)
        assert float((a - b).abs().max()) <= 1e-4 * float(b.abs().max())
    assert gen.lens == [70, 1, 33]


def test_generate_matches_whole_forward():
    """Greedy answers, token by token, past the window and round the sliding layers' rings."""
    model, eng = small_model()
    model.config.eos_token_id = None
    model.model.layers[1].add_module("micro_engram", eng)
    gen = Generator(model, 4, 120, chunk=16, page=16)
    answers = gen.generate(PROMPTS, 40)
    del model.model.layers[1].micro_engram
    cap = model.config.final_logit_softcapping
    for prompt, answer in zip(PROMPTS, answers):
        assert len(answer) == 40
        h = whole_forward(model, eng, prompt + answer)
        if hasattr(model.model.layers[1], "micro_engram"):
            del model.model.layers[1].micro_engram
        z = (h @ model.model.embed_tokens.weight.t()).double()
        z = cap * torch.tanh(z / cap)
        for i, t in enumerate(answer):  # the likeliest, up to what the two ways differ by
            row = z[len(prompt) - 1 + i]
            assert float(row.max() - row[t]) <= 1e-3


def test_generate_stops_and_samples():
    model, _ = small_model(engram=False)
    gen = Generator(model, 2, 100, chunk=32, page=16)
    first = gen.generate(PROMPTS[:2], 20, eos=-1)
    stop = first[0][3]
    cut = gen.generate(PROMPTS[:2], 20, eos=stop)
    assert cut[0] == first[0][:first[0].index(stop) + 1]
    g = lambda: torch.Generator().manual_seed(5)  # noqa: E731
    a = gen.generate(PROMPTS[:2], 20, temperature=1.5, top_p=0.9, eos=-1, generator=g())
    assert a == gen.generate(PROMPTS[:2], 20, temperature=1.5, top_p=0.9, eos=-1, generator=g())
    assert gen.generate(PROMPTS[:2], 20, temperature=1.5, top_p=1e-9, eos=-1, generator=g()) == first
    assert gen.generate(PROMPTS[:2], 20, temperature=1.5, top_k=1, eos=-1, generator=g()) == first


def test_sampling_follows_the_probabilities():
    model, _ = small_model(engram=False)
    gen = Generator(model, 1, 20, chunk=16, page=16)
    h = gen.extend([[5, 9, 11]])[-1:]
    z = (h @ model.model.embed_tokens.weight.t()).double()[0]
    cap = model.config.final_logit_softcapping
    p = torch.softmax(cap * torch.tanh(z / cap) / 0.7, 0)
    order = p.sort(descending=True)
    keep = order.values.cumsum(0) - order.values < 0.8
    want = torch.zeros(256, dtype=torch.float64)
    want[order.indices[keep]] = order.values[keep] / order.values[keep].sum()
    n = 20000
    drawn = gen.next_tokens(h.expand(n, -1), 0.7, 0.8, generator=torch.Generator().manual_seed(1))
    got = torch.bincount(drawn, minlength=256).double() / n
    assert float((got - want).abs().max()) <= 5 * math.sqrt(0.25 / n) and bool((got[want == 0] == 0).all())


def test_refusals():
    model, _ = small_model(engram=False)
    with pytest.raises(ValueError):
        Generator(model, 0, 10)
    with pytest.raises(ValueError):
        Generator(model, 1, 10, page=24)
    gen = Generator(model, 2, 40, chunk=16, page=16)
    for call in (lambda: gen.extend([[1]]), lambda: gen.extend([[1] * 17, []]), lambda: gen.generate([], 3), lambda: gen.generate([[1], []], 3),
                 lambda: gen.generate([[1]] * 3, 3), lambda: gen.generate([[1] * 30], 12)):
        with pytest.raises(ValueError):
            call()
    gen.extend([[1] * 16, []])
    gen.extend([[1] * 16, []])
    with pytest.raises(ValueError):
        gen.extend([[1] * 9, []])
    assert gen.extend([[], []]).shape == (0, 128)


def test_sliding_layers_keep_a_ring():
    model, _ = small_model(engram=False)
    gen = Generator(model, 2, 2000, chunk=16, page=16)
    full, ring = gen.cache.layers[3][0].shape[0], gen.cache.layers[0][0].shape[0]
    assert full == 2 * 125 and ring == 2 * 4  # 20 + 16 - 1 positions lie in 4 pages at most


def test_infer_native(tmp_path, monkeypatch, capsys):
    """The inference tool's --native path: folder -> decoder, engram, cache -> text."""
    from safetensors.torch import save_file

    from micro_engram.tools import infer

    model, eng = small_model()
    conf = model.config.to_dict()
    conf.update({"model_type": "gemma4_text", "eos_token_id": None})
    (tmp_path / "config.json").write_text(json.dumps(conf))
    save_file({k: v.clone().contiguous() for k, v in model.state_dict().items()}, str(tmp_path / "model.safetensors"))
    torch.save(eng.state_dict(), tmp_path / "engram.pt")

    class Tok:
        def __call__(self, text, return_tensors=None):
            return type("E", (), {"input_ids": torch.tensor([[ord(c) for c in text]])})

        def decode(self, ids, skip_special_tokens=False):
            return " ".join(map(str, ids))

    import transformers

    monkeypatch.setattr(transformers.AutoTokenizer, "from_pretrained", lambda *a, **k: Tok())
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    args = ["--model", str(tmp_path), "--engram-pt", str(tmp_path / "engram.pt"), "--layer", "1", "--heads", "2", "--prompt", "hello",
            "--max-new-tokens", "6", "--temperature", "0", "--native", "--max-len", "64"]
    from unittest import mock

    with mock.patch.dict(infer.DEFAULTS, {"seed": 3}):
        infer.main(args)
        with_engram = capsys.readouterr().out.rsplit("--- output ---\n", 1)[1].split()
        infer.main([*args, "--no-engram"])
        without = capsys.readouterr().out.rsplit("--- output ---\n", 1)[1].split()
        with pytest.raises(SystemExit):
            infer.main([*args[:-1], "3"])
    model.config.eos_token_id = None
    gen = Generator(model, 1, 64)
    assert list(map(str, gen.generate([[ord(c) for c in "hello"]], 6)[0])) == without
    model.model.layers[1].add_module("micro_engram", eng)
    assert list(map(str, gen.generate([[ord(c) for c in "hello"]], 6)[0])) == with_engram


def test_wrong_tokens_and_sampling():
    model, _ = small_model(engram=False)
    gen = Generator(model, 2, 40, chunk=16, page=16)
    for ids in ([256], [-1], [3, 10 ** 12]):
        with pytest.raises(ValueError):
            gen.extend([[1], ids])
        with pytest.raises(ValueError):
            gen.generate([ids], 3)
    assert gen.lens == [0, 0]
    h = gen.extend([[1], [2, 3]])
    for kw in ({"top_p": 0.0}, {"top_p": -1.0}, {"top_p": math.nan}, {"top_k": -1}):
        with pytest.raises(ValueError):
            gen.next_tokens(h, temperature=1.0, **kw)
    likeliest = gen.next_tokens(h)
    assert torch.equal(gen.next_tokens(h, temperature=1.0, top_p=1e-6), likeliest)
    assert torch.equal(gen.next_tokens(h, temperature=1.0, top_k=1), likeliest)


def test_every_end_token_ends_an_answer(tmp_path, monkeypatch, capsys):
    """Models with several end tokens: config.json's own, those beside its text_config, those of generation_config.json."""
    from safetensors.torch import save_file

    from micro_engram.tools import infer

    assert G.GemmaConfig.from_dict({"eos_token_id": [1, 106]}).eos_token_id == [1, 106]
    assert G.GemmaConfig.from_dict({"text_config": {"eos_token_id": 1}, "eos_token_id": [1, 106]}).eos_token_id == [1, 106]
    assert G.GemmaConfig.from_dict({"text_config": {"hidden_size": 64}, "eos_token_id": [106, 7]}).eos_token_id == [106, 7]
    for same, ids in ((1, {"eos_token_id": 1}), (1, {"eos_token_id": [1]}), (1, {}), (None, {"eos_token_id": None}), (None, {"eos_token_id": []}),
                      (1, {"text_config": {"eos_token_id": 1}, "eos_token_id": None}), (1, {"text_config": {}, "eos_token_id": None}), (0, {"eos_token_id": [0, 0]})):
        assert G.GemmaConfig.from_dict(ids).eos_token_id == same
    model, _ = small_model(engram=False)
    model.config.eos_token_id = None
    gen = Generator(model, 1, 64)
    answer = gen.generate([[5, 9, 11]], 20)[0]
    stop, want = answer[0], answer[:1]
    assert len(answer) == 20
    never = next(t for t in range(256) if t not in answer)
    model.config.eos_token_id = [never, stop]
    assert gen.generate([[5, 9, 11]], 20)[0] == want

    class Tok:
        def __call__(self, text, return_tensors=None):
            return type("E", (), {"input_ids": torch.tensor([[5, 9, 11]])})

        def decode(self, ids, skip_special_tokens=False):
            return " ".join(map(str, ids))

    import transformers

    monkeypatch.setattr(transformers.AutoTokenizer, "from_pretrained", lambda *a, **k: Tok())
    monkeypatch.setattr(torch.cuda, "is_available", lambda: False)
    monkeypatch.setattr(infer, "plan_engrams", lambda args: [])
    save_file({k: v.clone().contiguous() for k, v in model.state_dict().items()}, str(tmp_path / "model.safetensors"))
    text = {**model.config.to_dict(), "eos_token_id": never}
    places = [({**text, "eos_token_id": [never, stop]}, None), ({"text_config": text, "eos_token_id": [never, stop]}, None),
              (text, {"eos_token_id": [never, stop]}), (text, {"eos_token_id": stop})]
    for conf, generation in places:
        (tmp_path / "config.json").write_text(json.dumps({**conf, "model_type": "gemma4_text"}))
        (tmp_path / "generation_config.json").write_text(json.dumps(generation or {}))
        infer.main(["--model", str(tmp_path), "--prompt", "x", "--max-new-tokens", "20", "--temperature", "0", "--native", "--max-len", "64"])
        assert list(map(int, capsys.readouterr().out.rsplit("--- output ---\n", 1)[1].split())) == want


@pytest.mark.parametrize("top_p", [0.5, 0.9, 1.0])
def test_draws_stay_among_the_kept(top_p):
    """The smallest and the largest number that torch.rand gives draw a token that top_p has kept, of any row."""
    from micro_engram_fork_b200.models.generate import draw

    g = torch.Generator().manual_seed(0)
    p = torch.softmax(2 * torch.randn(4000, 256, generator=g), 1).sort(1, descending=True).values
    kept = p.cumsum(1) - p < top_p
    rows = torch.arange(4000)
    for u in (0.0, 1 - 2.0 ** -24):
        rank = draw(p, top_p, torch.full((4000, 1), u))[:, 0]
        assert bool(kept[rows, rank].all()) and bool((p[rows, rank] > 0).all())
    assert bool((draw(p, top_p, torch.zeros(4000, 1)) == 0).all())
    # a certain token and columns of nothing behind it
    p = torch.tensor([[1.0, 0.0, 0.0]]).expand(2, 3)
    assert draw(p, top_p, torch.tensor([[0.0], [1 - 2.0 ** -24]])).tolist() == [[0], [0]]
    assert draw(torch.full((1, 5), math.nan), top_p, torch.tensor([[0.5]])).tolist() == [[0]]  # (an index that exists)


def test_generate_raises_for_its_own_waits(monkeypatch):
    """Waits that ran out before a call, or that another caller has looked at, change nothing; those within it raise."""
    from micro_engram_fork_b200.ops import paged

    model, _ = small_model(engram=False)
    gen = Generator(model, 1, 64)
    state = {"count": 4, "new": 0}

    def waits(device):
        state["count"] += state["new"]
        return state["count"], 71

    monkeypatch.setattr(paged, "_waits", waits)
    answer = gen.generate([[5, 9]], 3, eos=-1)
    state["new"] = 1
    with pytest.raises(RuntimeError, match="ran out"):
        gen.generate([[5, 9]], 3, eos=-1)
    state["new"] = 0
    assert gen.generate([[5, 9]], 3, eos=-1) == answer


@pytest.mark.parametrize("text", ["", "{", "[1, 106]"])
def test_a_generation_config_that_cannot_be_read(tmp_path, text):
    """A folder that trains is not refused for it."""
    (tmp_path / "config.json").write_text(json.dumps({"hidden_size": 64, "eos_token_id": 7}))
    (tmp_path / "generation_config.json").write_text(text)
    with pytest.warns(UserWarning, match="generation_config"):
        assert G.GemmaConfig.from_pretrained(str(tmp_path)).eos_token_id == 7
