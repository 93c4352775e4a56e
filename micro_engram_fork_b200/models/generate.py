"""Generation with the framework's own decoder: a paged cache, prompts in chunks, one token a sequence after that.

    gen = Generator(model, sequences=8, max_len=4096)      # GemmaForCausalLM, with or without engrams in its layers
    answers = gen.generate([prompt_ids, ...], max_new_tokens=256, temperature=0.8, top_p=0.95)

`extend` is one step of it: new tokens of any of the sequences, packed, to the logits' hidden states. An engram that is nested in a
layer (`layer.micro_engram`, as attach_engram and the inference tool nest it) adds its memory after that layer, by the tokens that the
sequence has had (micro_engram/tools/infer.py does the same for an HF model's cache).

The cache (ops/paged.py) gives every sequence pages of its own. A sliding layer keeps its window and one chunk: its table goes round a ring of
pages. CUDA runs the sm_100a kernels, CPU the plain forms.
"""
import torch

from ..ops import paged
from ..ops.linear import linear
from ..ops.objectives import MAX_TOP, top_logits


def draw(p, top_p, u):
    """[rows, 1]: a rank for each row of falling probabilities p and uniform number u of [0, 1), among those that together have top_p."""
    p = torch.where(p.cumsum(1) - p < top_p, p, 0.0)
    upto = p.cumsum(1)
    last = ((p > 0).sum(1, keepdim=True) - 1).clamp_min(0)  # (a row of NaN: rank 0)
    # u times the last sum may round up to it, and behind the last kept rank the sums stay the same
    return (upto <= u * upto[:, -1:]).sum(1, keepdim=True).minimum(last)


class PagedCache:
    """Pages of all layers for `sequences` sequences of up to max_len tokens, extended by up to `chunk` tokens a call."""

    def __init__(self, config, sequences, max_len, chunk, page=64, device="cpu", dtype=torch.bfloat16):
        if sequences < 1 or max_len < 1 or chunk < 1 or page not in paged.PAGES:
            raise ValueError(f"sequences, max_len, chunk: positive numbers, page: one of {paged.PAGES}; got {sequences}, {max_len}, {chunk}, {page}")
        self.max_len, self.chunk, self.page = max_len, chunk, page
        width = -(-max_len // page)
        # a call's new tokens see window - 1 positions before the first of them
        ring = min(width, (config.sliding_window + chunk - 1 + page - 2) // page + 1)
        self.tables = {}
        for kind, pages in (("full_attention", width), ("sliding_attention", ring)):
            rows = torch.arange(sequences, dtype=torch.int32)[:, None] * pages + torch.arange(width, dtype=torch.int32)[None] % pages
            self.tables[kind] = rows.to(device)
        self.layers = []
        for i, kind in enumerate(config.layer_types):
            d, heads, _ = config.attn_shape(i)
            pages = sequences * (ring if config.layer_is_sliding(i) else width)
            both = torch.zeros(pages, 2, heads, page, d, dtype=dtype, device=device)
            self.layers.append((both[:, 0], both[:, 1], self.tables["sliding_attention" if config.layer_is_sliding(i) else "full_attention"]))

    def nbytes(self):
        return sum(2 * k.numel() * k.element_size() for k, _, _ in self.layers)


class Generator:
    """A model, its cache and the tokens of the sequences in it."""

    def __init__(self, model, sequences, max_len, chunk=1024, page=64):
        self.model, self.text = model, model.model
        w = self.text.embed_tokens.weight
        self.device, self.dtype = w.device, w.dtype
        self.cache = PagedCache(model.config, sequences, max_len, chunk, page, self.device, self.dtype)
        self.sequences = sequences
        self.tokens = torch.full((sequences, max_len), -1, dtype=torch.int64, device=self.device)  # what the cache holds
        self.lens = [0] * sequences
        self.engrams_on = True

    def reset(self, sequence=None):
        """Forget a sequence (or all of them)."""
        for b in range(self.sequences) if sequence is None else [sequence]:
            self.lens[b] = 0

    @torch.no_grad()
    def extend(self, new):
        """new: a list of token ids (possibly empty, at most `chunk`) for every sequence. Appends them and returns the
        final hidden states of all of them, packed [sum of lengths, hidden]."""
        if len(new) != self.sequences:
            raise ValueError(f"extend: a list of tokens for each of the {self.sequences} sequences is needed, got {len(new)}")
        counts = [len(n) for n in new]
        for b, n in enumerate(counts):
            if n > self.cache.chunk or self.lens[b] + n > self.cache.max_len:
                raise ValueError(f"extend: sequence {b} has {self.lens[b]} tokens and gets {n}; a call takes {self.cache.chunk}, the cache {self.cache.max_len}")
        vocab = self.text.embed_tokens.weight.shape[0]
        if any(not 0 <= t < vocab for n in new for t in n):
            raise ValueError(f"extend: token ids of 0 to {vocab - 1} are needed")
        ends = [a + n for a, n in zip(self.lens, counts)]
        starts = [0]
        for n in counts:
            starts.append(starts[-1] + n)
        if starts[-1] == 0:
            return torch.zeros(0, self.model.config.hidden_size, dtype=self.dtype, device=self.device)
        where = [(b, self.lens[b] + i) for b, n in enumerate(counts) for i in range(n)]
        host = torch.tensor([t for n in new for t in n] + [b for b, _ in where] + [p for _, p in where] + starts + ends)
        ids, seq, pos, cu, lens = host.to(self.device).split([starts[-1]] * 3 + [len(starts), len(ends)])
        self.tokens[seq, pos] = ids
        cu, lens = cu.int(), lens.int()
        x = self.text.embed_tokens.weight[ids]
        x = (x * torch.tensor(self.text.embed_scale, dtype=x.dtype)).to(x.dtype)
        for layer, (k, v, table) in zip(self.text.layers, self.cache.layers):
            x = layer.forward_cached(x, k, v, table, cu, lens, max(counts))
            engram = getattr(layer, "micro_engram", None)
            if engram is not None and self.engrams_on:
                x = engram.inject(x, engram.hash_prev(self._history(seq, pos, max(engram.orders)))).to(x.dtype)
        self.lens = ends
        return self.text.final_norm(x)

    def _history(self, seq, pos, reach):
        """[tokens, reach]: the token itself and those before it, -1 where there is none."""
        at = pos[:, None] - torch.arange(reach, device=pos.device)
        return torch.where(at >= 0, self.tokens[seq[:, None], at.clamp_min(0)], -1)

    @torch.no_grad()
    def next_tokens(self, hidden, temperature=0.0, top_p=1.0, top_k=0, generator=None):
        """A token for each row of final hidden states: the likeliest (temperature 0), or drawn from the likeliest ones that
        together have top_p of the probability, among at most top_k (0: MAX_TOP, the most that top_logits gives)."""
        z = linear(hidden.to(self.dtype), self.text.embed_tokens.weight)
        cap = self.model.config.final_logit_softcapping
        if temperature <= 0:
            return top_logits(z, 1, softcap=cap)[1][:, 0]
        if not top_p > 0 or top_k < 0:
            raise ValueError(f"top_p: a positive number, top_k: 0 or more; got {top_p} and {top_k}")
        k = min(top_k or MAX_TOP, MAX_TOP, z.shape[1])
        values, ids, lse = top_logits(z, k, softcap=cap, temperature=temperature)
        p = torch.exp(values / temperature - lse[:, None])
        return ids.gather(1, draw(p, top_p, torch.rand(p.shape[0], 1, device=p.device, generator=generator)))[:, 0]

    @torch.no_grad()
    def generate(self, prompts, max_new_tokens, temperature=0.0, top_p=1.0, top_k=0, eos=None, generator=None):
        """The answers to `prompts` (lists of token ids, one a sequence at most), each up to an `eos` token (an id or several,
        None: all that the model's configuration has) or max_new_tokens. What the sequences held before is forgotten."""
        if not prompts or len(prompts) > self.sequences or not all(len(p) for p in prompts):
            raise ValueError(f"generate: 1 to {self.sequences} prompts of at least a token are needed")
        longest = max(len(p) for p in prompts)
        if longest + max_new_tokens > self.cache.max_len + 1:  # (the last token is not extended by)
            raise ValueError(f"generate: a prompt of {longest} and {max_new_tokens} new tokens do not fit the cache's {self.cache.max_len}")
        eos = self.model.config.eos_token_id if eos is None else eos
        stop = set() if eos is None else set(eos) if isinstance(eos, (set, list, tuple)) else {eos}
        waits = paged.waits_out(self.device)
        self.reset()
        rest = [list(map(int, p)) for p in prompts] + [[]] * (self.sequences - len(prompts))
        last = [None] * len(prompts)  # final hidden state of a prompt's last token
        chunk = self.cache.chunk
        while any(rest):
            now = [r[:chunk] for r in rest]
            hidden = self.extend(now)
            end = 0
            for b, n in enumerate(now):
                end += len(n)
                if n and len(n) == len(rest[b]):
                    last[b] = hidden[end - 1]
            rest = [r[chunk:] for r in rest]
        answers = [[] for _ in prompts]
        live = list(range(len(prompts)))
        hidden = torch.stack(last)
        for step in range(max_new_tokens):
            drawn = self.next_tokens(hidden, temperature, top_p, top_k, generator).tolist()
            new = [[] for _ in range(self.sequences)]
            for b, t in zip(live, drawn):
                answers[b].append(t)
                if t not in stop:
                    new[b] = [t]
            live = [b for b in live if new[b]]
            if not live or step + 1 == max_new_tokens:
                break
            hidden = self.extend(new)
        paged.check_waits(self.device, waits)
        return answers
