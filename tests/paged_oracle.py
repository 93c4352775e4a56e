"""64-bit definitions of the paged cache's operators for their tests, written apart from micro_engram_fork_b200.ops.paged, a
batch to try them on, and how far results may be off; shared by the CPU and the GPU tests."""
import math
import random

import torch

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24, torch.float64: 2.0 ** -53}


class Batch:
    """Sequences (tokens in the cache before the call, new tokens) on pages in random order. Everything that no call may use is
    NaN: pages of no sequence, rows past a sequence's end, pages before every new token's window (which have no place in the table).
    before / after: tokens of no sequence at the batch's ends. together: keys and values as slices of one tensor."""

    def __init__(self, lens, hq, hk, d, page, window=None, dtype=torch.bfloat16, device="cpu", seed=0, before=0, after=0,
                 together=False, spare=2, index=torch.int32):
        r = random.Random(seed)
        g = torch.Generator().manual_seed(seed)
        self.lens, self.hq, self.hk, self.d, self.page, self.window = lens, hq, hk, d, page, window
        self.first = [max(0, c - window + 1) // page if window and n else 0 for c, n in lens]
        need = [-(-(c + n) // page) - a for (c, n), a in zip(lens, self.first)]
        width = max([a + n for a, n in zip(self.first, need)] + [1]) + 1
        pages = sum(need) + spare
        order = list(range(pages))
        r.shuffle(order)
        self.table = torch.full((len(lens), width), -1, dtype=index)
        self.k = torch.full((pages, hk, page, d), math.nan, dtype=dtype)
        self.v = torch.full((pages, hk, page, d), math.nan, dtype=dtype)
        at = 0
        for b, ((c, n), a) in enumerate(zip(lens, self.first)):
            for col in range(a, a + need[b]):
                p = order[at]
                at += 1
                self.table[b, col] = p
                rows = min(page, c + n - col * page)
                lo = max(0, c - window + 1 - col * page) if window and n else 0
                for t in (self.k, self.v):
                    t[p, :, lo:rows] = torch.randn(hk, rows - lo, d, generator=g).to(dtype)
        starts = [before]
        for _, n in lens:
            starts.append(starts[-1] + n)
        self.starts, self.tokens = starts, starts[-1] + after
        self.cu = torch.tensor(starts, dtype=index)
        self.seq_lens = torch.tensor([c + n for c, n in lens], dtype=index)
        self.q = (torch.randn(self.tokens, hq, d, generator=g) * (2.0 / math.sqrt(d))).to(dtype)
        if together:
            both = torch.stack([self.k, self.v], 1)
            self.k, self.v = both[:, 0], both[:, 1]
        if device != "cpu":
            if together:
                both = both.to(device)
                self.k, self.v = both[:, 0], both[:, 1]
            else:
                self.k, self.v = self.k.to(device), self.v.to(device)
            self.table, self.cu, self.seq_lens, self.q = (t.to(device) for t in (self.table, self.cu, self.seq_lens, self.q))

    def args(self):
        return self.k, self.v, self.table, self.cu, self.seq_lens

    def keys(self, b, cache):
        """[Hk, keys, D] of sequence b in fp64, from its first visible page on, and the position of the first."""
        c, n = self.lens[b]
        cols = range(self.first[b], -(-(c + n) // self.page))
        ids = [int(self.table[b, col]) for col in cols]
        rows = torch.cat([cache[i] for i in ids], 1) if ids else cache[0][:, :0]
        return rows[:, :c + n - self.first[b] * self.page].double(), self.first[b] * self.page


def attention(batch, scale=1.0):
    """(o, lse, spread of o, error of a score) in fp64: o may be off by its own rounding and a share of `spread`, the sum of
    p |v|; a score's sum of |q k| bounds what its 32-bit sum loses."""
    hq, hk, d = batch.hq, batch.hk, batch.d
    dev = batch.q.device
    o = torch.zeros(batch.tokens, hq, d, dtype=torch.float64, device=dev)
    spread = torch.zeros_like(o)
    lse = torch.full((hq, batch.tokens), -math.inf, dtype=torch.float64, device=dev)
    size = torch.zeros(hq, batch.tokens, dtype=torch.float64, device=dev)
    for b, (c, n) in enumerate(batch.lens):
        if n == 0:
            continue
        k, at = batch.keys(b, batch.k)
        v, _ = batch.keys(b, batch.v)
        s = batch.starts[b]
        for i in range(n):
            lo = max(0, c + i - batch.window + 1) if batch.window else 0
            kk, vv = k[:, lo - at:c + i + 1 - at], v[:, lo - at:c + i + 1 - at]
            qq = batch.q[s + i].double().view(hk, hq // hk, d)
            x = scale * torch.einsum("hgd,hkd->hgk", qq, kk)
            p = torch.softmax(x, -1)
            o[s + i] = torch.einsum("hgk,hkd->hgd", p, vv).reshape(hq, d)
            spread[s + i] = torch.einsum("hgk,hkd->hgd", p, vv.abs()).reshape(hq, d)
            lse[:, s + i] = torch.logsumexp(x, -1).reshape(hq)
            size[:, s + i] = abs(scale) * torch.einsum("hgd,hkd->hgk", qq.abs(), kk.abs()).amax(-1).reshape(hq)
    return o, lse, spread, size


def close_attention(got, want, d, single, dtype=torch.bfloat16):
    """o: half a step of its type, and of the terms p |v|: what p is rounded by (single tokens: two bf16 terms, 2^-17 in all; else one
    bf16, 2^-8), what the scores' errors make of p (twice: p and the sum), 2^-20 for exponentials and sums. A score of d products is
    added up in 32 bits in d / 16 steps and a few: each loses 2^-23 of the sum of |q k| at most."""
    o, lse = got
    want_o, want_lse, spread, size = want
    kernel = dtype == torch.bfloat16
    unit = 2.0 ** -23 if dtype != torch.float64 else 2.0 ** -50
    score = size * (d / 16 + 4 if kernel else d) * unit
    p = (2.0 ** -16 if single else 2.0 ** -8 * 1.01) if kernel else 0.0
    tol = HALF_STEP[dtype] * want_o.abs() * 1.01 + spread * (p + 2 * score.t()[..., None] + 8 * unit) + 1e-38
    bad = ~((o.double() - want_o).abs() <= tol)
    assert not bool(bad.any()), (f"{int(bad.sum())} of {bad.numel()} off, first at {bad.nonzero()[0].tolist()}: "
                                 f"{float(o[tuple(bad.nonzero()[0])])} for {float(want_o[tuple(bad.nonzero()[0])])}")
    none = want_lse == -math.inf
    assert bool((lse.double()[none] == -math.inf).all())
    err = (lse.double() - want_lse).abs()[~none]
    tol = (2 * score + 8 * unit * (1 + want_lse.abs()))[~none]
    assert bool((err <= tol).all()), f"lse off by {float((err - tol).max())} more than {float(tol.max())}"


def appended(batch, qkv, q_w, k_w, inv_freq, kv_shared, eps):
    """(q, k rows, v rows, slack of q, slack of k) in fp64 of the tokens in sequences: rows in token order [n, H, D], and
    {(sequence, position): token}. slack: |a| + |b| of what a rotated pair came from."""
    hq, hk, d = batch.hq, batch.hk, batch.d
    x = qkv.double().view(batch.tokens, -1, d)
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    where, pos = {}, torch.zeros(batch.tokens, dtype=torch.float64)
    for b, (c, n) in enumerate(batch.lens):
        for i in range(n):
            where[b, c + i] = batch.starts[b] + i
            pos[batch.starts[b] + i] = c + i
    angle = pos.to(x.device)[:, None, None] * inv_freq.double()

    def turned(y):
        a, b = y[..., :d // 2], y[..., d // 2:]
        c, s = torch.cos(angle), torch.sin(angle)
        size = (a.abs() + b.abs()).repeat(1, 1, 2)
        return torch.cat([a * c - b * s, a * s + b * c], -1), size

    q, q_size = turned(x[:, :hq] * q_w.double())
    k, k_size = turned(x[:, hq:hq + hk] * k_w.double())
    v = x[:, hq:] if kv_shared else x[:, hq + hk:]
    return q, k, v, q_size, k_size, where


def close_append(got, want, size, dtype=torch.bfloat16):
    """Half a step of the type, and of the pair's size what 32 bits lose: 2^-20 for norm, sine and products. In 64 bits (2^-46) the
    angle counts: here and there it is a product of up to 100001, rounded by 2^-53 of itself and by 2^-53 in its whole turns."""
    unit = 2.0 ** -20 if dtype != torch.float64 else 2.0 ** -46 + 4 * 100001 * 2.0 ** -53
    tol = HALF_STEP[dtype] * want.abs() * 1.01 + size * unit
    bad = ~((got.double() - want).abs() <= tol)
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, the worst by {float(((got.double() - want).abs() / tol).nan_to_num(1e9).max())} tolerances"


def attention_of_pages(batch, scale=1.0):
    """attention() of a batch whose table may have anything in it: what each token sees is worked out position by position from the table, the
    lengths and the window. Rows that see nothing: 0 and -inf."""
    hq, hk, d, page = batch.hq, batch.hk, batch.d, batch.page
    dev = batch.q.device
    o = torch.zeros(batch.tokens, hq, d, dtype=torch.float64, device=dev)
    spread = torch.zeros_like(o)
    lse = torch.full((hq, batch.tokens), -math.inf, dtype=torch.float64, device=dev)
    size = torch.zeros(hq, batch.tokens, dtype=torch.float64, device=dev)
    table, lengths = batch.table.tolist(), batch.seq_lens.tolist()
    for b, length in enumerate(lengths):
        s, n = batch.starts[b], batch.starts[b + 1] - batch.starts[b]
        lo = max(0, length - n - batch.window + 1) if batch.window else 0
        there = [p for p in range(lo, min(length, len(table[b]) * page)) if 0 <= table[b][p // page] < batch.k.shape[0]]
        if n == 0 or not there:
            continue
        ids = torch.tensor([table[b][p // page] for p in there], device=dev)
        row = torch.tensor([p % page for p in there], device=dev)
        pos = torch.tensor(there, device=dev)
        k, v = (t[ids, :, row].double().transpose(0, 1) for t in (batch.k, batch.v))  # [Hk, keys, D]
        for i in range(n):
            p = length - n + i
            seen = (pos <= p) & (pos > p - batch.window if batch.window else pos <= p)
            if not bool(seen.any()):
                continue
            kk, vv = k[:, seen], v[:, seen]
            qq = batch.q[s + i].double().view(hk, hq // hk, d)
            x = scale * torch.matmul(qq, kk.transpose(1, 2))
            w = torch.softmax(x, -1)
            o[s + i] = torch.matmul(w, vv).reshape(hq, d)
            spread[s + i] = torch.matmul(w, vv.abs()).reshape(hq, d)
            lse[:, s + i] = torch.logsumexp(x, -1).reshape(hq)
            size[:, s + i] = abs(scale) * torch.matmul(qq.abs(), kk.abs().transpose(1, 2)).amax(-1).reshape(hq)
    return o, lse, spread, size
