"""The paged cache's operators on CPU: the plain forms against the 64-bit definitions, edge rules, refusals."""
import math

import pytest
import torch

import paged_oracle as oracle
from micro_engram_fork_b200.ops import paged

F32, F64 = torch.float32, torch.float64


def append_inputs(batch, kv_shared, dtype, seed=1):
    g = torch.Generator().manual_seed(seed)
    heads = batch.hq + (1 if kv_shared else 2) * batch.hk
    dev = batch.q.device
    qkv = (torch.randn(batch.tokens, heads * batch.d, generator=g) * 1.5).to(dtype).to(dev)
    w = (1 + 0.2 * torch.randn(2, batch.d, generator=g)).to(dev)
    inv_freq = (10000.0 ** (-torch.arange(0, batch.d, 2).float() / batch.d)).to(dev)
    return qkv, w[0], w[1], inv_freq


def check_append(batch, kv_shared, dtype, call, eps=1e-6):
    """Appends to the batch's cache and looks at every row of it."""
    qkv, q_w, k_w, inv_freq = append_inputs(batch, kv_shared, dtype)
    before_k, before_v = batch.k.clone(), batch.v.clone()
    q = call(qkv, q_w, k_w, inv_freq, batch.k, batch.v, batch.table, batch.cu, batch.seq_lens, batch.hq, kv_shared, eps)
    want_q, want_k, want_v, q_size, k_size, where = oracle.appended(batch, qkv, q_w, k_w, inv_freq, kv_shared, eps)
    mine = torch.zeros(batch.tokens, dtype=torch.bool)
    mine[list(where.values())] = True
    oracle.close_append(q[mine], want_q[mine], q_size[mine], dtype)
    assert bool((q[~mine] == 0).all())
    for (b, pos), t in where.items():
        page, row = int(batch.table[b, pos // batch.page]), pos % batch.page
        oracle.close_append(batch.k[page, :, row], want_k[t], k_size[t], dtype)
        oracle.close_append(batch.v[page, :, row], want_v[t], want_v[t].abs(), dtype)
        before_k[page, :, row], before_v[page, :, row] = batch.k[page, :, row], batch.v[page, :, row]
    # nothing else was touched (NaN rows included)
    as_int = torch.int64 if dtype == F64 else torch.int32 if dtype == F32 else torch.int16
    for now, was in ((batch.k, before_k), (batch.v, before_v)):
        assert torch.equal(now.contiguous().view(as_int), was.contiguous().view(as_int))


@pytest.mark.parametrize("dtype", [F32, F64])
@pytest.mark.parametrize("lens,window", [([(0, 1)], None), ([(5, 3), (0, 17), (40, 0), (31, 1)], None), ([(70, 9), (3, 30)], 20)])
def test_attention(lens, window, dtype):
    batch = oracle.Batch(lens, 6, 2, 64, 16, window, dtype, before=1, after=2)
    got = paged.paged_attention(batch.q, *batch.args(), window=window, scale=0.7)
    oracle.close_attention(got, oracle.attention(batch, 0.7), 64, False, dtype)
    assert bool((got[0][0] == 0).all()) and bool((got[0][-2:] == 0).all()) and bool((got[1][:, -2:] == -math.inf).all())


@pytest.mark.parametrize("kv_shared", [False, True])
@pytest.mark.parametrize("dtype", [F32, F64])
def test_append(dtype, kv_shared):
    batch = oracle.Batch([(5, 3), (0, 17), (40, 0), (100000, 2)], 3, 1, 64, 16, None, dtype, before=2, after=1)
    check_append(batch, kv_shared, dtype, paged.qkv_norm_rope_append)


def bad_pages(device, dtype):
    """A batch one of whose sequences has numbers that are no pages, another a length past its table's row: (batch,
    the same with those keys left out as a list of visible keys for each sequence)."""
    batch = oracle.Batch([(60, 2), (33, 1), (10, 1)], 4, 2, 64, 16, None, dtype, device)
    batch.table[0, 1] = batch.k.shape[0]
    batch.table[0, 2] = -7
    batch.seq_lens[2] = 16 * batch.table.shape[1] + 5  # its row ends: the new token has no place, and sees what there is
    batch.table[2] = batch.table[1]                    # (pages that hold numbers: all but the last are whole)
    batch.table[2, 2:] = -1
    return batch


def check_bad_pages(device, dtype, single):
    batch = bad_pages(device, dtype)
    o, lse = paged.paged_attention(batch.q, *batch.args())
    assert bool(o.isfinite().all()) and bool(lse.isfinite().all())
    seen = {0: [0, 3], 1: [0, 1, 2], 2: [0, 1]}
    for b, (first, count, length) in enumerate([(0, 2, 62), (2, 1, 34), (3, 1, 32)]):
        ids = [int(batch.table[b, col]) for col in seen[b]]
        key = torch.cat([torch.arange(16 * c, 16 * c + 16) for c in seen[b]]).to(device)
        for i in range(count):
            pos = length - count + i
            ok = key <= pos if b < 2 else key < 32
            k = torch.cat([batch.k[p] for p in ids], 1)[:, ok].double()
            v = torch.cat([batch.v[p] for p in ids], 1)[:, ok].double()
            x = torch.einsum("hgd,hkd->hgk", batch.q[first + i].double().view(2, 2, 64), k)
            want = torch.einsum("hgk,hkd->hgd", torch.softmax(x, -1), v).reshape(4, 64)
            assert float((o[first + i].double() - want).abs().max()) < 2.0 ** -7 * float(v.abs().max())
            assert float((lse[:, first + i].double() - torch.logsumexp(x, -1).reshape(4)).abs().max()) < 1e-4
    # appending there stores nothing but in pages
    batch = bad_pages(device, dtype)
    batch.seq_lens[1] = 0  # one new token, none in all: its position is negative
    k, v = batch.k.clone(), batch.v.clone()
    q = paged.qkv_norm_rope_append(*append_inputs(batch, False, dtype), *batch.args(), 4)
    assert bool((q[2] == 0).all()) and bool((q[[0, 1, 3]] != 0).any(-1).all())
    page = int(batch.table[0, 3])
    k[page, :, 12:14], v[page, :, 12:14] = batch.k[page, :, 12:14], batch.v[page, :, 12:14]
    assert torch.equal(k.nan_to_num(7.0), batch.k.nan_to_num(7.0)) and torch.equal(v.nan_to_num(7.0), batch.v.nan_to_num(7.0))
    assert bool(batch.k[page, :, 12:14].isfinite().all())
    o, lse = paged.paged_attention(batch.q, *batch.args())
    assert bool((o[2] == 0).all()) and bool((lse[:, 2] == -math.inf).all())


def test_bad_pages():
    check_bad_pages("cpu", F32, False)


def check_bad_offsets(device, dtype):
    """cu_seqlens that leave the batch are taken within it."""
    batch = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, dtype, device)
    want = paged.paged_attention(batch.q, *batch.args())
    batch.cu[0], batch.cu[2] = -5, 1000
    got = paged.paged_attention(batch.q[:, :], *batch.args())
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    batch.cu[1] = 900  # the first sequence takes all five tokens, the second none
    o, lse = paged.paged_attention(batch.q, *batch.args())
    assert o.shape == batch.q.shape and bool(o.isfinite().all())
    batch.cu[:] = torch.tensor([4, 3, 2])
    o, lse = paged.paged_attention(batch.q, *batch.args())
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())


def test_bad_offsets():
    check_bad_offsets("cpu", F32)


def refusals(device, dtype):
    """(error, call) for every argument that is refused alike on CPU and GPU."""
    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, dtype, device)
    k, v, table, cu, lens = b.args()
    qkv, q_w, k_w, f = append_inputs(b, False, dtype)
    att = lambda *a, **kw: lambda: paged.paged_attention(*a, **kw)  # noqa: E731
    app = lambda *a, **kw: lambda: paged.qkv_norm_rope_append(*a, **kw)  # noqa: E731
    odd = k[:, :, :12].contiguous()
    calls = [
        att(b.q, k, v[:1], table, cu, lens), att(b.q, k[0], v[0], table, cu, lens), att(b.q, odd, odd, table, cu, lens),
        att(b.q, k[..., :32].contiguous(), v[..., :32].contiguous(), table, cu, lens), att(b.q, k, v, table[:1], cu, lens),
        att(b.q, k, v, table[0], cu, lens), att(b.q, k, v, table, cu[:2], lens), att(b.q, k, v, table, cu, lens.float()),
        att(b.q, k, v, table.float(), cu, lens), att(b.q[:, :3], k, v, table, cu, lens), att(b.q[..., :32], k, v, table, cu, lens),
        att(b.q[0], k, v, table, cu, lens), att(b.q, k, v, table, cu, lens, window=0), att(b.q, k, v, table, cu, lens, window=-3),
        att(b.q, k, v, table, cu, lens, max_q=0), att(b.q, k, v, table, cu, lens, scale=math.nan),
        att(b.q, k, v, table, cu, lens, scale=math.inf), att(b.q, k, v, table, cu, lens, scale=0.0), att(b.q, k, v, table, cu, lens, scale=-1.0), att(b.q, k, v, table, cu, lens, out=b.q[:2].clone()),
        att(b.q.clone().requires_grad_(), k, v, table, cu, lens), att(b.q, k[:0], v[:0], table, cu, lens),
        app(qkv, q_w, k_w, f, k, v, table, cu, lens, 5), app(qkv, q_w, k_w, f, k, v, table, cu, lens, 4, True),
        app(qkv, q_w, k_w, f, k, v, table, cu, lens, 0), app(qkv[0], q_w, k_w, f, k, v, table, cu, lens, 4),
        app(qkv, q_w[:32], k_w, f, k, v, table, cu, lens, 4), app(qkv, q_w, k_w[None], f, k, v, table, cu, lens, 4),
        app(qkv, q_w, k_w, q_w, k, v, table, cu, lens, 4), app(qkv, q_w, k_w, f, k, v[1:], table, cu, lens, 4),
        app(qkv, q_w.clone().requires_grad_(), k_w, f, k, v, table, cu, lens, 4), app(qkv, q_w, k_w, f, k, v, table, cu[1:], lens, 4),
    ]
    return [(ValueError, c) for c in calls]


def test_refusals():
    for i, (error, call) in enumerate(refusals("cpu", F32)):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was taken")


def test_empty():
    b = oracle.Batch([(20, 0), (9, 0)], 4, 2, 64, 16, None, F32)
    o, lse = paged.paged_attention(b.q, *b.args())
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)
    none = torch.zeros(0, dtype=torch.int32)
    o, lse = paged.paged_attention(torch.ones(3, 4, 64), b.k, b.v, b.table[:0], torch.zeros(1, dtype=torch.int32), none)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    qkv, q_w, k_w, f = append_inputs(b, False, F32)
    assert paged.qkv_norm_rope_append(qkv, q_w, k_w, f, *b.args(), 4).shape == (0, 4, 64)


def test_out():
    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, F32, before=1, after=2)
    want, _ = paged.paged_attention(b.q, *b.args())
    out = torch.full_like(b.q, 9.0)
    got, lse = paged.paged_attention(b.q, *b.args(), out=out)
    assert got is out and torch.equal(out[1:-2], want[1:-2]) and bool((out[0] == 9).all()) and bool((out[-2:] == 9).all())


def test_together():
    """Appending a prompt in pieces and attending gives what the whole prompt gives at once."""
    from micro_engram_fork_b200.ops.attention import attention_ref
    from micro_engram_fork_b200.ops import norm as N

    g = torch.Generator().manual_seed(0)
    hq, hk, d, T = 4, 2, 64, 50
    qkv = torch.randn(T, (hq + 2 * hk) * d, generator=g)
    q_w, k_w = 1 + 0.1 * torch.randn(2, d, generator=g)
    f = 10000.0 ** (-torch.arange(0, d, 2).float() / d)
    cos, sin = N.rope_cos_sin(torch.arange(T), f, F32)
    x = qkv.view(T, -1, d)
    q = N.rope_ref(N.rmsnorm_ref(x[:, :hq], q_w), cos[:, None], sin[:, None])
    k = N.rope_ref(N.rmsnorm_ref(x[:, hq:hq + hk], k_w), cos[:, None], sin[:, None])
    want, _ = attention_ref(q, k, N.rmsnorm_ref(x[:, hq + hk:]), torch.zeros(T), 20, 0.3)
    kp, vp = torch.full((2, 5, hk, 16, d), math.nan)
    table = torch.tensor([[3, 0, 4, 1]], dtype=torch.int32)
    parts, at = [], 0
    for n in (7, 1, 30, 1, 11):
        cu, lens = torch.tensor([0, n]), torch.tensor([at + n])
        rows = paged.qkv_norm_rope_append(qkv[at:at + n], q_w, k_w, f, kp, vp, table, cu, lens, hq)
        parts.append(paged.paged_attention(rows, kp, vp, table, cu, lens, window=20, scale=0.3)[0])
        at += n
    assert float((torch.cat(parts) - want).abs().max()) < 1e-5


def alias_refusals(device, dtype):
    """`out` in q's memory: units of work read q after others have written."""
    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, dtype, device)
    two = torch.zeros(b.tokens, 8, 64, dtype=dtype, device=device)
    odd = torch.zeros(b.tokens, 4, 66, dtype=dtype, device=device)[..., :64]  # (q is copied first)
    return [lambda: paged.paged_attention(b.q, *b.args(), out=b.q), lambda: paged.paged_attention(two[:, :4], *b.args(), out=two[:, 2:6]),
            lambda: paged.paged_attention(odd, *b.args(), out=odd)]


def test_out_is_not_q():
    for call in alias_refusals("cpu", F32):
        with pytest.raises(ValueError):
            call()


def check_wide_numbers(device, dtype):
    """64-bit page numbers that would be pages if they were cut to 32 bits are none."""
    batch = oracle.Batch([(60, 2), (33, 1)], 4, 2, 64, 16, None, dtype, device)
    table = batch.table.long()
    table[0, 1] = -1
    want = paged.paged_attention(batch.q, batch.k, batch.v, table, batch.cu, batch.seq_lens)
    for wrong in (2 ** 32, -2 ** 32, 2 ** 63 - 1, -2 ** 63):
        table[0, 1] = wrong + int(batch.table[0, 1]) if abs(wrong) == 2 ** 32 else wrong
        got = paged.paged_attention(batch.q, batch.k, batch.v, table, batch.cu.long(), batch.seq_lens.long())
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_wide_numbers():
    check_wide_numbers("cpu", F32)


def check_negative_positions(device, dtype):
    """Tokens at negative positions before others, under windows of any size: those see nothing, the others what they would alone."""
    for count, max_q in ((6, None), (6, 1), (40, None)):
        batch = oracle.Batch([(0, count), (20, 3)], 4, 2, 64, 16, None, dtype, device)
        batch.seq_lens[0] = 2  # its last two tokens have positions 0 and 1
        want = paged.paged_attention(batch.q, *batch.args(), max_q=max_q)
        assert bool((want[0][:count - 2] == 0).all()) and bool((want[1][:, count - 2:] > -math.inf).all())
        for window in (2 ** 31 - 1, 2 ** 31 - 3, 1000):  # no key lies that far back
            got = paged.paged_attention(batch.q, *batch.args(), window=window, max_q=max_q)
            assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_negative_positions():
    check_negative_positions("cpu", F32)


def more_refusals(device, dtype):
    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, dtype, device)
    qkv, q_w, k_w, f = append_inputs(b, False, dtype)
    return [lambda: paged.paged_attention(b.q, *b.args(), scale=1e-60), lambda: paged.paged_attention(b.q, *b.args(), scale=1e60),
            lambda: paged.paged_attention(b.q, *b.args(), out=torch.zeros_like(b.q).requires_grad_()),
            lambda: paged.qkv_norm_rope_append(qkv, q_w, k_w, f.clone().requires_grad_(), *b.args(), 4)]


def test_more_refusals():
    for call in more_refusals("cpu", F32):
        with pytest.raises(ValueError):
            call()


def test_a_wait_that_ran_out(monkeypatch):
    class Native:
        words = [(7, 71), (0, 0)]

        def paged_status(self, device):
            assert device == 3
            return self.words.pop(0)

    fake = Native()
    monkeypatch.setattr(paged, "native", lambda: fake)
    paged.check_waits("cpu")
    with pytest.raises(RuntimeError, match="ran out"):
        paged.check_waits("cuda:3")
    paged.check_waits("cuda:3")


def check_lse_of_padding(device, dtype, lens, max_q):
    """Tokens of no sequence have a log-sum-exp of -inf whether or not the rows' place is the caller's."""
    batch = oracle.Batch(lens, 4, 2, 64, 16, None, dtype, device, before=2, after=5)
    want, want_lse = paged.paged_attention(batch.q, *batch.args(), max_q=max_q)
    out = torch.full_like(batch.q, 9.0)
    free = [torch.full_like(want_lse, math.nan) for _ in range(8)]  # what a new tensor may lie on
    del free
    got, lse = paged.paged_attention(batch.q, *batch.args(), max_q=max_q, out=out)
    assert torch.equal(lse, want_lse) and bool((lse[:, :2] == -math.inf).all()) and bool((lse[:, -5:] == -math.inf).all())
    assert torch.equal(got[2:-5], want[2:-5]) and bool((got[:2] == 9).all()) and bool((got[-5:] == 9).all())


def test_lse_of_padding():
    check_lse_of_padding("cpu", F32, [(30, 1), (100, 3)], None)


def check_forward_mode(device, dtype):
    """There is no gradient of either mode: tensors with a tangent are refused, in a dual level and under torch.func."""
    from torch.autograd import forward_ad

    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, dtype, device)
    qkv, q_w, k_w, f = append_inputs(b, False, dtype)
    calls = [(b.q, lambda t: paged.paged_attention(t, *b.args())), (b.k, lambda t: paged.paged_attention(b.q, t, *b.args()[1:])),
             (b.q.clone(), lambda t: paged.paged_attention(b.q, *b.args(), out=t)),
             (qkv, lambda t: paged.qkv_norm_rope_append(t, q_w, k_w, f, *b.args(), 4)),
             (q_w, lambda t: paged.qkv_norm_rope_append(qkv, t, k_w, f, *b.args(), 4))]
    for t, call in calls:
        t = t.nan_to_num(1.0)
        with forward_ad.dual_level():
            with pytest.raises(ValueError, match="no gradient"):
                call(forward_ad.make_dual(t, torch.ones_like(t)))
            call(t)
        with pytest.raises(ValueError, match="no gradient"):
            torch.func.jvp(call, (t,), (torch.ones_like(t),))


def test_forward_mode():
    check_forward_mode("cpu", F32)


def test_a_wait_that_ran_out_is_every_callers(monkeypatch):
    """Two callers on a device: the one that looks first takes nothing from the other."""
    class Native:
        words = [2, 71]

        def paged_status(self, device):
            assert device == 1
            return list(self.words)

    fake = Native()
    monkeypatch.setattr(paged, "native", lambda: fake)
    assert paged.waits_out("cpu") == 0
    first, second = paged.waits_out("cuda:1"), paged.waits_out("cuda:1")
    paged.check_waits("cuda:1", first)
    fake.words = [5, 72]
    for since in (first, second, first):
        with pytest.raises(RuntimeError, match="3 waits .* ran out .*at 72"):
            paged.check_waits("cuda:1", since)
    paged.check_waits("cuda:1", paged.waits_out("cuda:1"))
    with pytest.raises(RuntimeError):
        paged.check_waits("cuda:1")


def with_missing_pages(lens, hq, hk, d, page, window, dtype, device, index=torch.int32):
    """A batch with numbers that are no pages first, last and between those that its tokens see, a sequence without any page, and a length that passes
    the table's row (the row's last place has a page, so what a page has past its sequence's end is seen too: all rows are numbers)."""
    batch = oracle.Batch(lens, hq, hk, d, page, window, dtype, device, seed=page + d, before=1, after=2, index=index)
    for t in (batch.k, batch.v):
        t.copy_(torch.randn(t.shape, generator=torch.Generator().manual_seed(d)).to(t))
    pages, width = batch.k.shape[0], batch.table.shape[1]
    wrong = [pages, -1, 2 ** 31 - 1, -2 ** 31] + ([2 ** 32, 2 ** 32 + 1, -2 ** 32, 2 ** 63 - 1] if index == torch.int64 else [])
    for b, (c, n) in enumerate(lens):
        first, last = batch.first[b], (c + n - 1) // page
        for i, col in enumerate({0: [first], 1: [last], 2: [(first + last) // 2, (first + last) // 2 + 1], 3: range(first, width), 4: [first, last]}[b % 5]):
            if col < width:
                batch.table[b, col] = wrong[(b + i) % len(wrong)]
    last = len(lens) - 1
    batch.table[last] = torch.arange(width) % pages
    batch.seq_lens[last] = width * page + max(1, lens[last][1] // 2)
    return batch


@pytest.mark.parametrize("window", [None, 40])
def test_missing_pages(window):
    for index in (torch.int32, torch.int64):
        batch = with_missing_pages([(60, 20), (100, 3), (90, 30), (20, 5), (33, 1), (50, 20)], 4, 2, 64, 16, window, F64, "cpu", index)
        got = paged.paged_attention(batch.q, *batch.args(), window=window)
        oracle.close_attention(got, oracle.attention_of_pages(batch), 64, False, F64)
    whole = oracle.Batch([(60, 20), (100, 3), (0, 4)], 4, 2, 64, 16, window, F64)
    for a, b in zip(oracle.attention_of_pages(whole, 0.5), oracle.attention(whole, 0.5)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)


def check_pages_over_one_another(device, dtype):
    """Appending refuses keys and values in the same memory, and takes them side by side; attention reads them anyhow."""
    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, dtype, device)
    args = append_inputs(b, False, dtype)
    n, whole = b.k.shape[0], 2 * 16 * 64
    room = torch.zeros(4 * n * whole, dtype=dtype, device=device)

    def pages(at, stride):
        return room.as_strided((n, 2, 16, 64), (stride, 16 * 64, 64, 1), at)

    def append(k, v):
        return paged.qkv_norm_rope_append(*args, k, v, b.table, b.cu, b.seq_lens, 4)

    for k, v in (((0, whole), (0, whole)), ((0, 2 * whole), (whole // 2, 2 * whole)), ((whole, 2 * whole), (8, 2 * whole)), ((0, whole), ((n - 1) * whole, whole)),
                 ((0, 2 * whole), (whole, 3 * whole)), ((2 * whole, 3 * whole), (0, whole))):
        for one, two in ((k, v), (v, k)):
            with pytest.raises(ValueError, match="over one another"):
                append(pages(*one), pages(*two))
    want = append(b.k, b.v)
    for k, v in (((0, 2 * whole), (whole, 2 * whole)), ((0, whole), (n * whole, whole)), ((0, 4 * whole), (2 * whole, 4 * whole)),
                 ((0, 2 * whole), (2 * (n - 1) * whole + whole, whole))):
        for one, two in ((k, v), (v, k)):
            assert torch.equal(append(pages(*one), pages(*two)), want)
    o, lse = paged.paged_attention(b.q, pages(0, whole), pages(0, whole), b.table, b.cu, b.seq_lens)
    assert bool(o.isfinite().all())


def test_pages_over_one_another():
    check_pages_over_one_another("cpu", F32)


def check_largest_scale(device, dtype, lens):
    """A scale whose 1 / ln 2 fold passes 32 bits is refused; below, equal scores share alike."""
    b = oracle.Batch(lens, 4, 2, 64, 16, None, dtype, device)
    for scale in (2.0 ** 127, 3.0e38, 3.4e38):
        with pytest.raises(ValueError):
            paged.paged_attention(b.q, *b.args(), scale=scale)
    b.q.zero_()
    want = paged.paged_attention(b.q, *b.args())
    for scale in (1.7e38, 1e-44):
        got = paged.paged_attention(b.q, *b.args(), scale=scale)
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and bool(got[0].isfinite().all())


def test_largest_scale():
    check_largest_scale("cpu", F32, [(20, 2), (9, 3)])


def check_out_is_no_page(device, dtype):
    """`out` in the cache's memory: sequences are read after others' rows were written."""
    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, dtype, device)
    for pages in (b.k, b.v):
        with pytest.raises(RuntimeError, match="not the pages"):
            paged.paged_attention(b.q, *b.args(), out=pages.view(-1)[:b.q.numel()].view_as(b.q))


def test_out_is_no_page():
    check_out_is_no_page("cpu", F32)
