"""The paged cache's operators on the sm_100a kernels: against the 64-bit definitions at the sizes, layouts and lengths where they
can go wrong, with NaN wherever nothing may be read; edge rules as on the CPU; streams, graphs, repeatability, refusals."""
import math

import pytest
import torch

import paged_oracle as oracle
import test_paged
from micro_engram_fork_b200.ops import paged
from test_paged import alias_refusals, append_inputs, check_append, check_bad_offsets, check_bad_pages, check_negative_positions, check_wide_numbers, more_refusals, refusals

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF = torch.bfloat16

# (query heads, key heads, dim): the decoders' layers, groups of one, odd groups, one key head
HEADS = [(32, 16, 256), (32, 4, 512), (4, 2, 64), (4, 1, 128), (3, 3, 128), (15, 3, 128), (16, 1, 64), (6, 2, 256), (2, 2, 512), (9, 1, 512)]


@pytest.fixture(autouse=True)
def no_wait_ran_out():
    yield
    from micro_engram_fork_b200 import native

    assert native().paged_status(0) == [0, 0]


def _attend(batch, single, scale=1.0, max_q=None):
    got = paged.paged_attention(batch.q, *batch.args(), window=batch.window, scale=scale, max_q=max_q)
    oracle.close_attention(got, oracle.attention(batch, scale), batch.d, single)
    return got


@pytest.mark.parametrize("page", [16, 64, 128])
@pytest.mark.parametrize("window", [None, 1, 100])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_single_tokens(hq, hk, d, window, page):
    """Answers: one token a sequence, lengths around pages, tiles of 16 and blocks of 64, an empty sequence between."""
    lens = [(c, 1) for c in (0, 1, 14, 15, 16, 17, 62, 63, 64, 127, 128, 200, 333)]
    lens.insert(4, (50, 0))
    batch = oracle.Batch(lens, hq, hk, d, page, window, BF, DEV, seed=hq + d)
    _attend(batch, True, max_q=1)


@pytest.mark.parametrize("max_q", [None, 7, 1])
@pytest.mark.parametrize("window", [None, 5, 70])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_few_tokens(hq, hk, d, window, max_q):
    """Drafts, and a max_q that is too low."""
    lens = [(0, 7), (9, 2), (60, 5), (100, 7), (63, 3), (250, 1), (0, 1)]
    batch = oracle.Batch(lens, hq, hk, d, 32, window, BF, DEV, seed=hq + d, before=1, after=3)
    o, lse = _attend(batch, False, max_q=max_q)
    assert bool((o[0] == 0).all()) and bool((o[-3:] == 0).all()) and bool((lse[:, -3:] == -math.inf).all())


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("window", [None, 64, 130])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_chunks(hq, hk, d, window, page):
    """Chunks of prompts beside answers."""
    lens = [(0, 129), (37, 1), (200, 65), (5, 30), (127, 64), (0, 1), (300, 17)]
    batch = oracle.Batch(lens, hq, hk, d, page, window, BF, DEV, seed=page)
    _attend(batch, False)


@pytest.mark.parametrize("hq,hk,d,window", [(8, 2, 256, None), (8, 1, 512, None), (4, 2, 64, 900), (4, 1, 128, None)])
@pytest.mark.parametrize("lens", [[(20000, 1)], [(6000, 1), (3, 1), (9000, 1)], [(5000, 40)], [(700, 300), (4000, 2)]])
def test_long(lens, hq, hk, d, window):
    """Work that is cut into many pieces."""
    batch = oracle.Batch(lens, hq, hk, d, 64, window, BF, DEV, seed=5)
    single = all(n == 1 for _, n in lens)
    _attend(batch, single, max_q=1 if single else None)


def test_many_sequences():
    """More sequences than a block has threads, most of them empty."""
    lens = [((i * 7) % 90, 1 if i % 3 == 0 else 0) for i in range(700)]
    batch = oracle.Batch(lens, 4, 2, 64, 16, None, BF, DEV)
    _attend(batch, True, max_q=1)
    _attend(batch, False)
    check_append(oracle.Batch(lens, 4, 2, 64, 16, None, BF, DEV), False, BF, paged.qkv_norm_rope_append)


@pytest.mark.parametrize("kv_shared", [False, True])
@pytest.mark.parametrize("hq,hk,d", HEADS)
def test_append(hq, hk, d, kv_shared):
    lens = [(5, 3), (0, 37), (40, 0), (100000, 2), (63, 1), (0, 1), (15, 18)]
    batch = oracle.Batch(lens, hq, hk, d, 16, 40, BF, DEV, seed=d, before=2, after=3)
    check_append(batch, kv_shared, BF, paged.qkv_norm_rope_append)


@pytest.mark.parametrize("lens", [[(0, 1)], [(1000, 1)], [(3, 700), (70, 900)], [(7, 1)] * 300])
def test_append_sizes(lens):
    check_append(oracle.Batch(lens, 4, 1, 128, 64, 128, BF, DEV), True, BF, paged.qkv_norm_rope_append)


def test_layouts():
    """Keys and values as slices of one tensor, q and out as slices of rows, int64 lengths and tables, a table's slice."""
    lens = [(30, 1), (100, 9), (64, 2)]
    want = _attend(oracle.Batch(lens, 6, 2, 128, 32, None, BF, DEV), False)
    batch = oracle.Batch(lens, 6, 2, 128, 32, None, BF, DEV, together=True, index=torch.int64)
    wide = torch.full((batch.tokens, 7, 3, 128), math.nan, dtype=BF, device=DEV)
    wide[:, :6, 1] = batch.q
    batch.table = torch.cat([batch.table, batch.table + 1], 1)[:, :batch.table.shape[1]]
    out = torch.full_like(wide, 5.0)
    o, lse = paged.paged_attention(wide[:, :6, 1], *batch.args(), out=out[:, :6, 1])
    assert torch.equal(o, want[0]) and torch.equal(lse, want[1])
    assert bool((out[:, 6] == 5).all()) and bool((out[:, :, 0] == 5).all())
    odd = torch.cat([batch.q.reshape(-1), batch.q.reshape(-1)[:1]])[1:].view_as(batch.q)  # off 16 bytes: copied
    odd.copy_(batch.q)
    assert torch.equal(paged.paged_attention(odd, *batch.args())[0], want[0])
    qkv, q_w, k_w, f = append_inputs(batch, False, BF)
    first = paged.qkv_norm_rope_append(qkv, q_w, k_w, f, *batch.args(), 6)
    k, v = batch.k.clone(), batch.v.clone()
    rows = torch.full((batch.tokens, qkv.shape[1] + 8), math.nan, dtype=BF, device=DEV)
    rows[:, 8:] = qkv
    assert torch.equal(paged.qkv_norm_rope_append(rows[:, 8:], q_w, k_w, f, *batch.args(), 6), first)
    assert torch.equal(batch.k.nan_to_num(3.0), k.nan_to_num(3.0)) and torch.equal(batch.v.nan_to_num(3.0), v.nan_to_num(3.0))


def test_large_offsets():
    """Pages past 2^31 elements."""
    hk, page, d = 16, 128, 512
    pages = (1 << 31) // (hk * page * d) + 8
    small = oracle.Batch([(200, 3), (31, 1)], 32, hk, d, page, None, BF, DEV)
    big = oracle.Batch([(200, 3), (31, 1)], 32, hk, d, page, None, BF, DEV)
    k, v = torch.empty(2, pages, hk, page, d, dtype=BF, device=DEV)
    k[-small.k.shape[0]:], v[-small.k.shape[0]:] = small.k, small.v
    big.table = torch.where(small.table >= 0, small.table + pages - small.k.shape[0], -1)
    want = paged.paged_attention(small.q, *small.args())
    got = paged.paged_attention(big.q, k, v, big.table, big.cu, big.seq_lens)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    for n in (1, 300):
        small = oracle.Batch([(200, n)], 32, hk, d, page, None, BF, DEV)
        k[-small.k.shape[0]:], v[-small.k.shape[0]:] = small.k, small.v
        args = append_inputs(small, False, BF)
        want = paged.qkv_norm_rope_append(*args, *small.args(), 32)
        table = torch.where(small.table >= 0, small.table + pages - small.k.shape[0], -1)
        assert torch.equal(paged.qkv_norm_rope_append(*args, k, v, table, small.cu, small.seq_lens, 32), want)
        for now, was in ((k, small.k), (v, small.v)):
            assert torch.equal(now[-small.k.shape[0]:].nan_to_num(3.0), was.nan_to_num(3.0))


def test_values_at_the_edge():
    """Keys and values that are infinite or NaN reach the rows that see them and no others (single tokens); equal scores of any size."""
    for bad in (math.nan, math.inf):
        batch = oracle.Batch([(40, 1), (70, 1)], 4, 2, 64, 16, None, BF, DEV)
        clean = paged.paged_attention(batch.q, *batch.args(), max_q=1)[0]
        batch.v[int(batch.table[0, 1]), 0, 3, 5] = bad
        o = paged.paged_attention(batch.q, *batch.args(), max_q=1)[0]
        assert torch.equal(o[1], clean[1]) and torch.equal(o[0, 2:], clean[0, 2:])
        assert not bool(o[0, :2, 5].isfinite().any()) and torch.equal(o[0, :2, :5], clean[0, :2, :5])
    batch = oracle.Batch([(300, 1), (2, 1)], 4, 2, 64, 16, None, BF, DEV)
    batch.k.fill_(1000.0)
    batch.q.fill_(1000.0)
    o, lse = paged.paged_attention(batch.q, *batch.args(), max_q=1)
    assert torch.allclose(lse, (torch.tensor([301.0, 3.0], device=DEV).log() + 6.4e7).expand(4, 2), rtol=1e-6)
    o, lse = paged.paged_attention(-batch.q, *batch.args(), scale=1e20, max_q=1)
    assert bool(o.isfinite().all())


@pytest.mark.parametrize("single", [True, False])
def test_bad_pages(single):
    check_bad_pages(DEV, BF, single)


def test_bad_offsets():
    check_bad_offsets(DEV, BF)


def test_shared_pages_and_rings():
    """Sequences that share their first pages; a table that goes round a ring of pages under a window."""
    batch = oracle.Batch([(130, 1), (140, 1)], 4, 2, 64, 64, None, BF, DEV)
    batch.table[1, :2] = batch.table[0, :2]
    oracle.close_attention(paged.paged_attention(batch.q, *batch.args(), max_q=1), oracle.attention(batch), 64, True)
    want = oracle.Batch([(500, 20)], 4, 2, 64, 16, 40, BF, DEV)
    ring = 5  # 40 + 20 - 1 positions lie in 5 pages at most
    k, v = torch.full((2, ring, 2, 16, 64), math.nan, dtype=BF, device=DEV)
    table = torch.arange(33, dtype=torch.int32, device=DEV)[None] % ring
    for col in range(want.first[0], 33):
        k[col % ring], v[col % ring] = want.k[want.table[0, col]], want.v[want.table[0, col]]
    a = paged.paged_attention(want.q, k, v, table, want.cu, want.seq_lens, window=40)
    b = paged.paged_attention(want.q, *want.args(), window=40)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_out_and_padding():
    """Rows of no sequence: zeros, or left alone with out."""
    for lens in ([(30, 1), (100, 1)], [(30, 100), (7, 1)]):
        batch = oracle.Batch(lens, 4, 2, 64, 16, None, BF, DEV, before=1, after=5)
        want, lse = paged.paged_attention(batch.q, *batch.args())
        assert bool((want[0] == 0).all()) and bool((want[-5:] == 0).all()) and bool((lse[:, -5:] == -math.inf).all())
        out = torch.full_like(batch.q, 9.0)
        got, _ = paged.paged_attention(batch.q, *batch.args(), out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out[1:-5], want[1:-5])
        assert bool((out[0] == 9).all()) and bool((out[-5:] == 9).all())
    none = torch.zeros(0, dtype=torch.int32, device=DEV)
    o, lse = paged.paged_attention(batch.q, batch.k, batch.v, batch.table[:0], torch.zeros(1, dtype=torch.int32, device=DEV), none)
    assert bool((o == 0).all()) and bool((lse == -math.inf).all())
    o, lse = paged.paged_attention(batch.q[:0], *batch.args())
    assert o.shape == (0, 4, 64) and lse.shape == (4, 0)


@pytest.mark.parametrize("lens,max_q", [([(3000, 1), (50, 1)], 1), ([(900, 40), (50, 1)], None)])
def test_streams_and_graphs(lens, max_q):
    """Two streams at once, a captured call replayed on other lengths and pages, two graphs replayed in turn: the same bits."""
    batch = oracle.Batch(lens, 8, 2, 128, 32, None, BF, DEV)
    call = lambda: paged.paged_attention(batch.q, *batch.args(), max_q=max_q)  # noqa: E731
    want = [t.clone() for t in call()]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call()
        graphs.append((graph, out))
    for _ in range(3):
        for graph, out in graphs:
            graph.replay()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
    batch.seq_lens -= 7
    want = call()
    for graph, out in graphs:
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_append_graph():
    batch = oracle.Batch([(30, 1), (64, 1)], 4, 2, 64, 16, None, BF, DEV)
    args = append_inputs(batch, False, BF)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q = paged.qkv_norm_rope_append(*args, *batch.args(), 4)
    batch.seq_lens -= 1
    k = batch.k.clone()
    graph.replay()
    got = q.clone(), batch.k.clone(), batch.v.clone()
    want = paged.qkv_norm_rope_append(*args, *batch.args(), 4)
    assert torch.equal(got[0], want) and torch.equal(got[1].nan_to_num(3.0), batch.k.nan_to_num(3.0))
    assert not torch.equal(k.nan_to_num(3.0), batch.k.nan_to_num(3.0))


def test_refusals():
    for i, (error, call) in enumerate(refusals(DEV, BF)):
        with pytest.raises(error):
            call()
            pytest.fail(f"call {i} was taken")
    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, BF, DEV)
    k, v, table, cu, lens = b.args()
    qkv, q_w, k_w, f = append_inputs(b, False, BF)
    swapped = k.transpose(1, 2).contiguous().transpose(1, 2)
    calls = [
        lambda: paged.paged_attention(b.q.half(), k, v, table, cu, lens),
        lambda: paged.paged_attention(b.q, k.half(), v.half(), table, cu, lens),
        lambda: paged.paged_attention(b.q, k.float(), v.float(), table, cu, lens),
        lambda: paged.paged_attention(b.q, swapped, swapped, table, cu, lens),
        lambda: paged.paged_attention(b.q.cpu(), k, v, table, cu, lens),
        lambda: paged.paged_attention(b.q, k, v, table.cpu(), cu, lens),
        lambda: paged.paged_attention(b.q, k, v, table, cu.cpu(), lens),
        lambda: paged.paged_attention(b.q, k, v, table, cu, lens, out=b.q.float()),
        lambda: paged.paged_attention(b.q, k, v, table, cu, lens, out=b.q.clone().transpose(1, 2).contiguous().transpose(1, 2)),
        lambda: paged.qkv_norm_rope_append(qkv.float(), q_w, k_w, f, k, v, table, cu, lens, 4),
        lambda: paged.qkv_norm_rope_append(qkv, q_w.to(BF), k_w, f, k, v, table, cu, lens, 4),
        lambda: paged.qkv_norm_rope_append(qkv, q_w, k_w.cpu(), f, k, v, table, cu, lens, 4),
    ]
    for i, call in enumerate(calls):
        with pytest.raises(RuntimeError):
            call()
            pytest.fail(f"call {i} was taken")


def test_out_is_not_q():
    for call in alias_refusals(DEV, BF):
        with pytest.raises(ValueError):
            call()


def test_wide_numbers():
    check_wide_numbers(DEV, BF)


def test_negative_positions():
    check_negative_positions(DEV, BF)


def test_more_refusals():
    for call in more_refusals(DEV, BF):
        with pytest.raises(ValueError):
            call()
    b = oracle.Batch([(20, 2), (9, 3)], 4, 2, 64, 16, None, BF, DEV)
    room = torch.zeros(5 * 4 * 64, dtype=BF, device=DEV)
    for strides in ((8, 64, 1), (256, 32, 1), (128, 64, 1), (64, 256, 1)):  # heads that lie over one another
        with pytest.raises(RuntimeError):
            paged.paged_attention(b.q, *b.args(), out=room.as_strided((5, 4, 64), strides))
    got = paged.paged_attention(b.q, *b.args(), out=room.as_strided((5, 4, 64), (64, 320, 1)))[0]
    assert torch.equal(got, paged.paged_attention(b.q, *b.args())[0])


@pytest.mark.parametrize("hq,hk,d", [(4, 2, 256), (16, 1, 128), (5, 1, 64), (8, 1, 512)])
@pytest.mark.parametrize("window", [None, 1500])
def test_long_drafts(hq, hk, d, window):
    """Up to 16 rows a sequence that go through long caches together, in units that are cut, with single tokens between."""
    most = 16 // (hq // hk)
    lens = [(9000, most), (3, 1), (4000, max(most - 1, 1)), (2100, 0), (700, most), (0, most)]
    batch = oracle.Batch(lens, hq, hk, d, 32, window, BF, DEV, seed=d, before=2, after=1)
    _attend(batch, most == 1, max_q=most)


@pytest.mark.parametrize("hq,hk,d", [(3, 1, 64), (6, 2, 256), (2, 2, 512)])
def test_append_many(hq, hk, d):
    """More tokens than a wave has blocks: several a block, a last block that is not full, sequences that end inside one."""
    for tokens in (451, 1409):
        batch = oracle.Batch([(5, 301), (77, 1), (0, 0), (9, tokens - 302)], hq, hk, d, 64, None, BF, DEV, seed=d, before=1, after=2)
        check_append(batch, False, BF, paged.qkv_norm_rope_append)


@pytest.mark.parametrize("lens,max_q", [([(30, 1), (100, 1)], 1), ([(30, 100), (7, 1)], None), ([(30, 40), (7, 1), (9, 1), (50, 1), (3, 1)], None)])
def test_lse_of_padding(lens, max_q):
    """The kernel of few rows, that of chunks, both."""
    test_paged.check_lse_of_padding(DEV, BF, lens, max_q)


def test_forward_mode():
    test_paged.check_forward_mode(DEV, BF)


def test_waits_are_counted_beside_a_capture():
    """Looking at the count in one thread leaves another's capture whole; a stream that is captured is refused."""
    import threading

    batch = oracle.Batch([(900, 40), (50, 1)], 8, 2, 128, 32, None, BF, DEV)
    want = [t.clone() for t in paged.paged_attention(batch.q, *batch.args())]
    seen = []
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = paged.paged_attention(batch.q, *batch.args())
        look = threading.Thread(target=lambda: (paged.check_waits(DEV), seen.append(paged.waits_out(DEV))))
        look.start()
        look.join()
        with pytest.raises(RuntimeError, match="captured"):
            paged.waits_out(DEV)
    assert seen == [0]
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.cuda.stream(torch.cuda.Stream()):
        paged.check_waits(DEV, paged.waits_out(DEV))


@pytest.mark.parametrize("page", [16, 32, 64, 128])
@pytest.mark.parametrize("lens", [[(300, 1), (400, 1)], [(530, 40)], [(500, 1), (330, 70), (1000, 1), (40, 1), (900, 2)]])
def test_places_before_the_window(lens, page):
    """What the table holds for pages that no new token sees (here others' pages) changes nothing, with pages that are none among those seen or not."""
    for gap in (False, True):
        batch = oracle.Batch(lens, 4, 2, 64, page, 150, BF, DEV, seed=page)
        if gap:
            for b in range(len(lens)):
                batch.table[b, batch.first[b] + 1] = -1
        want = paged.paged_attention(batch.q, *batch.args(), window=150)
        for b, first in enumerate(batch.first):
            batch.table[b, :first] = batch.table[0, batch.first[0]] if b else batch.k.shape[0] - 1
            batch.table[b, -1] = 0
        got = paged.paged_attention(batch.q, *batch.args(), window=150)
        assert all(torch.equal(x, y) for x, y in zip(got, want)) and bool(got[0].isfinite().all())


# Batches that the kernel of few rows takes, that of chunks, and both of them (with 2 rows a token; the last sequence's length passes its table's row).
MIXES = {"rows": [(60, 3), (100, 1), (90, 4), (20, 5), (33, 1), (50, 2)], "chunks": [(300, 40), (120, 130)],
         "both": [(300, 30), (100, 1), (500, 2), (20, 5), (133, 1), (40, 1), (50, 20)]}


@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("window", [None, 100])
@pytest.mark.parametrize("d,page", [(64, 16), (128, 32), (256, 64), (512, 128), (512, 16), (256, 128)])
def test_missing_pages(d, page, window, mix):
    for index in (torch.int32, torch.int64):
        batch = test_paged.with_missing_pages(MIXES[mix], 4, 2, d, page, window, BF, DEV, index)
        got = paged.paged_attention(batch.q, *batch.args(), window=window)
        oracle.close_attention(got, oracle.attention_of_pages(batch), d, mix == "rows")
    assert bool((got[0][0] == 0).all()) and bool((got[1][:, -2:] == -math.inf).all())


@pytest.mark.parametrize("scale", [0.04, 0.3, 2.5])
@pytest.mark.parametrize("mix", MIXES)
@pytest.mark.parametrize("d", [64, 256, 512])
def test_scales(d, mix, scale):
    batch = oracle.Batch(MIXES[mix], 4, 2, d, 32, 200, BF, DEV, seed=d)
    _attend(batch, mix == "rows", scale=scale)


@pytest.mark.parametrize("group,d", [(17, 64), (17, 512), (24, 256), (40, 128), (64, 64), (65, 256), (100, 512), (128, 64), (128, 256)])
@pytest.mark.parametrize("lens", [[(5, 1), (300, 1), (64, 1), (0, 1), (1000, 1)], [(200, 9), (37, 1)], [(60, 3), (250, 2), (0, 4), (90, 1), (130, 2)]])
def test_many_query_heads(lens, group, d):
    """Up to 128 query heads a key head: tiles of few tokens, rows of a tile that no token has."""
    for hk in (1, 2):
        _attend(oracle.Batch(lens, group * hk, hk, d, 16, None, BF, DEV, seed=group, before=1, after=1), False)


@pytest.mark.parametrize("d", [64, 256, 512])
@pytest.mark.parametrize("lens", [[(3000, 40), (5000, 1)], [(2000, 300), (700, 5), (4000, 2)], [(9, 70), (4000, 5), (3000, 1), (20, 17), (100, 1), (8, 1), (5, 2)]])
def test_max_q_too_low_for_chunks(lens, d):
    """Longer runs than max_q says: such sequences are not cut, the others are."""
    for max_q in (5, 9):
        _attend(oracle.Batch(lens, 8, 2, d, 64, None, BF, DEV, seed=d), False, max_q=max_q)


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("window", [None, 70])
def test_sixteen_rows_keep_both_terms(d, window):
    """Drafts of 9 to 16 rows a key head, in units that are cut and whole ones: as near as single tokens."""
    for hq, hk in ((8, 2), (3, 1)):
        lens = [(900, 4), (63, 3), (0, 4), (2000, 3), (17, 1), (128, 4)]
        _attend(oracle.Batch(lens, hq, hk, d, 16, window, BF, DEV, seed=hq), True, max_q=4)


@pytest.mark.parametrize("d", [64, 256, 512])
@pytest.mark.parametrize("lens", [[(400, 40), (90, 130)], [(6000, 40)], [(400, 30), (60, 1), (300, 2), (2000, 1), (7, 1)]])
def test_values_at_the_edge_in_chunks(lens, d):
    """Values and keys that are infinite or NaN, at a position that every new token of a sequence sees: they reach that sequence's rows and
    columns and no others; a score of -inf is a key that is not seen."""
    for bad in (math.nan, math.inf):
        batch = oracle.Batch(lens, 4, 2, d, 16, None, BF, DEV, seed=d)
        clean, clean_lse = paged.paged_attention(batch.q, *batch.args())
        n = lens[0][1]
        page = int(batch.table[0, 1])
        was = float(batch.v[page, 0, 3, 5])
        batch.v[page, 0, 3, 5] = bad
        o, lse = paged.paged_attention(batch.q, *batch.args())
        assert not bool(o[:n, :2, 5].isfinite().any()) and torch.equal(lse, clean_lse)
        o[:n, :2, 5] = clean[:n, :2, 5]
        assert torch.equal(o, clean)
        batch.v[page, 0, 3, 5] = was
        batch.k[page, 0, 3] = bad
        batch.q[:n, 0], batch.q[:n, 1] = 1.0, -1.0  # scores of inf, and of -inf
        o, lse = paged.paged_attention(batch.q, *batch.args())
        assert not bool(o[:n, 0].isfinite().any()) and torch.equal(o[n:], clean[n:]) and torch.equal(o[:, 2:], clean[:, 2:])
        assert not bool(lse[0, :n].isfinite().any()) and torch.equal(lse[:, n:], clean_lse[:, n:])
        if bad == math.inf:
            k = batch.k.clone()
            k[page, 0, 3] = 100.0  # a score of -100 d: no share in 32 bits either
            want = paged.paged_attention(batch.q, k, *batch.args()[1:])
            assert torch.equal(o[:n, 1], want[0][:n, 1]) and torch.equal(lse[1, :n], want[1][1, :n])
        else:
            assert not bool(o[:n, 1].isfinite().any())


def test_pages_over_one_another():
    test_paged.check_pages_over_one_another(DEV, BF)


@pytest.mark.parametrize("mix", MIXES)
def test_largest_scale(mix):
    test_paged.check_largest_scale(DEV, BF, MIXES[mix])


def test_out_is_no_page():
    test_paged.check_out_is_no_page(DEV, BF)
