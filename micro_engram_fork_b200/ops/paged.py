"""A paged cache of keys and values: appending new tokens to it, and their attention over it (serving).

A layer's cache is two tensors of pages, k_pages and v_pages [P, Hk, page, D] (bf16 on a GPU; page 16, 32, 64 or 128
positions; D 64, 128, 256 or 512; a page contiguous, pages any multiple of 8 elements apart, so both may be slices of
one tensor). Position p of sequence b lies in row p % page of page block_table[b, p // page]. A call brings the new tokens
of a batch, packed: sequence b has the tokens cu_seqlens[b] .. cu_seqlens[b + 1] - 1, its last ones, and seq_lens[b]
tokens in all, so its new tokens have the positions seq_lens[b] - (their number) and on.

  qkv_norm_rope_append  the projection's heads normalised, q and k rotated by the position, k and v into their
                        pages, q out (what ops.norm.qkv_norm_rope does, with a cache)
  paged_attention       the new tokens' attention over all that their sequence has in the cache, themselves
                        included (what ops.attention.attention_fwd does, with a cache)

CUDA tensors run the sm_100a kernels (csrc/paged_append.cu, paged_attention.cu, paged_tiles.cu) on the current stream; nothing is read
back to the host, so a call can be captured into a graph and replayed with other lengths and pages of the same shapes.
CPU tensors run the plain PyTorch forms below, which compute in fp32 (fp64 for fp64 inputs). Rules that hold for both:

  pages      A page number outside [0, P), or a position past the table's row, is no page: nothing is stored there, and its keys
             are not seen. Pages that lie before every new token's window are never read, nor is their place in the table; a
             row of the table may name a page more than once (a sliding layer's ring), sequences may share pages that they
             only read.
  stale rows Rows of a page at positions past seq_lens, or before every new token's window, are never used: they may hold anything.
             A row that a new token sees and another does not (the chunk's own) must be finite for the other.
  tokens     Tokens of no sequence (before cu_seqlens[0], from cu_seqlens[-1] on) give rows of zeros (lse -inf) and store
             nothing; with `out`, its rows there stay as they were. Sequences without new tokens are left alone. cu_seqlens is
             taken within [0, tokens]; a token whose position is negative is stored nowhere and sees nothing. cu_seqlens must not fall:
             tokens that two sequences claim get either's result, or zeros.
  empty rows a row that sees no key: 0, lse -inf.

On a GPU, sums, maxima and outputs in the making are 32-bit. What multiplies the values, exp(score - maximum), is rounded to two bf16 terms
(relative error 2^-17) by the kernel of single tokens and drafts, and to one (2^-8, as the values have) by that of chunks: errors of o against 64 bits are
0.0017 and 0.0022 of its mean size, where rounding o alone makes 0.0017. A batch of few sequences, or one of 32 rows (new tokens times query heads a key
head) a sequence on average, goes through the second one whole, single tokens among them: their last bits depend on what they are batched with.
The log-sum-exp is that of the unrounded terms either way. A batch of single tokens alone with max_q = 1 always takes the first kernel, up to 16 query
heads a key head.

Every wait inside the attention kernels is bounded; one that ran out (which no input causes) leaves its results wrong
and is counted on the device, for good: a caller takes the count (waits_out) before its calls and compares it after them
(check_waits), whoever else does; another caller's between the two raises as well. Both wait for the current stream.

There is no gradient: a call on tensors that require one is refused while gradients are recorded, and one on tensors with a tangent.
"""
import torch
from torch.autograd import forward_ad

from .. import native
from . import use_native
from .objectives import kernel_call

PAGES = (16, 32, 64, 128)
DIMS = (64, 128, 256, 512)


def _no_gradient(what, *tensors):
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError(f"{what} has no gradient: call it under torch.no_grad()")
    # (without a level there are no tangents, and looking at six tensors would cost a call 3.4 us)
    if forward_ad._current_level >= 0 and any(forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise ValueError(f"{what} has no gradient: a tensor has a tangent")


# ------------------------------------------------------------------------- argument checks of the plain forms
# (the kernels' entry points check the same in C++)
def _check_cache(k_pages, v_pages):
    if k_pages.dim() != 4 or k_pages.shape != v_pages.shape or k_pages.numel() == 0:
        raise ValueError(f"k_pages and v_pages: [pages, heads, page, dim] each is needed, got {tuple(k_pages.shape)} and {tuple(v_pages.shape)}")
    if k_pages.shape[2] not in PAGES:
        raise ValueError(f"k_pages: pages of 16, 32, 64 or 128 positions are needed, got {k_pages.shape[2]}")
    if k_pages.shape[3] not in DIMS:
        raise ValueError(f"k_pages: a head dimension of 64, 128, 256 or 512 is needed, got {k_pages.shape[3]}")


def _overlap(k_pages, v_pages):
    """Whether a page of keys lies over one of values (pages whose elements are contiguous, as the kernels take them)."""
    pages, whole, size = len(k_pages), k_pages[0].numel(), k_pages.element_size()
    k, v = k_pages.data_ptr() // size, v_pages.data_ptr() // size
    if not (k_pages[0].is_contiguous() and v_pages[0].is_contiguous()):
        return k == v
    sk, sv = (whole, whole) if pages == 1 else (k_pages.stride(0), v_pages.stride(0))
    if k + (pages - 1) * sk + whole <= v or v + (pages - 1) * sv + whole <= k:
        return False
    if sk == sv and sk > 0:  # each other's gaps
        return (v - k) % sk < whole or (v - k) % sk > sk - whole
    at = sorted([(k + i * sk, 0) for i in range(pages)] + [(v + i * sv, 1) for i in range(pages)])
    return any(b - a < whole and of != other for (a, of), (b, other) in zip(at, at[1:]))


def _check_batch(block_table, cu_seqlens, seq_lens):
    if seq_lens.dim() != 1 or cu_seqlens.dim() != 1 or cu_seqlens.numel() != seq_lens.numel() + 1:
        raise ValueError(f"cu_seqlens, seq_lens: [sequences + 1] and [sequences] are needed, got {tuple(cu_seqlens.shape)} and {tuple(seq_lens.shape)}")
    if block_table.dim() != 2 or block_table.shape[0] != seq_lens.numel():
        raise ValueError(f"block_table: [sequences, pages of the longest] is needed, got {tuple(block_table.shape)}")
    for t, what in ((cu_seqlens, "cu_seqlens"), (seq_lens, "seq_lens"), (block_table, "block_table")):
        if t.dtype not in (torch.int32, torch.int64):
            raise ValueError(f"{what}: int32 or int64 is needed, got {t.dtype}")


def _sequences(cu_seqlens, seq_lens, tokens):
    """(index, first new token, new tokens, tokens in the cache before them) of the sequences that have new tokens."""
    cu = [min(max(c, 0), tokens) for c in cu_seqlens.tolist()]
    for b, n in enumerate(seq_lens.tolist()):
        count = max(cu[b + 1], cu[b]) - cu[b]
        if count:
            yield b, cu[b], count, max(n, 0) - count


def _pages_of(block_table, b, positions, page, pages):
    """(the pages of these positions of sequence b, which of them are pages)."""
    col = positions // page
    ok = (positions >= 0) & (col < block_table.shape[1])
    if block_table.shape[1] == 0:
        return torch.zeros_like(positions), ok
    ids = block_table[b].long()[col.clamp(0, block_table.shape[1] - 1)]
    ok = ok & (ids >= 0) & (ids < pages)
    return torch.where(ok, ids, 0), ok


def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


# ------------------------------------------------------------------------- append
def qkv_norm_rope_append_ref(qkv, q_w, k_w, inv_freq, k_pages, v_pages, block_table, cu_seqlens, seq_lens, q_heads, kv_shared=False, eps=1e-6):
    hk, page, d = k_pages.shape[1:]
    tokens = qkv.shape[0]
    x = _wide(qkv).reshape(tokens, qkv.shape[1] // d, d)
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps)
    q = torch.zeros(tokens, q_heads, d, dtype=qkv.dtype, device=qkv.device)
    for b, first, count, context in _sequences(cu_seqlens, seq_lens, tokens):
        skip = max(0, -context)  # tokens at negative positions
        if skip >= count:
            continue
        n = x[first + skip:first + count]
        pos = torch.arange(context + skip, context + count, device=qkv.device)
        # the angle of a far position keeps no fraction in 32 bits
        angle = torch.remainder(pos.double()[:, None] * inv_freq.double(), 2 * torch.pi)[:, None]
        cos, sin = angle.cos().to(x.dtype), angle.sin().to(x.dtype)

        def rotated(y):
            lo, hi = y[..., :d // 2], y[..., d // 2:]
            return torch.cat((lo * cos - hi * sin, hi * cos + lo * sin), -1).to(qkv.dtype)

        q[first + skip:first + count] = rotated(n[:, :q_heads] * q_w)
        ids, ok = _pages_of(block_table, b, pos, page, k_pages.shape[0])
        at, row = ids[ok], (pos % page)[ok]
        k_pages[at, :, row] = rotated(n[:, q_heads:q_heads + hk] * k_w)[ok].to(k_pages.dtype)
        v_pages[at, :, row] = n[:, -hk:].to(qkv.dtype)[ok].to(v_pages.dtype)
    return q


def qkv_norm_rope_append(qkv, q_w, k_w, inv_freq, k_pages, v_pages, block_table, cu_seqlens, seq_lens, q_heads, kv_shared=False, eps=1e-6):
    """q [T, Hq, D] of the fused projection's rows qkv [T, (Hq + 2 Hk) D] (or [T, (Hq + Hk) D] with kv_shared: v is
    the raw k); k and v are written into their pages. Each head is normalised (y = x / sqrt(mean x^2 + eps)), q and k take their
    weights [D] and are rotated by position * inv_freq [D / 2] (fp32), v takes neither. All in 32 bits (the angle in 64), rounded
    once. Two new tokens must not share a place in the cache, nor pages of keys and of values memory."""
    _no_gradient("qkv_norm_rope_append", qkv, q_w, k_w, inv_freq, k_pages, v_pages)
    args = (qkv, q_w, k_w, inv_freq, k_pages, v_pages, block_table, cu_seqlens, seq_lens, int(q_heads), bool(kv_shared), float(eps))
    if use_native(qkv, k_pages):
        return kernel_call("paged_append", *args)
    _check_cache(k_pages, v_pages)
    _check_batch(block_table, cu_seqlens, seq_lens)
    d = k_pages.shape[3]
    width = (q_heads + (1 if kv_shared else 2) * k_pages.shape[1]) * d
    if q_heads < 1 or qkv.dim() != 2 or qkv.shape[1] != width:
        raise ValueError(f"qkv: [tokens, {width}] is needed for {q_heads} q heads, got {tuple(qkv.shape)}")
    for t, n, what in ((q_w, d, "q_w"), (k_w, d, "k_w"), (inv_freq, d // 2, "inv_freq")):
        if t.shape != (n,):
            raise ValueError(f"{what}: [{n}] is needed, got {tuple(t.shape)}")
    if _overlap(k_pages, v_pages):
        raise ValueError("k_pages and v_pages: they lie over one another, and both are written")
    with torch.no_grad():
        return qkv_norm_rope_append_ref(*args)


# ------------------------------------------------------------------------- attention
def paged_attention_ref(q, k_pages, v_pages, block_table, cu_seqlens, seq_lens, window=0, scale=1.0, out=None):
    tokens, hq, d = q.shape
    pages, hk, page, _ = k_pages.shape
    o = torch.zeros_like(q) if out is None else out
    lse = torch.full((hq, tokens), -float("inf"), dtype=_wide(q).dtype, device=q.device)
    for b, first, count, context in _sequences(cu_seqlens, seq_lens, tokens):
        end = min(context + count, block_table.shape[1] * page)
        key = torch.arange(max(0, context - window + 1) if window else 0, max(end, 0), device=q.device)
        ids, ok = _pages_of(block_table, b, key, page, pages)
        key, ids = key[ok], ids[ok]
        k = _wide(k_pages[ids, :, key % page]).transpose(0, 1).repeat_interleave(hq // hk, 0)
        v = _wide(v_pages[ids, :, key % page]).transpose(0, 1).repeat_interleave(hq // hk, 0)
        pos = torch.arange(context, context + count, device=q.device)[:, None]
        seen = key[None] <= pos
        if window:
            seen &= key[None] > pos - window
        x = torch.matmul(_wide(q[first:first + count]).transpose(0, 1), k.transpose(1, 2)) * scale
        x = x.masked_fill(~seen, -float("inf"))
        e = torch.logsumexp(x, -1) if key.numel() else lse[:, first:first + count]
        p = torch.exp(x - torch.where(e == -float("inf"), 0.0, e)[..., None])
        o[first:first + count] = torch.matmul(p, v).transpose(0, 1).to(q.dtype)
        lse[:, first:first + count] = e
    return o, lse


def paged_attention(q, k_pages, v_pages, block_table, cu_seqlens, seq_lens, window=None, scale=1.0, max_q=None, out=None):
    """(o [T, Hq, D], lse [Hq, T] fp32) of q [T, Hq, D]: softmax(scale q . k) v over the keys at positions
    [max(0, p - window + 1), p] of the row's sequence (p: the row's position; window None: all of them). Hq is a multiple of Hk; the
    pages hold the new tokens too (append first). max_q: the longest run of new tokens if the host knows it; with it a batch of
    single tokens skips what only longer runs need, and goes to the kernel that is made for them (a longer run than max_q says is still right, and
    slower). out: where o goes,
    a tensor of its own."""
    _no_gradient("paged_attention", q, k_pages, v_pages, *(() if out is None else (out,)))
    if window is not None and window < 1 or max_q is not None and max_q < 1:
        raise ValueError(f"window, max_q: a positive number or None, got {window} and {max_q}")
    if use_native(q, k_pages):
        return tuple(kernel_call("paged_attention", q, k_pages, v_pages, block_table, cu_seqlens, seq_lens, int(window or 0), float(scale),
                                 int(max_q or 0), out))
    _check_cache(k_pages, v_pages)
    _check_batch(block_table, cu_seqlens, seq_lens)
    hk, d = k_pages.shape[1], k_pages.shape[3]
    if q.dim() != 3 or q.shape[2] != d:
        raise ValueError(f"q: [tokens, heads, {d}] is needed, got {tuple(q.shape)}")
    if q.shape[1] < hk or q.shape[1] % hk or q.shape[1] // hk > 128:
        raise ValueError(f"q: heads a multiple of the pages' {hk} (up to 128 times) are needed, got {q.shape[1]}")
    if not 0 < float(torch.tensor(scale, dtype=torch.float32)) < 2.0 ** 127:
        raise ValueError(f"scale: a positive number (in 32 bits) below 2^127 is needed, got {scale}")
    if out is not None and out.shape != q.shape:
        raise ValueError(f"out: q's shape {tuple(q.shape)} is needed, got {tuple(out.shape)}")
    if out is not None and out.numel() and out.untyped_storage().data_ptr() == q.untyped_storage().data_ptr():
        raise ValueError("out: a tensor of its own is needed, not q's memory")
    if out is not None and out.numel() and out.untyped_storage().data_ptr() in (k_pages.untyped_storage().data_ptr(), v_pages.untyped_storage().data_ptr()):
        raise RuntimeError("out: a tensor of its own is needed, not the pages")
    with torch.no_grad():
        return paged_attention_ref(q, k_pages, v_pages, block_table, cu_seqlens, seq_lens, int(window or 0), float(scale), out)


def _waits(device):
    device = torch.device(device)
    if device.type != "cuda":
        return 0, 0
    return native().paged_status(torch.cuda.current_device() if device.index is None else device.index)


def waits_out(device):
    """How often a bounded wait of the attention kernels has run out on this device in this process, up to what its current stream
    has ahead."""
    return _waits(device)[0]


def check_waits(device, since=0):
    """Raises if a bounded wait of the attention kernels ran out on this device since waits_out gave `since` (0: in this process)."""
    count, where = _waits(device)
    if count != since:
        raise RuntimeError(f"paged_attention: {count - since} waits on the device ran out (the last at {where}); results since the count was "
                           f"{since} are not valid")
