"""Training objectives over the vocabulary: a teacher's top logits, distillation from them, token
log-probabilities and the paired preference loss.

Every function takes rows of raw logits [..., V] (the output head's product, bf16, fp16 or fp32; a
row's logits contiguous, any distance between rows) and applies the model's final softcap
z = c tanh(x / c) itself. Gradients are those in the raw logits, in their type, rounded once.

  top_logits              what a teacher records: its k largest logits, their ids, the log-sum-exp
  distill_loss            weighted KL(teacher || student) of each token (autograd)
  distill_loss_grad       the same with its gradient in one call, optionally in place of the logits
  token_logprobs          log softmax(z)[target] of each token (autograd)
  token_logprobs_grad     the same with its gradient for given coefficients in one call
  preference_loss         paired log-ratio loss of packed chosen / rejected sequences, on token
                          log-probabilities (autograd)
  preference_loss_grad    the same with its gradient in the log-probabilities in one call
  preference_logits_grad  from logits to the loss and its gradient in the logits in one call

CUDA tensors run the sm_100a kernels (csrc/objectives.cu, top_logits.cu, preference.cu) on the current
stream; CPU tensors run the plain PyTorch forms below, which compute in fp32 (fp64 for fp64 logits)
and are the tests' second opinion. Rules that hold for both:

  targets       -100 is an untrained token: log-probability 0, gradient 0, its logits are not read.
                Any other target outside [0, V) gives NaN.
  logits        V is at most 2^31 - 4097 for the kernels, k (teacher's entries, top logits) at most 256
  teacher_ids   an id outside [0, V) is an unused entry; ids of one row are distinct (a repeated id
                counts as the sum of its probabilities)
  weights       0 is an untrained token: loss 0, gradient 0, whatever its logits hold (as where there is nothing to
                match: no entry, and no teacher_lse)
  non-finite    -inf logits have probability 0; a NaN or +inf logit makes its row's results NaN
                (with a softcap +-inf are +-c)
"""
import torch

from .. import native
from . import use_native

IGNORE = -100
MAX_TOP = 256
KINDS = ("sigmoid", "hinge", "ipo")


# ------------------------------------------------------------------------- argument checks
# (of the plain forms; the kernels' entry points check the same in C++, where it costs a call next to nothing)
def _kernel(name, *args):
    """A kernel's entry point; its complaints about an argument's value are ValueErrors."""
    try:
        return getattr(native(), name)(*args)
    except RuntimeError as e:
        head, mark, text = str(e).partition("value: ")
        if head or not mark:
            raise
        raise ValueError(text.split("\nException raised from", 1)[0]) from None


def _cap(softcap):
    cap = 0.0 if softcap is None else float(softcap)
    if not 0.0 <= cap < float("inf"):
        raise ValueError(f"softcap: a positive number or None, got {softcap}")
    return cap


def _temperature(t):
    t = float(t)
    if not 0.0 < t < float("inf"):
        raise ValueError(f"temperature: a positive number, got {t}")
    return t


def _rows(x):
    """[..., V] logits as [N, V] (a view where the leading dimensions allow one)."""
    if x.dim() < 1 or not x.is_floating_point():
        raise ValueError(f"logits [..., V] of a floating type are needed, got {x.dtype} of shape {tuple(x.shape)}")
    if x.shape[-1] == 0:
        raise ValueError("logits of an empty vocabulary")
    return x.flatten(0, -2) if x.dim() > 2 else x.unsqueeze(0) if x.dim() == 1 else x


def _per_row(t, lead, what):
    if t is None:
        return None
    if tuple(t.shape) != tuple(lead):
        raise ValueError(f"{what}: shape {tuple(lead)} (one value a row of logits) is needed, got {tuple(t.shape)}")
    return t.reshape(-1)


def _out_rows(out, x):
    if out is None:
        return None
    if out.shape != x.shape or out.dtype != x.dtype or out.device != x.device:
        raise ValueError("out: the logits' shape, type and device are needed")
    rows = _rows(out)
    if rows.data_ptr() != out.data_ptr():
        raise ValueError("out: its leading dimensions have to flatten without a copy")
    return rows


def _targets(targets, lead):
    t = _per_row(targets, lead, "targets")
    if t.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"targets: int64 or int32 is needed, got {t.dtype}")
    return t


def _teacher(ids, logits, lead):
    if ids.shape != logits.shape or tuple(ids.shape[:-1]) != tuple(lead):
        raise ValueError(f"teacher_ids and teacher_logits: shape {tuple(lead)} + [k] is needed, got {tuple(ids.shape)} "
                         f"and {tuple(logits.shape)}")
    if not 1 <= ids.shape[-1] <= MAX_TOP:
        raise ValueError(f"teacher_ids: 1 to {MAX_TOP} entries a row, got {ids.shape[-1]}")
    if ids.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"teacher_ids: int64 or int32 is needed, got {ids.dtype}")
    return ids.reshape(-1, ids.shape[-1]), logits.reshape(-1, ids.shape[-1])


def _pair_args(beta, label_smoothing, kind):
    if kind not in KINDS:
        raise ValueError(f"kind: one of {', '.join(KINDS)}, got {kind!r}")
    if not 0.0 < beta < float("inf"):
        raise ValueError(f"beta: a positive number, got {beta}")
    if not 0.0 <= label_smoothing <= 0.5 or (label_smoothing and kind != "sigmoid"):
        raise ValueError(f"label_smoothing: 0 to 0.5, of the sigmoid loss only, got {label_smoothing} with {kind}")
    return KINDS.index(kind), float(beta), float(label_smoothing)


def _check_offsets(cu_seqlens):
    if cu_seqlens.dim() != 1 or cu_seqlens.numel() % 2 != 1:
        raise ValueError("cu_seqlens: offsets [2 pairs + 1] of packed sequences (chosen, rejected, chosen, ...) are "
                         f"needed, got shape {tuple(cu_seqlens.shape)}")
    if cu_seqlens.dtype not in (torch.int64, torch.int32):
        raise ValueError(f"cu_seqlens: int64 or int32 is needed, got {cu_seqlens.dtype}")


# ------------------------------------------------------------------------- plain PyTorch forms
def _softcapped(x, cap):
    """(z, dz/dx), in fp32 or wider."""
    x = x if x.dtype == torch.float64 else x.float()
    if not cap:
        return x, torch.ones_like(x)
    t = torch.tanh(x / cap)
    return t * cap, 1 - t * t


def top_logits_ref(x, k, cap=0.0, temperature=1.0):
    z, _ = _softcapped(x, cap)
    key = x if x.dtype == torch.float64 else x.float()
    ids = torch.sort(key, dim=1, descending=True, stable=True)[1][:, :k].contiguous()
    return z.gather(1, ids), ids, _log_sum_exp(z / temperature)


def _log_sum_exp(y):
    """log sum exp of rows; NaN where a row holds +inf (as in the kernels)."""
    lse = torch.logsumexp(y, dim=1)
    return torch.where(lse == float("inf"), float("nan"), lse)


def token_logprobs_ref(x, targets, cap=0.0):
    """(logp [N], gradient function: coefficients [N] -> [N, V])."""
    z, slope = _softcapped(x, cap)
    V = x.shape[1]
    targets = targets.long()
    trained = targets != IGNORE
    valid = (targets >= 0) & (targets < V)
    col = targets.clamp(0, V - 1).unsqueeze(1)
    log_p = z - _log_sum_exp(z).unsqueeze(1)
    logp = torch.where(valid, log_p.gather(1, col).squeeze(1), float("nan"))
    logp = torch.where(trained, logp, 0.0)

    def grad(g):
        c = torch.where(valid, g.to(z.dtype), float("nan")).unsqueeze(1)
        d = -log_p.exp()
        d.scatter_add_(1, col, torch.ones_like(col, dtype=z.dtype))
        return torch.where(trained.unsqueeze(1), c * d * slope, 0.0).to(x.dtype)

    return logp, grad


def _merge_repeats(ids, used, t):
    """(used, t) with repeated ids merged: an id's first entry has the log of its entries' summed exponentials, the
    others are unused."""
    at = torch.where(used, ids, -1).sort(dim=1)[0]
    rows = ((at[:, 1:] == at[:, :-1]) & (at[:, 1:] >= 0)).any(dim=1).nonzero().squeeze(1)
    if rows.numel() == 0:
        return used, t
    mine, use = ids[rows], used[rows]
    same = (mine.unsqueeze(2) == mine.unsqueeze(1)) & use.unsqueeze(1) & use.unsqueeze(2)
    first = use & ~same.tril(-1).any(dim=2)
    sums = torch.where(same, t[rows].unsqueeze(1), float("-inf")).logsumexp(dim=2)
    one = torch.where(same.sum(dim=2) > 1, sums, t[rows])
    return used.index_copy(0, rows, first), t.index_copy(0, rows, torch.where(first, one, float("-inf")))


def distill_ref(x, ids, top, lse=None, weights=None, cap=0.0, temperature=1.0):
    """(loss [N], gradient of sum(loss) [N, V])."""
    z, slope = _softcapped(x, cap)
    N, V = x.shape
    y = z / temperature
    ids = ids.long()
    used = (ids >= 0) & (ids < V)
    col = ids.clamp(0, V - 1)
    used, t = _merge_repeats(ids, used, torch.where(used, top.to(z.dtype) / temperature, float("-inf")))
    log_p = y - _log_sum_exp(y).unsqueeze(1)
    p = log_p.exp()
    some = t.amax(dim=1, keepdim=True) != float("-inf")
    if lse is None:
        log_q = t - torch.where(some, torch.logsumexp(t, dim=1, keepdim=True), 0.0)
    else:
        log_q = t - lse.to(z.dtype).unsqueeze(1)
    q = log_q.exp()
    kl = torch.where(q != 0, q * (log_q - log_p.gather(1, col)), 0.0).sum(1)
    if lse is not None:
        entry = torch.zeros(N, V + 1, dtype=torch.bool, device=x.device)
        entry = entry.scatter_(1, torch.where(used, ids, V), True)[:, :V]
        log_rest = torch.logsumexp(torch.where(entry, float("-inf"), log_p), dim=1)
        q_rest = (1 - q.sum(1)).clamp_min(0)
        q_rest = torch.where(used.sum(1) < V, q_rest, torch.zeros_like(q_rest))
        kl = kl + torch.where(q_rest > 0, q_rest * (q_rest.log() - log_rest), 0.0)
        share = torch.where(entry | (log_rest == float("-inf")).unsqueeze(1), 0.0, (log_p - log_rest.unsqueeze(1)).exp())
        d = p * (q.sum(1) + q_rest).unsqueeze(1) - q_rest.unsqueeze(1) * share  # the entries may sum to more than 1
    else:
        d = torch.where(some, p, 0.0)
    d = d.scatter_add(1, col, -torch.where(used, q, 0.0)) * slope * temperature
    w = torch.ones(N, dtype=z.dtype, device=x.device) if weights is None else weights.to(z.dtype)
    on = w != 0 if lse is not None else (w != 0) & some.squeeze(1)  # (no entry and no rest: nothing to match)
    return (torch.where(on, w * temperature ** 2 * kl, 0.0),
            torch.where(on.unsqueeze(1), w.unsqueeze(1) * d, 0.0).to(x.dtype))


def preference_ref(logps, ref_logps, cu_seqlens, kind=0, beta=0.1, smooth=0.0, scale=1.0, targets=None):
    """(loss [P], rewards [P, 2], scale * gradient of sum(loss) in the log-probabilities [T])."""
    lp = logps if logps.dtype == torch.float64 else logps.float()
    ratio = lp if ref_logps is None else lp - ref_logps.to(lp.dtype)
    if targets is not None:
        ratio = torch.where(targets != IGNORE, ratio, 0.0)
    T, pairs = lp.numel(), cu_seqlens.numel() // 2
    cu = torch.cummax(cu_seqlens.long(), 0)[0].clamp(0, T)
    seq = torch.searchsorted(cu, torch.arange(T, device=lp.device), right=True) - 1  # -1 / 2 pairs: outside
    sums = torch.zeros(2 * pairs + 2, dtype=lp.dtype, device=lp.device).index_add_(0, seq + 1, ratio)
    sums = sums[1:-1].view(pairs, 2)
    h = sums[:, 0] - sums[:, 1]
    u = beta * h
    if kind == 0:
        loss = (1 - smooth) * torch.nn.functional.softplus(-u)
        if smooth:  # (0 times infinity where the rejected answer is impossible)
            loss = loss + smooth * torch.nn.functional.softplus(u)
        d = beta * (smooth - torch.sigmoid(-u))
    elif kind == 1:
        loss = (1 - u).clamp_min(0)
        d = torch.where(u.isnan(), u, torch.where(u < 1, -beta, 0.0))
    else:
        loss = (h - 0.5 / beta).square()
        d = 2 * (h - 0.5 / beta)
    d = torch.nn.functional.pad(torch.stack([d, -d], 1).reshape(-1) * scale, (1, 1))
    return loss, beta * sums, d[seq + 1]


# ------------------------------------------------------------------------- teacher's top logits
def top_logits(logits, k, softcap=None, temperature=1.0):
    """The k largest logits of each row, after the softcap, in descending order (equal logits by the
    lower id; NaN above +inf): (values [..., k] fp32, ids [..., k] int64, lse [...] fp32), lse the
    log-sum-exp of the whole row at `temperature`, which distill_loss takes as teacher_lse. k is at
    most 256. No gradient."""
    if logits.dim() != 2:
        lead = logits.shape[:-1]
        values, ids, lse = top_logits(_rows(logits), k, softcap, temperature)
        return values.view(*lead, k), ids.view(*lead, k), lse.view(lead)
    if use_native(logits):
        return tuple(_kernel("top_logits", logits, k, softcap, temperature))
    x, cap, temperature = _rows(logits), _cap(softcap), _temperature(temperature)
    if not 1 <= k <= min(x.shape[1], MAX_TOP):
        raise ValueError(f"k: 1 to {min(x.shape[1], MAX_TOP)}, got {k}")
    with torch.no_grad():
        return top_logits_ref(x, k, cap, temperature)


# ------------------------------------------------------------------------- token log-probabilities
class _TokenLogprobsRef(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, targets, cap):
        ctx.cap = cap
        ctx.save_for_backward(x, targets)
        return token_logprobs_ref(x, targets, cap)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, targets = ctx.saved_tensors
        return token_logprobs_ref(x, targets, ctx.cap)[1](g), None, None


def token_logprobs(logits, targets, softcap=None):
    """log softmax(z)[target] of each row, fp32 [...]; targets [...] with -100 untrained (0)."""
    if logits.dim() != 2:
        lead = logits.shape[:-1]
        return token_logprobs(_rows(logits), _per_row(targets, lead, "targets"), softcap).view(lead)
    if use_native(logits):
        return _kernel("token_logprobs", logits, targets, softcap)
    return _TokenLogprobsRef.apply(_rows(logits), _targets(targets, logits.shape[:1]), _cap(softcap))


def token_logprobs_grad(logits, targets, coefficients=None, softcap=None, out=None):
    """(token_logprobs [...], gradient of sum(coefficients * token_logprobs) [..., V]) in one call;
    coefficients [...] are 1 unless given. `out` as in distill_loss_grad."""
    if logits.dim() != 2:
        lead = logits.shape[:-1]
        logp, dx = token_logprobs_grad(_rows(logits), _per_row(targets, lead, "targets"),
                                       _per_row(coefficients, lead, "coefficients"), softcap, _out_rows(out, logits))
        return logp.view(lead), dx.view(logits.shape) if out is None else out
    if use_native(logits):
        logp, dx = _kernel("token_logprobs_grad", logits, targets, coefficients, softcap, out)
        return logp, dx if out is None else out
    x, lead = _rows(logits), logits.shape[:1]
    t, g = _targets(targets, lead), _per_row(coefficients, lead, "coefficients")
    _out_rows(out, logits)
    with torch.no_grad():
        logp, grad = token_logprobs_ref(x, t, _cap(softcap))
        dx = grad(torch.ones_like(logp) if g is None else g)
        return logp, dx if out is None else out.copy_(dx)


# ------------------------------------------------------------------------- distillation
class _DistillRef(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, ids, top, lse, weights, cap, temperature):
        ctx.args = cap, temperature
        ctx.save_for_backward(x, ids, top, lse, weights)
        return distill_ref(x, ids, top, lse, weights, cap, temperature)[0]

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g):
        x, ids, top, lse, weights = ctx.saved_tensors
        w = g if weights is None else torch.where(weights != 0, weights * g, 0.0)
        return distill_ref(x, ids, top, lse, w, *ctx.args)[1], None, None, None, None, None, None


def _flat_teacher(logits, ids, top, lse, weights):
    """The arguments of logits with other than two dimensions, by rows."""
    lead = logits.shape[:-1]
    ids, top = _teacher(ids, top, lead)
    return _rows(logits), ids, top, _per_row(lse, lead, "teacher_lse"), _per_row(weights, lead, "weights")


def _checked_teacher(logits, ids, top, lse, weights, softcap, temperature):
    return (*_flat_teacher(logits, ids, top, lse, weights), _cap(softcap), _temperature(temperature))


def distill_loss(logits, teacher_ids, teacher_logits, teacher_lse=None, weights=None, softcap=None, temperature=1.0):
    """weights * temperature^2 * KL(teacher || student) of each row, fp32 [...].

    teacher_ids / teacher_logits [..., k]: the teacher's entries (its logits after its own softcap),
    k at most 256. Without teacher_lse the teacher's distribution is the softmax of its entries; with
    teacher_lse [...] (top_logits' lse at the same temperature) the entries keep their probabilities
    and all other tokens together form one more class. The gradient goes to `logits` alone."""
    if logits.dim() != 2:
        flat = _flat_teacher(logits, teacher_ids, teacher_logits, teacher_lse, weights)
        return distill_loss(*flat, softcap, temperature).view(logits.shape[:-1])
    if use_native(logits):
        return _kernel("distill_loss", logits, teacher_ids, teacher_logits, teacher_lse, weights, softcap, temperature)
    return _DistillRef.apply(*_checked_teacher(logits, teacher_ids, teacher_logits, teacher_lse, weights, softcap,
                                               temperature))


def distill_loss_grad(logits, teacher_ids, teacher_logits, teacher_lse=None, weights=None, softcap=None,
                      temperature=1.0, out=None):
    """(distill_loss [...], gradient of its sum [..., V]) in one call. `out` takes the gradient; it may
    be `logits` itself, and must not overlap it otherwise (a graph that has saved the overwritten values
    refuses its backward pass, as after any PyTorch operator in place)."""
    if logits.dim() != 2:
        flat = _flat_teacher(logits, teacher_ids, teacher_logits, teacher_lse, weights)
        loss, dx = distill_loss_grad(*flat, softcap, temperature, _out_rows(out, logits))
        return loss.view(logits.shape[:-1]), dx.view(logits.shape) if out is None else out
    if use_native(logits):
        loss, dx = _kernel("distill_grad", logits, teacher_ids, teacher_logits, teacher_lse, weights, softcap, temperature,
                                         out)
        return loss, dx if out is None else out
    args = _checked_teacher(logits, teacher_ids, teacher_logits, teacher_lse, weights, softcap, temperature)
    _out_rows(out, logits)
    with torch.no_grad():
        loss, dx = distill_ref(*args)
        return loss, dx if out is None else out.copy_(dx)


# ------------------------------------------------------------------------- preference pairs
class _PreferenceRef(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logps, ref, cu, kind, beta, smooth):
        loss, rewards, grad = preference_ref(logps, ref, cu, kind, beta, smooth)
        ctx.save_for_backward(grad, cu)
        ctx.dtype = logps.dtype
        ctx.mark_non_differentiable(rewards)
        return loss, rewards

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, g, _):
        grad, cu = ctx.saved_tensors
        cu = torch.cummax(cu.long(), 0)[0].clamp(0, grad.numel())
        pair = torch.searchsorted(cu, torch.arange(grad.numel(), device=grad.device), right=True) - 1
        g = torch.nn.functional.pad(g.repeat_interleave(2), (1, 1))[pair + 1]
        return (grad * g).to(ctx.dtype), None, None, None, None, None


def _check_tokens(logps, ref_logps):
    if logps.dim() != 1 or not logps.is_floating_point():
        raise ValueError(f"log-probabilities [tokens] are needed, got {logps.dtype} of shape {tuple(logps.shape)}")
    _per_row(ref_logps, logps.shape, "ref_logps")


def preference_loss(logps, ref_logps, cu_seqlens, beta=0.1, label_smoothing=0.0, kind="sigmoid"):
    """(loss [P], rewards [P, 2]) of P pairs of packed sequences.

    logps [T]: the policy's token log-probabilities (token_logprobs; 0 at untrained tokens), ref_logps [T]:
    the reference policy's, or None for a reference-free loss. cu_seqlens [2 P + 1]: the sequences'
    offsets, chosen and rejected in turn, non-decreasing from 0 to T at most; an empty sequence sums to 0.
    rewards: beta times each sequence's summed log ratio (chosen, rejected), without a gradient.
    kind: "sigmoid" (with label_smoothing, the share of wrong labels), "hinge" or "ipo"."""
    kind, beta, smooth = _pair_args(beta, label_smoothing, kind)
    if use_native(logps):
        return tuple(_kernel("preference_loss", logps, ref_logps, cu_seqlens, kind, beta, smooth))
    _check_tokens(logps, ref_logps)
    _check_offsets(cu_seqlens)
    return _PreferenceRef.apply(logps, ref_logps, cu_seqlens, kind, beta, smooth)


def _mean_scale(scale, cu_seqlens):
    return 1.0 / max(1, cu_seqlens.numel() // 2) if scale is None else float(scale)


def preference_loss_grad(logps, ref_logps, cu_seqlens, beta=0.1, label_smoothing=0.0, kind="sigmoid", scale=None):
    """(loss [P], rewards [P, 2], scale * gradient of sum(loss) in logps [T]); scale None is 1 / P, the
    mean over the pairs."""
    kind, beta, smooth = _pair_args(beta, label_smoothing, kind)
    if use_native(logps):
        return tuple(_kernel("preference_pairs", logps, ref_logps, cu_seqlens, kind, beta, smooth, scale, None))
    _check_tokens(logps, ref_logps)
    _check_offsets(cu_seqlens)
    with torch.no_grad():
        return preference_ref(logps, ref_logps, cu_seqlens, kind, beta, smooth, _mean_scale(scale, cu_seqlens))


def preference_logits_grad(logits, targets, ref_logps, cu_seqlens, beta=0.1, label_smoothing=0.0, kind="sigmoid",
                           scale=None, softcap=None, out=None):
    """From the logits [T, V] of packed sequences (see preference_loss) and their targets [T] (-100
    untrained, the reference's value there is not read) to (loss [P], rewards [P, 2], logps [T],
    scale * gradient of sum(loss) in the logits [T, V]). `out` as in distill_loss_grad."""
    kind, beta, smooth = _pair_args(beta, label_smoothing, kind)
    if use_native(logits):
        loss, rewards, logps, dx = _kernel("preference_logits", logits, targets, ref_logps, cu_seqlens, kind, beta, smooth,
                                                              scale, softcap, out)
        return loss, rewards, logps, dx if out is None else out
    if logits.dim() != 2:
        raise ValueError(f"logits [tokens, V] are needed, got shape {tuple(logits.shape)}")
    x, cap = _rows(logits), _cap(softcap)
    t = _targets(targets, x.shape[:1])
    _per_row(ref_logps, x.shape[:1], "ref_logps")
    _out_rows(out, logits)
    _check_offsets(cu_seqlens)
    with torch.no_grad():
        logps, grad = token_logprobs_ref(x, t, cap)
        loss, rewards, g = preference_ref(logps, ref_logps, cu_seqlens, kind, beta, smooth,
                                          _mean_scale(scale, cu_seqlens), t)
        dx = grad(g)
        return loss, rewards, logps, dx if out is None else out.copy_(dx)
