"""Likelihood and distillation on profile logits.

A profile's logits are one categorical distribution per example and signal
group: a joint softmax over the group's channels and positions (as in
``ExpectedCountsWrapper``). ``profile_log_probs`` gives the log probabilities
of given cells (reads, cut sites), the entropy and the most likely cells;
``distillation_loss`` trains a student on a teacher's most likely cells, which
``TopCellsWrapper`` writes for a whole data set through ``predict``.

Layout. With ``signal_groups`` the logits are (N, n_outputs, W), as the model
returns them, and the row of example n and group g holds the group's channels
one after the other: cell ``c * W + w`` is position w of the group's channel c.
Per-row results have the leading shape (N, n_groups). Without it every vector
along the last axis is a row, and per-row results have the remaining shape.

Cells that take part. ``mask`` (bool, broadcastable to the logits) is True
where a cell takes part; masked cells and cells whose logit is -inf have
probability 0 whatever they hold, and gradient 0. A row with no cell left has
log normaliser -inf, entropy 0, loss 0 and gradient 0. A row with NaN or +inf
among its cells has no distribution: it answers NaN, and index -1.

Dispatch. CUDA logits run the sm_100a kernels (one launch per call up to 64
groups, and one more for a reduced loss), with or without gradients, and
raise if the library is missing. CPU logits run the same formulas in PyTorch.
Sums, maxima and log probabilities are fp32; a teacher's masses and the loss
of a row are formed in 64 bits; the gradient is rounded once to the logits'
type. Nothing is summed by atomics: the same call gives the same bits.

Under CUDA graph capture, capture a training step whole. A backward pass that
is captured while an eager graph of the same leaves is alive is not safe in
autograd itself; ``distillation_loss_and_grad`` needs no autograd.
"""

import functools
from typing import NamedTuple

import torch
from torch.autograd.function import once_differentiable

from .model import _validate_signal_groups

MAX_ENTRIES = 1 << 20      # cells of one row
MAX_TARGETS = 1024         # given or listed cells per row
MAX_TOP = 128              # top cells per row
_DTYPES = (torch.float32, torch.bfloat16, torch.float16)
_MIN_T, _MAX_T = 1.0 / 1024.0, 1024.0


class ProfileLogProbs(NamedTuple):
    """What ``profile_log_probs`` returns; ``lead`` is the rows' shape."""
    log_probs: torch.Tensor        # (*lead, S) fp32
    entropy: torch.Tensor          # lead, fp32, in nats
    log_normalizer: torch.Tensor   # lead, fp32
    top_log_probs: torch.Tensor    # (*lead, top_k) fp32
    top_indices: torch.Tensor      # (*lead, top_k) int64


class _Layout(NamedTuple):
    """Where the rows are: n examples, per group its first element and its size."""
    lead: tuple
    n: int
    stride: int
    offsets: tuple
    sizes: tuple


def _fail(text):
    raise RuntimeError("cherimoya_b200: " + text)


@functools.lru_cache(maxsize=256)
def _group_layout(groups, width, channel_stride):
    _validate_signal_groups(list(groups))
    offsets, first = [], 0
    for g in groups:
        offsets.append(first * channel_stride)
        first += g
    return tuple(offsets), tuple(g * width for g in groups)


def _place(x, groups):
    """(x, or a contiguous copy where its strides have no such rows; its layout)."""
    if groups is None:
        width, lead = x.shape[-1], tuple(x.shape[:-1])
        if x.dim() != 2:
            x = x.reshape(_numel(lead), width)
        if width > 1 and x.stride(1) != 1:
            x = x.contiguous()
        return x, _Layout(lead, x.shape[0], x.stride(0), (0,), (width,))
    n, _, width = x.shape
    whole = all(g == 1 for g in groups)
    if (width > 1 and x.stride(2) != 1) or not (whole or x.stride(1) == width):
        x = x.contiguous()
    offsets, sizes = _group_layout(groups, width, x.stride(1))
    return x, _Layout((n, len(groups)), n, x.stride(0), offsets, sizes)


def _numel(shape):
    n = 1
    for s in shape:
        n *= s
    return n


def _check(logits, mask, signal_groups, temperature):
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES:
        _fail("logits must be a float32, bfloat16 or float16 tensor, got {}".format(
            getattr(logits, "dtype", type(logits).__name__)))
    groups = None
    if signal_groups is not None:
        groups = tuple(signal_groups)
        if logits.dim() != 3:
            _fail("logits with signal_groups must be (N, n_outputs, W), got {}".format(
                tuple(logits.shape)))
        _group_layout(groups, 1, 1)
        if sum(groups) != logits.shape[1]:
            _fail("signal_groups {} do not add up to the {} channels of the logits".format(
                list(groups), logits.shape[1]))
        largest = max(groups) * logits.shape[2]
    else:
        if logits.dim() < 1:
            _fail("logits need at least one axis")
        largest = logits.shape[-1]
    if largest > MAX_ENTRIES:
        _fail("a row has {} cells; at most {} are supported".format(largest, MAX_ENTRIES))
    if not _MIN_T <= temperature <= _MAX_T:
        raise ValueError("temperature must be between 1/1024 and 1024, got {!r}".format(
            temperature))
    if mask is not None:
        if mask.dtype != torch.bool:
            _fail("mask must be a bool tensor, True where a cell takes part")
        if mask.device != logits.device:
            _fail("mask must be on the logits' device")
        if mask.shape != logits.shape:
            try:
                mask = mask.expand(logits.shape)
            except RuntimeError:
                _fail("mask of shape {} does not broadcast to the logits' {}".format(
                    tuple(mask.shape), tuple(logits.shape)))
    return groups, mask


def _check_list(t, name, lead, device, count):
    if t.dtype not in (torch.int64, torch.int32):
        _fail("{} must be int64 or int32, got {}".format(name, t.dtype))
    if tuple(t.shape[:-1]) != lead or t.dim() != len(lead) + 1:
        _fail("{} must have the shape {} + (count,), got {}".format(name, lead, tuple(t.shape)))
    if t.device != device:
        _fail("{} must be on the logits' device".format(name))
    if t.shape[-1] > MAX_TARGETS:
        _fail("{} has {} entries per row; at most {} are supported".format(
            name, t.shape[-1], MAX_TARGETS))
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.long().contiguous()


# ------------------------------------------------------------ CPU formulas
def _cpu_rows(z, mask, lay, temperature):
    """Rows padded to the widest group: logits (R, V) fp32 with -inf outside, in example order."""
    width = max(lay.sizes, default=0)
    out = torch.full((lay.n, len(lay.sizes), width), float("-inf"), dtype=torch.float32)
    for g, (o, s) in enumerate(zip(lay.offsets, lay.sizes)):
        v = torch.as_strided(z, (lay.n, s), (lay.stride, 1), z.storage_offset() + o).float()
        if mask is not None:
            m, ml = mask
            v = v.masked_fill(~torch.as_strided(m, (lay.n, s), (ml.stride, 1),
                                                m.storage_offset() + ml.offsets[g]),
                              float("-inf"))
        out[:, g, :s] = v
    sizes = torch.tensor(lay.sizes).expand(lay.n, -1).reshape(-1)
    return out.reshape(lay.n * len(lay.sizes), width), sizes


def _cpu_write(grad, rows, glay):
    rows = rows.reshape(glay.n, len(glay.sizes), rows.shape[-1])
    for g, (o, s) in enumerate(zip(glay.offsets, glay.sizes)):
        torch.as_strided(grad, (glay.n, s), (glay.stride, 1),
                         grad.storage_offset() + o).copy_(rows[:, g, :s])


def _cpu_max(z):
    if z.shape[1] == 0:
        return z.new_zeros(z.shape[0], 1)
    m = torch.where(torch.isnan(z), float("-inf"), z).amax(-1, keepdim=True)
    return torch.where(m == float("-inf"), 0.0, m)


def _cpu_gather(z, idx, sizes):
    """(logits at idx, -inf where there is none; which indices lie past the row)"""
    past = idx >= sizes[:, None]
    if z.shape[1] == 0:
        return torch.full(idx.shape, float("-inf")), past
    got = z.gather(-1, idx.clamp(0, z.shape[1] - 1))
    return torch.where((idx < 0) | past, float("-inf"), got), past


def _cpu_log_probs(z, mask, lay, targets, top_k, temperature):
    z, sizes = _cpu_rows(z, mask, lay, temperature)
    R = z.shape[0]
    m = _cpu_max(z)
    x = (z - m) / temperature
    e = torch.exp(x)
    s = e.sum(-1, keepdim=True)
    log_s = torch.log(s)
    x = torch.where(x == float("-inf"), 0.0, x)
    h = torch.where(s == 0, 0.0, log_s - (e * x).sum(-1, keepdim=True) / s).reshape(R)
    bad = torch.isnan(s)
    t = targets.reshape(R, targets.shape[-1])
    zt, past = _cpu_gather(z, t, sizes)
    lp = torch.where(zt == float("-inf"), zt, (zt - m) / temperature - log_s)
    lp = torch.where(bad | past, float("nan"), lp)
    lp = torch.where(t < 0, 0.0, lp)
    k = min(top_k, z.shape[1])
    top, at = torch.sort(torch.where(bad, float("-inf"), z), dim=-1, descending=True, stable=True)
    top, at = top[:, :k], at[:, :k]
    none = top == float("-inf")
    at = torch.where(none, -1, at)
    top = torch.where(none, top, (top - m) / temperature - log_s)
    top = torch.nn.functional.pad(top, (0, top_k - k), value=float("-inf"))
    at = torch.nn.functional.pad(at, (0, top_k - k), value=-1)
    top = torch.where(bad, float("nan"), top)
    stats = torch.cat([m, log_s], -1)
    return lp, h, (m / temperature + log_s).reshape(R), top, at, stats


def _cpu_log_probs_backward(z, mask, lay, targets, top_indices, stats, entropy, g_lp, g_h, g_norm,
                            g_top, temperature, grad, glay):
    z, sizes = _cpu_rows(z, mask, lay, temperature)
    R = z.shape[0]
    m, log_s = stats[:, :1], stats[:, 1:]
    lists = [(i.reshape(R, i.shape[-1]), g.reshape(R, i.shape[-1])) for i, g in ((targets, g_lp), (top_indices, g_top))
             if g is not None]
    idx = torch.cat([i for i, _ in lists], -1) if lists else torch.empty(R, 0, dtype=torch.int64)
    g = torch.cat([x for _, x in lists], -1) if lists else torch.empty(R, 0)
    zt, past = _cpu_gather(z, idx, sizes)
    g = torch.where(past, float("nan"), torch.where(zt == float("-inf"), 0.0, g))
    a = -g.sum(-1, keepdim=True)
    if g_norm is not None:
        a = a + g_norm.reshape(R, 1)
    lq = (z - m) / temperature - log_s
    q = torch.exp(lq)
    d = q * a
    if g_h is not None:
        d = d - torch.where(q > 0, q * (lq + entropy.reshape(R, 1)), 0.0) * g_h.reshape(R, 1)
    if idx.shape[1] and z.shape[1]:
        d.scatter_add_(-1, idx.clamp(0, z.shape[1] - 1),
                       torch.where((idx < 0) | past, 0.0, g))
    _cpu_write(grad, torch.where(z == float("-inf"), 0.0, d / temperature), glay)


def _cpu_distill(z, mask, lay, idx, t_lp, renormalize, weight, scale, upstream, temperature, grad,
                 glay):
    z, sizes = _cpu_rows(z, mask, lay, temperature)
    R, V = z.shape
    inf = float("inf")
    w = torch.ones(R, 1) if weight is None else weight.reshape(R, 1)
    skip = w == 0
    w = w.double() * scale
    if upstream is not None:
        w = w * upstream.reshape(-1, 1).double()
    zu, past = _cpu_gather(z, idx.reshape(R, idx.shape[-1]), sizes)
    idx = idx.reshape(R, idx.shape[-1]).clamp(0, max(V - 1, 0))
    there = zu != -inf
    lp = t_lp.reshape(R, t_lp.shape[-1]).double()
    bad = (past | (there & ~(lp < inf))).any(-1, keepdim=True)
    lp = torch.where(there, lp, -inf)
    if renormalize and idx.shape[1]:
        top = lp.amax(-1, keepdim=True)
        lp = lp - torch.where(torch.isfinite(top), top, 0.0)
    # on the row itself: the teacher's mass of every entry, and which are listed
    mass = torch.zeros(R, V, dtype=torch.float64)
    listed = torch.zeros(R, V, dtype=torch.bool)
    if V and idx.shape[1]:
        mass.scatter_add_(-1, idx, torch.exp(lp))
        listed = torch.zeros(R, V, dtype=torch.int32).scatter_add_(-1, idx, there.int()) > 0
    total = mass.sum(-1, keepdim=True)
    zr = torch.where(listed, -inf, z)
    zl = torch.where(listed, z, -inf).double()
    m = _cpu_max(zr)
    e = torch.exp((zr - m) / temperature)
    s = e.sum(-1, keepdim=True)
    rest = s != 0
    big = torch.maximum(torch.where(rest, m, -inf).double(), _cpu_max(zl)) if V else m.double()
    big = torch.where(rest | listed.any(-1, keepdim=True), big, 0.0)
    bad |= torch.isnan(s)
    el = torch.exp((zl - big) / temperature)
    log_r = torch.where(rest, (m.double() - big) / temperature + torch.log(s.double()), -inf)
    norm = el.sum(-1, keepdim=True) + torch.exp(log_r)
    bad |= torch.isnan(norm)
    log_all = torch.log(norm)
    whole = (total > 1) | ~rest | bool(renormalize)
    p = torch.where(whole & (total > 0), mass / total, mass)
    p_r = torch.where(whole, 0.0, 1.0 - total)
    live = (norm > 0) & ((total > 0) | ~whole)
    logq = torch.where(listed, (zl - big) / temperature - log_all, 0.0)
    loss = torch.where(p > 0, p * (torch.log(p) - logq), 0.0).sum(-1, keepdim=True)
    loss = loss + torch.where(p_r > 0, p_r * (torch.log(p_r) - (log_r - log_all)), 0.0)
    loss = torch.where(live, loss, 0.0) * temperature ** 2 * w
    loss = torch.where(bad, float("nan"), loss)
    loss = torch.where(skip, 0.0, loss)
    if grad is not None:
        q_r = torch.exp(log_r - log_all)
        d = torch.where(rest, e.double() / s.double(), 0.0) * (q_r - p_r)
        d = torch.where(listed, el / norm - p, d) * (w * temperature)
        d = torch.where(live, d, 0.0)
        d = torch.where(bad, float("nan"), d)
        d = torch.where(skip | (z == -inf), 0.0, d)
        _cpu_write(grad, d.to(grad.dtype), glay)
    return loss.float().reshape(R)


# ------------------------------------------------------------ dispatch
def _compiled():
    return torch.compiler.is_compiling()


def _grad_layout(shape, groups):
    """(row stride, group offsets) of a contiguous tensor of the logits' shape."""
    if groups is None:
        return shape[-1], (0,)
    return shape[1] * shape[2], _group_layout(groups, shape[2], shape[2])[0]


def _run_log_probs(logits, mask, groups, targets, top_k, temperature, want_stats):
    z, lay = _place(logits, groups)
    m, ml = _place(mask, groups) if mask is not None else (None, lay)
    if not z.is_cuda:
        out = _cpu_log_probs(z, m if m is None else (m, ml), lay, targets, top_k, temperature)
        lead = [lay.lead + (targets.shape[-1],), lay.lead, lay.lead, lay.lead + (top_k,),
                lay.lead + (top_k,)]
        return tuple(o.reshape(s) for o, s in zip(out, lead)) + (out[5],)
    from . import ops
    fn = ops.log_probs if _compiled() else ops.log_probs_impl
    return fn(z, m, lay.lead, lay.n, lay.stride, lay.offsets, lay.sizes, ml.stride, ml.offsets,
              targets, top_k, temperature, want_stats)


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, groups, targets, top_k, temperature):
        lp, h, norm, top, at, stats = _run_log_probs(logits, mask, groups, targets, top_k,
                                                     temperature, True)
        ctx.save_for_backward(logits, mask, targets, at, stats, h)
        ctx.how = (groups, temperature)
        ctx.mark_non_differentiable(at)
        ctx.set_materialize_grads(False)
        return lp, h, norm, top, at

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_h, g_norm, g_top, _):
        logits, mask, targets, at, stats, h = ctx.saved_tensors
        groups, temperature = ctx.how
        z, lay = _place(logits, groups)
        m, ml = _place(mask, groups) if mask is not None else (None, lay)
        gs = [None if g is None else g.contiguous() for g in (g_lp, g_h, g_norm, g_top)]
        if z.is_cuda:
            from . import ops
            fn = ops.log_probs_backward if _compiled() else ops.log_probs_backward_impl
            grad = fn(z, m, logits.shape, lay.n, lay.stride, lay.offsets, lay.sizes, ml.stride,
                      ml.offsets, *_grad_layout(logits.shape, groups), targets, at, stats, h, *gs,
                      temperature)
        else:
            grad = torch.empty(logits.shape, dtype=logits.dtype)
            _cpu_log_probs_backward(z, m if m is None else (m, ml), lay, targets, at, stats, h,
                                    *gs, temperature, *_place(grad, groups))
        return grad, None, None, None, None, None


def profile_log_probs(logits, targets=None, *, top_k=0, mask=None, signal_groups=None,
                      temperature=1.0):
    """Log probabilities of given cells, entropy and most likely cells of every row.

    logits: float32, bfloat16 or float16, (N, n_outputs, W) with
    ``signal_groups``, else (..., V). targets: None or int64/int32
    (*lead, S), S up to 1024; a negative index is an empty place (log
    probability 0, no gradient), one past the row answers NaN, a cell that
    does not take part -inf (no gradient). top_k: up to 128 cells, the most
    likely first, equal logits by ascending index; places without a cell hold
    -inf and index -1. temperature divides the logits.

    Returns ``ProfileLogProbs``; all but ``top_indices`` are differentiable
    with respect to the logits (once).
    """
    groups, mask = _check(logits, mask, signal_groups, temperature)
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 0 <= top_k <= MAX_TOP:
        raise ValueError("top_k must be an int between 0 and {}, got {!r}".format(MAX_TOP, top_k))
    lead = tuple(logits.shape[:-1]) if groups is None else (logits.shape[0], len(groups))
    if targets is None:
        targets = torch.empty(lead + (0,), dtype=torch.int64, device=logits.device)
    else:
        targets = _check_list(targets, "targets", lead, logits.device, MAX_TARGETS)
    if torch.is_grad_enabled() and logits.requires_grad:
        return ProfileLogProbs(*_LogProbs.apply(logits, mask, groups, targets, top_k, temperature))
    return ProfileLogProbs(*_run_log_probs(logits.detach(), mask, groups, targets, top_k,
                                           temperature, False)[:5])


# ------------------------------------------------------------ distillation
def _run_distill(logits, mask, groups, idx, t_lp, renormalize, weight, scale, upstream, reduce,
                 want_grad, temperature):
    """(per-row losses, their sum or None, gradient or None)"""
    z, lay = _place(logits, groups)
    m, ml = _place(mask, groups) if mask is not None else (None, lay)
    if not z.is_cuda:
        grad = torch.empty(logits.shape, dtype=logits.dtype) if want_grad else None
        rows = _cpu_distill(z, m if m is None else (m, ml), lay, idx, t_lp, renormalize, weight,
                            scale, upstream, temperature,
                            *(_place(grad, groups) if want_grad else (None, None)))
        return rows.reshape(lay.lead), rows.double().sum().float() if reduce else None, grad
    from . import ops
    fn = ops.distill if _compiled() else ops.distill_impl
    return fn(z, m, logits.shape, lay.lead, lay.n, lay.stride, lay.offsets, lay.sizes, ml.stride,
              ml.offsets, *_grad_layout(logits.shape, groups), idx, t_lp, renormalize, weight,
              scale, upstream, reduce, want_grad, temperature)


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, groups, idx, t_lp, renormalize, weight, scale, reduce,
                temperature):
        rows, loss, _ = _run_distill(logits, mask, groups, idx, t_lp, renormalize, weight, scale,
                                     None, reduce, False, temperature)
        ctx.save_for_backward(logits, mask, idx, t_lp, weight)
        ctx.how = (groups, renormalize, scale, temperature)
        return loss if reduce else rows

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, mask, idx, t_lp, weight = ctx.saved_tensors
        groups, renormalize, scale, temperature = ctx.how
        _, _, grad = _run_distill(logits, mask, groups, idx, t_lp, renormalize, weight, scale,
                                  g.contiguous(), False, True, temperature)
        return (grad,) + (None,) * 9


def _check_distill(logits, indices, log_probs, mask, signal_groups, temperature, weight,
                   reduction):
    groups, mask = _check(logits, mask, signal_groups, temperature)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be 'mean', 'sum' or 'none', got {!r}".format(reduction))
    lead = tuple(logits.shape[:-1]) if groups is None else (logits.shape[0], len(groups))
    indices = _check_list(indices, "teacher_indices", lead, logits.device, MAX_TARGETS)
    if log_probs.shape != indices.shape or not log_probs.is_floating_point():
        _fail("teacher_log_probs must be floating and of teacher_indices' shape {}".format(
            tuple(indices.shape)))
    if weight is not None:
        if tuple(weight.shape) != lead or not weight.is_floating_point():
            _fail("weight must be floating and of shape {}, got {}".format(
                lead, tuple(weight.shape)))
    for t, name in ((log_probs, "teacher_log_probs"), (weight, "weight")):
        if t is None:
            continue
        if t.device != logits.device:
            _fail("{} must be on the logits' device".format(name))
        if t.requires_grad and torch.is_grad_enabled():
            _fail("{} takes no gradient: detach it".format(name))
    log_probs = log_probs.detach().float().contiguous()
    weight = weight.detach().float().contiguous() if weight is not None else None
    rows = _numel(lead)
    scale = 1.0 / rows if reduction == "mean" and rows else 1.0
    return groups, mask, indices, log_probs, weight, scale


def distillation_loss(logits, teacher_indices, teacher_log_probs, *, renormalize=False, mask=None,
                      signal_groups=None, temperature=1.0, weight=None, reduction="mean"):
    """Cross-distribution loss of a student against a teacher's listed cells.

    teacher_indices (*lead, K) int64/int32 and teacher_log_probs (*lead, K):
    the teacher's most likely cells and their log probabilities at the same
    temperature, as ``profile_log_probs(teacher_logits, top_k=K,
    temperature=temperature)`` or ``TopCellsWrapper`` give them; K up to 1024.
    Per row, with P the teacher's and q the student's probabilities,

        T^2 (sum_u P_u log(P_u / q_u) + P_rest log(P_rest / q_rest))

    where "rest" is the single outcome "none of the listed" with the mass that
    the list leaves. With ``renormalize`` (and where the listed mass exceeds 1,
    or no cell is left outside the list) P is scaled to sum to 1 over the list
    and there is no rest; then any common shift of teacher_log_probs cancels,
    so logits over the temperature do as well. Index -1 is an empty place;
    cells that do not take part are dropped from the list; a cell listed twice
    counts once with both masses; an index past the row makes the row NaN.

    weight (lead): a factor per row; a row of weight 0 is not looked at.
    reduction: 'mean' over all rows, 'sum', or 'none' (lead). The result is
    fp32 and differentiable with respect to the logits (once).
    """
    groups, mask, idx, t_lp, weight, scale = _check_distill(
        logits, teacher_indices, teacher_log_probs, mask, signal_groups, temperature, weight,
        reduction)
    reduce = reduction != "none"
    if torch.is_grad_enabled() and logits.requires_grad:
        out = _Distill.apply(logits, mask, groups, idx, t_lp, bool(renormalize), weight, scale,
                             reduce, temperature)
    else:
        rows, loss, _ = _run_distill(logits.detach(), mask, groups, idx, t_lp, bool(renormalize),
                                     weight, scale, None, reduce, False, temperature)
        out = loss if reduce else rows
    return out


def distillation_loss_and_grad(logits, teacher_indices, teacher_log_probs, *, renormalize=False,
                               mask=None, signal_groups=None, temperature=1.0, weight=None,
                               reduction="mean"):
    """``distillation_loss`` and its gradient in one pass over the logits.

    Takes the same arguments and returns (loss, gradient with respect to the
    logits, in their shape and type); with reduction 'none' the gradient is
    that of the losses' sum. Neither carries an autograd graph: continue with
    ``logits.backward(grad)``. What multiplies the loss goes into ``weight``.
    """
    groups, mask, idx, t_lp, weight, scale = _check_distill(
        logits, teacher_indices, teacher_log_probs, mask, signal_groups, temperature, weight,
        reduction)
    reduce = reduction != "none"
    rows, loss, grad = _run_distill(logits.detach(), mask, groups, idx, t_lp, bool(renormalize),
                                    weight, scale, None, reduce, True, temperature)
    return (loss if reduce else rows), grad
