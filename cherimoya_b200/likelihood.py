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
from torch.autograd import forward_ad
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


def _fail(text):
    raise RuntimeError("cherimoya_b200: " + text)


_compiled = torch.compiler.is_compiling
_transforms = torch._C._are_functorch_transforms_active


def _check_reverse(t, name):
    """Refuses tangents of forward mode and the tensors of torch.func's transforms: the formulas
    run on the tensor's memory and would drop them without a word. A tensor that is traced shows
    neither, so there an open dual level or an active transform is refused."""
    if forward_ad._current_level < 0 and not _transforms():
        return
    if _compiled() or torch._C._functorch.is_functorch_wrapped_tensor(t) or \
            forward_ad.unpack_dual(t).tangent is not None:
        _fail("{} must be a plain tensor: forward-mode derivatives and torch.func transforms are "
              "not supported".format(name))


def _check_constant(t, name):
    _check_reverse(t, name)
    if t.requires_grad and torch.is_grad_enabled():
        _fail("{} takes no gradient: detach it".format(name))


@functools.lru_cache(maxsize=1024)
def _check_shape(shape, groups):
    """The shape of the per-row results; groups: None, or a tuple."""
    if groups is None:
        if len(shape) < 1:
            _fail("logits need at least one axis")
        lead, largest = shape[:-1], shape[-1]
    else:
        if len(shape) != 3:
            _fail("logits with signal_groups must be (N, n_outputs, W), got {}".format(
                tuple(shape)))
        _validate_signal_groups(list(groups))
        if sum(groups) != shape[1]:
            _fail("signal_groups {} do not add up to the {} channels of the logits".format(
                list(groups), shape[1]))
        lead, largest = (shape[0], len(groups)), max(groups) * shape[2]
    if largest > MAX_ENTRIES:
        _fail("a row has {} cells; at most {} are supported".format(largest, MAX_ENTRIES))
    return tuple(lead)


def _check(logits, mask, signal_groups, temperature):
    """(groups as a tuple, empty for none; the mask in the logits' shape; the rows' shape; the
    temperature as a number)"""
    if not isinstance(logits, torch.Tensor) or logits.dtype not in _DTYPES:
        _fail("logits must be a float32, bfloat16 or float16 tensor, got {}".format(
            getattr(logits, "dtype", type(logits).__name__)))
    _check_reverse(logits, "logits")
    groups = None if signal_groups is None else tuple(signal_groups)
    lead = _check_shape(logits.shape, groups)
    if isinstance(temperature, torch.Tensor):
        _check_constant(temperature, "temperature")
        temperature = float(temperature.detach())
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
    return groups or (), mask, lead, temperature


def _check_list(t, name, lead, device):
    if t.dtype not in (torch.int64, torch.int32):
        _fail("{} must be int64 or int32, got {}".format(name, t.dtype))
    if t.dim() != len(lead) + 1 or t.shape[:-1] != lead:
        _fail("{} must have the shape {} + (count,), got {}".format(name, lead, tuple(t.shape)))
    if t.device != device:
        _fail("{} must be on the logits' device".format(name))
    if t.shape[-1] > MAX_TARGETS:
        _fail("{} has {} entries per row; at most {} are supported".format(
            name, t.shape[-1], MAX_TARGETS))
    return t if t.dtype == torch.int64 and t.is_contiguous() else t.long().contiguous()


# ------------------------------------------------------------ CPU formulas
def _lead_rows(x):
    n = 1
    for extent in x.shape[:-1]:
        n *= extent
    return n


def _cpu_rows(logits, mask, groups):
    """Rows padded to the widest group, example by example: logits (R, V) fp32 with -inf where
    no entry takes part, and each row's size."""
    z = logits.detach().float()
    if mask is not None:
        z = z.masked_fill(~mask, float("-inf"))
    width = z.shape[-1]
    sizes = [g * width for g in groups] or [width]
    n = z.shape[0] if groups else _lead_rows(z)
    out = torch.full((n, len(sizes), max(sizes)), float("-inf"))
    first = 0
    for i, size in enumerate(sizes):
        if groups:
            part = z[:, first:first + groups[i]].reshape(n, size)
            first += groups[i]
        else:
            part = z.reshape(n, size)
        out[:, i, :size] = part
    return (out.reshape(n * len(sizes), max(sizes)),
            torch.tensor(sizes).expand(n, -1).reshape(-1))


def _cpu_write(logits, rows, groups):
    """A gradient of the logits' shape and type from padded rows."""
    width = logits.shape[-1]
    if not groups:
        return rows.reshape(logits.shape).to(logits.dtype)
    n = logits.shape[0]
    rows = rows.reshape(n, len(groups), rows.shape[-1])
    parts = [rows[:, i, :g * width].reshape(n, g, width) for i, g in enumerate(groups)]
    return torch.cat(parts, 1).to(logits.dtype)


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


def _cpu_log_probs(logits, mask, groups, targets, top_k, temperature):
    z, sizes = _cpu_rows(logits, mask, groups)
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


def _cpu_log_probs_backward(logits, mask, groups, targets, top_indices, stats, entropy, g_lp, g_h,
                            g_norm, g_top, temperature):
    z, sizes = _cpu_rows(logits, mask, groups)
    R = z.shape[0]
    m, log_s = stats[:, :1], stats[:, 1:]
    lists = [(i.reshape(R, i.shape[-1]), g.reshape(R, i.shape[-1]))
             for i, g in ((targets, g_lp), (top_indices, g_top)) if g is not None]
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
        at = torch.zeros(z.shape, dtype=torch.float64).scatter_add_(
            -1, idx.clamp(0, z.shape[1] - 1), torch.where((idx < 0) | past, 0.0, g).double())
        d = d + at.float()
    return _cpu_write(logits, torch.where(z == float("-inf"), 0.0, d / temperature), groups)


def _cpu_distill(logits, mask, groups, idx, t_lp, renormalize, weight, scale, upstream,
                 want_grad, temperature):
    z, sizes = _cpu_rows(logits, mask, groups)
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
    grad = None
    if want_grad:
        q_r = torch.exp(log_r - log_all)
        d = torch.where(rest, e.double() / s.double(), 0.0) * (q_r - p_r)
        d = torch.where(listed, el / norm - p, d) * (w * temperature)
        d = torch.where(live, d, 0.0)
        d = torch.where(bad, float("nan"), d)
        d = torch.where(skip | (z == -inf), 0.0, d)
        grad = _cpu_write(logits, d, groups)
    return loss.float().reshape(R), grad


# ------------------------------------------------------------ dispatch
def _run_log_probs(logits, mask, groups, lead, targets, top_k, temperature, want_stats):
    if logits.is_cuda:
        from . import ops
        fn = ops.log_probs if _compiled() else ops.log_probs_impl
        return fn(logits, mask, groups, targets, top_k, temperature, want_stats)
    out = _cpu_log_probs(logits, mask, groups, targets, top_k, temperature)
    shapes = (lead + (targets.shape[-1],), lead, lead, lead + (top_k,), lead + (top_k,))
    return tuple(o.reshape(s) for o, s in zip(out, shapes)) + (out[5],)


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, groups, lead, targets, top_k, temperature):
        lp, h, norm, top, at, stats = _run_log_probs(logits, mask, groups, lead, targets, top_k,
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
        gs = [g if g is None or g.is_contiguous() else g.contiguous()
              for g in (g_lp, g_h, g_norm, g_top)]
        if not logits.is_cuda:
            fn = _cpu_log_probs_backward
        else:
            from . import ops
            fn = ops.log_probs_backward if _compiled() else ops.log_probs_backward_impl
        grad = fn(logits, mask, groups, targets, at, stats, h, *gs, temperature)
        return grad, None, None, None, None, None, None


def profile_log_probs(logits, targets=None, *, top_k=0, mask=None, signal_groups=None,
                      temperature=1.0):
    """Log probabilities of given cells, entropy and most likely cells of every row.

    logits: float32, bfloat16 or float16, (N, n_outputs, W) with
    ``signal_groups``, else (..., V). targets: None or int64/int32
    (*lead, S), S up to 1024; a negative index is an empty place (log
    probability 0, no gradient), one past the row answers NaN, a cell that
    does not take part -inf (no gradient). top_k: up to 128 cells, the most
    likely first, equal logits by ascending index; places without a cell hold
    -inf and index -1. temperature, a number, divides the logits.

    Returns ``ProfileLogProbs``; all but ``top_indices`` are differentiable
    with respect to the logits (once, in reverse mode; forward mode and the
    transforms of ``torch.func`` are refused).
    """
    groups, mask, lead, temperature = _check(logits, mask, signal_groups, temperature)
    if isinstance(top_k, bool) or not isinstance(top_k, int) or not 0 <= top_k <= MAX_TOP:
        raise ValueError("top_k must be an int between 0 and {}, got {!r}".format(MAX_TOP, top_k))
    if targets is None:
        targets = torch.empty(lead + (0,), dtype=torch.int64, device=logits.device)
    else:
        targets = _check_list(targets, "targets", lead, logits.device)
    if logits.requires_grad and torch.is_grad_enabled():
        return ProfileLogProbs(*_LogProbs.apply(logits, mask, groups, lead, targets, top_k,
                                                temperature))
    return ProfileLogProbs(*_run_log_probs(logits, mask, groups, lead, targets, top_k,
                                           temperature, False)[:5])


# ------------------------------------------------------------ distillation
def _run_distill(logits, mask, groups, lead, idx, t_lp, renormalize, weight, scale, upstream,
                 want_losses, reduce, want_grad, temperature):
    """(per-row losses, their sum, gradient: what is asked for)"""
    if logits.is_cuda:
        from . import ops
        fn = ops.distill if _compiled() else ops.distill_impl
        return fn(logits, mask, groups, idx, t_lp, renormalize, weight, scale, upstream,
                  want_losses, reduce, want_grad, temperature)
    rows, grad = _cpu_distill(logits, mask, groups, idx, t_lp, renormalize, weight, scale,
                              upstream, want_grad, temperature)
    return rows.reshape(lead), rows.double().sum().float() if reduce else None, grad


class _Distill(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, mask, groups, lead, idx, t_lp, renormalize, weight, scale, reduce,
                temperature):
        rows, loss, _ = _run_distill(logits, mask, groups, lead, idx, t_lp, renormalize, weight,
                                     scale, None, not reduce, reduce, False, temperature)
        ctx.save_for_backward(logits, mask, idx, t_lp, weight)
        ctx.how = (groups, lead, renormalize, scale, temperature)
        return loss if reduce else rows

    @staticmethod
    @once_differentiable
    def backward(ctx, g):
        logits, mask, idx, t_lp, weight = ctx.saved_tensors
        groups, lead, renormalize, scale, temperature = ctx.how
        if not g.is_contiguous():
            g = g.contiguous()
        grad = _run_distill(logits, mask, groups, lead, idx, t_lp, renormalize, weight, scale, g,
                            False, False, True, temperature)[2]
        return grad, None, None, None, None, None, None, None, None, None, None


def _check_distill(logits, indices, log_probs, mask, signal_groups, temperature, weight,
                   reduction):
    groups, mask, lead, temperature = _check(logits, mask, signal_groups, temperature)
    if reduction not in ("mean", "sum", "none"):
        raise ValueError("reduction must be 'mean', 'sum' or 'none', got {!r}".format(reduction))
    device = logits.device
    indices = _check_list(indices, "teacher_indices", lead, device)
    if log_probs.shape != indices.shape or not log_probs.is_floating_point():
        _fail("teacher_log_probs must be floating and of teacher_indices' shape {}".format(
            tuple(indices.shape)))
    if weight is not None and (weight.shape != lead or not weight.is_floating_point()):
        _fail("weight must be floating and of shape {}, got {}".format(
            lead, tuple(weight.shape)))
    log_probs = _constant(log_probs, "teacher_log_probs", device)
    if weight is not None:
        weight = _constant(weight, "weight", device)
    rows = 1
    for extent in lead:
        rows *= extent
    scale = 1.0 / rows if reduction == "mean" and rows else 1.0
    return groups, mask, lead, temperature, indices, log_probs, weight, scale


def _constant(t, name, device):
    """t in fp32 and contiguous; it carries no gradient."""
    if t.device != device:
        _fail("{} must be on the logits' device".format(name))
    _check_constant(t, name)
    if t.requires_grad:
        t = t.detach()
    return t if t.dtype == torch.float32 and t.is_contiguous() else t.float().contiguous()


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
    fp32 and differentiable with respect to the logits (once, in reverse mode;
    forward mode and the transforms of ``torch.func`` are refused).
    """
    groups, mask, lead, temperature, idx, t_lp, weight, scale = _check_distill(
        logits, teacher_indices, teacher_log_probs, mask, signal_groups, temperature, weight,
        reduction)
    reduce, renormalize = reduction != "none", bool(renormalize)
    if logits.requires_grad and torch.is_grad_enabled():
        return _Distill.apply(logits, mask, groups, lead, idx, t_lp, renormalize, weight, scale,
                              reduce, temperature)
    rows, loss, _ = _run_distill(logits, mask, groups, lead, idx, t_lp, renormalize, weight, scale,
                                 None, not reduce, reduce, False, temperature)
    return loss if reduce else rows


def distillation_loss_and_grad(logits, teacher_indices, teacher_log_probs, *, renormalize=False,
                               mask=None, signal_groups=None, temperature=1.0, weight=None,
                               reduction="mean"):
    """``distillation_loss`` and its gradient in one pass over the logits.

    Takes the same arguments and returns (loss, gradient with respect to the
    logits, in their shape and type); with reduction 'none' the gradient is
    that of the losses' sum. Neither carries an autograd graph: continue with
    ``logits.backward(grad)``. What multiplies the loss goes into ``weight``.
    """
    groups, mask, lead, temperature, idx, t_lp, weight, scale = _check_distill(
        logits, teacher_indices, teacher_log_probs, mask, signal_groups, temperature, weight,
        reduction)
    reduce = reduction != "none"
    rows, loss, grad = _run_distill(logits, mask, groups, lead, idx, t_lp, bool(renormalize),
                                    weight, scale, None, not reduce, reduce, True, temperature)
    return (loss if reduce else rows), grad
