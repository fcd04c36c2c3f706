"""The cases of the likelihood and distillation tests, run on the device they are given."""

import math

import pytest
import torch

import cherimoya_b200 as cb
import likelihood_common as C

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = math.inf

# (shape, groups, dtype, targets, top_k, temperature, mask)
SCORE = [
    ((1, 1), None, F32, 1, 1, 1.0, None),
    ((3, 2), None, BF16, 2, 3, 1.0, None),
    ((4, 31), None, F16, 3, 5, 0.7, None),
    ((2, 33), None, F32, 0, 40, 1.0, "some"),
    ((5, 127), None, BF16, 4, 0, 2.0, "some"),
    ((3, 1, 1000), [1], F32, 1, 8, 1.0, None),
    ((2, 9, 1000), [1, 2, 2, 2, 2], F32, 17, 16, 1.0, "some"),
    ((2, 4, 501), [3, 1], BF16, 9, 7, 1.5, "channel"),
    ((2, 3, 4), [1, 1, 1], F32, 2, 2, 1.0, None),
    ((2, 3, 7, 65), None, F32, 2, 4, 1.0, None),
    ((77,), None, F32, 2, 4, 1.0, None),
    ((3, 1024), None, F32, 300, 32, 1.0, None),
    ((3, 2047), None, BF16, 2, 128, 1.0, None),
    ((2, 4097), None, F16, 2, 100, 1.0, "some"),
    ((2, 16385), None, BF16, 1, 20, 1.0, None),
    ((2, 50001), None, BF16, 1, 50, 1.0, "some"),
    ((2, 65536), None, F32, 3, 10, 0.5, None),
]
LONG = [
    ((1, 131072 + 3), None, BF16, 1, 64, 1.0, None),
    ((2, 300001), None, F32, 2, 128, 1.0, None),
    ((2, 300001), None, F16, 2, 5, 1.0, "some"),
    ((1, 1 << 20), None, F32, 1, 3, 1.0, None),
    ((1, 1 << 20), None, BF16, 1, 3, 1.0, None),
]


def make_mask(kind, shape, g):
    if kind is None:
        return None
    if kind == "channel":      # broadcast over the channels
        m = torch.rand(shape[0], 1, shape[-1], generator=g) < 0.8
    else:
        m = torch.rand(*shape, generator=g) < 0.8
    m[0] = False               # nothing is left of the first example's rows
    return m


def case_scores(dev, shape, groups, dtype, s, k, T, mask, seed=0):
    z, g = C.logits(shape, dtype, seed)
    t = C.make_targets(shape, groups, s, g)
    m = make_mask(mask, shape, g)
    z, t, m = z.to(dev).requires_grad_(), t.to(dev), m.to(dev) if m is not None else None
    how = dict(top_k=k, mask=m, signal_groups=groups, temperature=T)
    with torch.no_grad():
        out = cb.profile_log_probs(z, t, **how)
    C.check_scores(z, out, t, k, m, groups, T)
    out = cb.profile_log_probs(z, t, **how)
    gs = dict(lp=torch.randn(t.shape, generator=g), h=torch.randn(out.entropy.shape, generator=g),
              norm=torch.randn(out.entropy.shape, generator=g),
              top=torch.randn(out.top_log_probs.shape, generator=g))
    gs = {n: v.to(dev) for n, v in gs.items()}
    grad, = torch.autograd.grad(out[:4], z, (gs["lp"], gs["h"], gs["norm"], gs["top"]))
    C.check_scores(z, out, t, k, m, groups, T, gs, grad)
    if s:                      # only the given cells are differentiated
        out = cb.profile_log_probs(z, t, **how)
        grad, = torch.autograd.grad(out.log_probs, z, gs["lp"])
        only = {n: v if n == "lp" else torch.zeros_like(v) for n, v in gs.items()}
        C.check_scores(z, out, t, k, m, groups, T, only, grad)


# (shape, groups, dtype, listed, renormalize, temperature, mask, weight)
DISTILL = [
    ((1, 1), None, F32, 1, False, 1.0, None, False),
    ((3, 2), None, F32, 1, False, 1.0, None, True),
    ((3, 2), None, BF16, 2, False, 1.0, None, True),
    ((4, 31), None, F16, 5, True, 0.7, None, True),
    ((4, 33), None, F32, 40, False, 1.0, "some", False),
    ((4, 65), None, F32, 0, False, 1.0, None, False),
    ((3, 1, 1000), [1], F32, 32, False, 1.0, None, True),
    ((2, 9, 1000), [1, 2, 2, 2, 2], BF16, 16, True, 2.0, "some", True),
    ((2, 9, 1000), [1, 2, 2, 2, 2], F32, 16, False, 2.0, "some", True),
    ((2, 4, 501), [3, 1], F16, 9, False, 1.5, "channel", True),
    ((2, 3, 7, 65), None, F32, 4, False, 1.0, None, True),
    ((77,), None, F32, 4, True, 1.0, None, False),
    ((3, 1024), None, F32, 300, False, 1.0, None, False),
    ((2, 2047), None, BF16, 1024, False, 1.0, None, True),
    ((2, 4097), None, F16, 100, False, 1.0, "some", True),
    ((2, 16385), None, BF16, 64, False, 1.0, None, True),
    ((2, 50001), None, BF16, 100, True, 1.0, None, True),
    ((2, 65536), None, F32, 10, False, 0.5, "some", True),
]
DISTILL_LONG = [
    ((1, 131072 + 3), None, BF16, 64, False, 1.0, None, True),
    ((2, 300001), None, F32, 128, False, 1.0, "some", True),
    ((1, 1 << 20), None, F32, 30, False, 1.0, None, True),
    ((1, 1 << 20), None, BF16, 30, True, 1.0, None, True),
]


def case_distill(dev, shape, groups, dtype, k, renorm, T, mask, weight, seed=1):
    z, g = C.logits(shape, dtype, seed)
    idx, lp = C.make_teacher(z, groups, k, T, g)
    m = make_mask(mask, shape, g)
    lead = C.lead_of(shape, groups)
    w = (0.5 + torch.rand(lead, generator=g)) if weight else None
    if weight and len(lead) and lead[0] > 2:
        w[1] = 0.0
    z, idx, lp = z.to(dev).requires_grad_(), idx.to(dev), lp.to(dev)
    m, w = m.to(dev) if m is not None else None, w.to(dev) if w is not None else None
    how = dict(renormalize=renorm, mask=m, signal_groups=groups, temperature=T, weight=w)
    for reduction in ("mean", "none"):
        loss, grad = cb.distillation_loss_and_grad(z, idx, lp, reduction=reduction, **how)
        assert not loss.requires_grad and grad.dtype == z.dtype and grad.shape == z.shape
        C.check_distill(z, idx, lp, renorm, m, groups, T, w, reduction, loss, grad)
    with torch.no_grad():
        again = cb.distillation_loss(z, idx, lp, reduction="none", **how)
    # without a gradient long rows are cut otherwise: the same bound, not the same bits
    C.check_distill(z, idx, lp, renorm, m, groups, T, w, "none", again, None)
    up = torch.randn(lead, generator=g).to(dev)
    loss = cb.distillation_loss(z, idx, lp, reduction="none", **how)
    auto, = torch.autograd.grad(loss, z, up)
    C.check_distill(z, idx, lp, renorm, m, groups, T, w, "none", loss.detach(), auto, up)
    loss = cb.distillation_loss(z, idx, lp, reduction="sum", **how)
    auto, = torch.autograd.grad(loss, z, torch.tensor(-2.5, device=dev))
    C.check_distill(z, idx, lp, renorm, m, groups, T, w, "sum", loss.detach(), auto, -2.5)


# ------------------------------------------------------------ values that need care
def odd_rows(dtype):
    """Rows of 40 entries with infinities, NaN, the type's extremes and large offsets."""
    g = torch.Generator().manual_seed(5)
    big = torch.finfo(dtype).max
    z = torch.randn(12, 40, generator=g).to(dtype)
    z[0, 3] = -INF
    z[1, :] = -INF
    z[2, :] = -big                       # a uniform row at the lowest value
    z[3, :] = -big
    z[3, 7] = 1.0                        # one entry above a row of the lowest value
    z[4, 5] = INF
    z[5, 6] = float("nan")
    z[6, :] = big                        # a uniform row at the largest value
    z[7, 1:] = -INF                      # one entry left
    z[8] = (z[8].float() + 1000.0).to(dtype)
    z[9, :] = 0.0
    z[9, ::2] = -0.0                     # equal to +0: ties go by index alone
    z[10, 4], z[10, 9] = big, -big       # differences that overflow
    z[11, 11:30] = z[11, 10].clone()     # ties
    return z


def case_odd_values(dev, dtype, masked):
    z = odd_rows(dtype)
    mask = None
    if masked:                           # what is masked may hold anything
        mask = torch.ones(z.shape, dtype=torch.bool)
        mask[:, 5:8] = False
        mask[9] = False
        z[8, 5], z[8, 6], z[8, 7] = float("nan"), INF, -INF
        z[9] = float("nan")
    t = torch.tensor([[3, 7, -1, 5, 40, 10, 3]]).expand(12, -1).contiguous()
    z, t = z.to(dev).requires_grad_(), t.to(dev)
    mask = mask.to(dev) if mask is not None else None
    out = cb.profile_log_probs(z, t, top_k=45, mask=mask)
    C.check_scores(z, out, t, 45, mask, None, 1.0)
    t[:, 4] = 39                         # a target past the row would make the gradient NaN
    g = torch.Generator().manual_seed(6)
    out = cb.profile_log_probs(z, t, top_k=6, mask=mask)
    gs = dict(lp=torch.randn(t.shape, generator=g), h=torch.randn(12, generator=g),
              norm=torch.randn(12, generator=g), top=torch.randn(12, 6, generator=g))
    gs = {n: v.to(dev) for n, v in gs.items()}
    grad, = torch.autograd.grad(out[:4], z, tuple(gs.values()))
    C.check_scores(z, out, t, 6, mask, None, 1.0, gs, grad)
    # the same entries listed twice, an empty place, a dropped one, masses above 1
    idx = torch.tensor([[3, 10, 3, -1, 7, 12, 3, 20]]).expand(12, -1).contiguous()
    lp = torch.log(torch.tensor([.1, .2, .05, .3, .1, .0, .02, .05])).expand(12, -1).contiguous()
    over = lp + 1.5
    for renorm in (False, True):
        for teacher in (lp, over):
            how = dict(renormalize=renorm, mask=mask)
            i, p = idx.to(dev), teacher.to(dev)
            loss, grad = cb.distillation_loss_and_grad(z, i, p, reduction="none", **how)
            C.check_distill(z, i, p, renorm, mask, None, 1.0, None, "none", loss, grad)


def case_bad_indices(dev):
    """Indices past the row answer NaN, in that row alone, and read nothing."""
    z, g = C.logits((3, 50), F32, 3)
    z = z.to(dev).requires_grad_()
    t = torch.tensor([[1, 2], [50, 2], [1 << 40, -(1 << 40)]]).to(dev)
    out = cb.profile_log_probs(z, t)
    C.check_scores(z, out, t, 0, None, None, 1.0)
    grad, = torch.autograd.grad(out.log_probs.sum(), z)
    assert torch.isfinite(grad[0]).all() and torch.isnan(grad[1:]).all()
    lp = torch.full((3, 2), -1.0).to(dev)
    loss, grad = cb.distillation_loss_and_grad(z, t, lp, reduction="none")
    C.check_distill(z, t, lp, False, None, None, 1.0, None, "none", loss, grad)
    assert torch.isnan(loss[1:]).all() and torch.isfinite(loss[0])
    for bad in (INF, float("nan")):
        lp2 = lp.clone()
        lp2[1, 1] = bad
        t2 = torch.tensor([[1, 2]] * 3).to(dev)
        loss, grad = cb.distillation_loss_and_grad(z, t2, lp2, reduction="none")
        C.check_distill(z, t2, lp2, False, None, None, 1.0, None, "none", loss, grad)
        # a row of weight 0 is not looked at
        w = torch.tensor([1.0, 0.0, 1.0]).to(dev)
        loss, grad = cb.distillation_loss_and_grad(z, t2, lp2, weight=w)
        assert torch.isfinite(loss) and float(grad[1].abs().max()) == 0.0


def case_empty(dev):
    for shape, groups in (((0, 9), None), ((3, 0), None), ((0, 2, 5), [1, 1]),
                          ((2, 2, 0), [2])):
        z = torch.zeros(shape, device=dev, requires_grad=True)
        lead = C.lead_of(shape, groups)
        t = torch.full(lead + (2,), -1, dtype=torch.int64, device=dev)
        out = cb.profile_log_probs(z, t, top_k=2, signal_groups=groups)
        assert out.log_probs.shape == lead + (2,) and out.top_indices.shape == lead + (2,)
        assert (out.top_indices == -1).all() and (out.entropy == 0).all()
        assert (out.log_normalizer == -INF).all()
        grad, = torch.autograd.grad(out.log_probs.sum() + out.entropy.sum(), z)
        assert grad.shape == z.shape
        loss, grad = cb.distillation_loss_and_grad(z, t, t.float(), signal_groups=groups)
        assert float(loss) == 0.0 and grad.shape == z.shape


def case_layouts(dev):
    """Windows, transposed and broadcast logits, a mask with its own strides."""
    g = torch.Generator().manual_seed(8)
    full = torch.randn(3, 4, 700, generator=g).to(dev)
    wide = full[:, :, 57:557]                                  # the model's trimmed window
    cases = [(wide, [1, 1, 1, 1]), (wide, [3, 1]), (full.transpose(0, 2)[:5], [1, 2]),
             (wide[0], None), (wide.transpose(1, 2), None), (full[0, 0].expand(6, 700), None),
             (full[:, :, ::2], [2, 2]), (full[1:2, :, 1:], [4])]
    for z, groups in cases:
        if groups and sum(groups) != z.shape[1]:
            z = z[:, :sum(groups)]
        mask = (torch.rand(z.shape[-1], generator=g) < 0.7).to(dev)
        t = C.make_targets(z.shape, groups, 5, g).to(dev)
        zl = z.detach()
        zl.requires_grad_()
        out = cb.profile_log_probs(zl, t, top_k=4, mask=mask, signal_groups=groups)
        gs = dict(lp=torch.randn(t.shape, generator=g),
                  h=torch.randn(out.entropy.shape, generator=g),
                  norm=torch.randn(out.entropy.shape, generator=g),
                  top=torch.randn(out.top_log_probs.shape, generator=g))
        gs = {n: v.to(dev) for n, v in gs.items()}
        grad, = torch.autograd.grad(out[:4], zl, (gs["lp"], gs["h"], gs["norm"], gs["top"]))
        C.check_scores(zl, out, t, 4, mask, groups, 1.0, gs, grad)
        lp = out.top_log_probs.detach().clone()
        loss, grad = cb.distillation_loss_and_grad(zl, out.top_indices, lp - 0.1, mask=mask,
                                                   signal_groups=groups)
        C.check_distill(zl, out.top_indices, lp - 0.1, False, mask, groups, 1.0, None, "mean",
                        loss, grad)


def case_differences(dev):
    """Gradients against central differences of the operators' own values, in 64 bits where
    the function allows: a smooth direction through the logits, step 2^-6. The difference is
    off by h^2/6 of the third derivative (below 1e-3 here: |f'''| <= 20, h^2/6 = 4e-5) and by
    the values' error over h (1e-5 * 64 = 6e-4)."""
    z, g = C.logits((4, 200), F32, 11, 1.0)
    z = z.to(dev)
    t = C.make_targets((4, 200), None, 3, g, empty=0.0).to(dev)
    idx, lp = C.make_teacher(z.cpu(), None, 6, 1.0, g)
    idx, lp = idx.to(dev), lp.to(dev)
    v = torch.randn(4, 200, generator=g).to(dev)
    v /= v.norm(dim=-1, keepdim=True)
    h = 2.0 ** -6
    fs = [lambda x: cb.profile_log_probs(x, t).log_probs.sum(-1),
          lambda x: cb.profile_log_probs(x).entropy,
          lambda x: cb.profile_log_probs(x).log_normalizer,
          lambda x: cb.distillation_loss(x, idx, lp, reduction="none"),
          lambda x: cb.distillation_loss(x, idx, lp, reduction="none", renormalize=True)]
    for f in fs:
        x = z.clone().requires_grad_()
        grad, = torch.autograd.grad(f(x).sum(), x)
        slope = (grad.double() * v.double()).sum(-1)
        diff = (f(z + h * v).double() - f(z - h * v).double()) / (2 * h)
        assert float((slope - diff).abs().max()) < 2e-3


def case_teacher_student(dev):
    """The run of them together: a teacher's lists through predict, then the student's steps."""
    torch.manual_seed(0)
    teacher = cb.Cherimoya(n_filters=16, n_layers=2, signal_groups=[1, 2], trimming=40,
                           compile=False).to(dev).eval()
    student = cb.Cherimoya(n_filters=8, n_layers=1, signal_groups=[1, 2], trimming=40,
                           compile=False).to(dev)
    g = torch.Generator().manual_seed(2)
    X = torch.nn.functional.one_hot(torch.randint(0, 4, (6, 200), generator=g), 4)
    X = X.transpose(1, 2).float().contiguous()
    top_lp, top_at, entropy, counts = cb.predict(cb.TopCellsWrapper(teacher, top_k=12), X,
                                                 batch_size=4, device=dev)
    assert top_lp.shape == (6, 2, 12) and top_at.dtype == torch.int64
    with torch.no_grad():
        y, c = teacher(X.to(dev))
    ref = cb.profile_log_probs(y.cpu(), top_k=12, signal_groups=[1, 2])
    assert float((ref.entropy - entropy).abs().max()) < 1e-4 and counts.shape == c.shape
    logits, _ = student(X.to(dev))
    loss = cb.distillation_loss(logits, top_at.to(dev), top_lp.to(dev), signal_groups=[1, 2])
    loss.backward()
    by_loss = [p.grad.clone() for p in student.parameters() if p.grad is not None]
    assert by_loss and all(torch.isfinite(x).all() for x in by_loss)
    student.zero_grad()
    logits, _ = student(X.to(dev))
    value, grad = cb.distillation_loss_and_grad(logits, top_at.to(dev), top_lp.to(dev),
                                                signal_groups=[1, 2])
    C.check_distill(logits, top_at, top_lp, False, None, [1, 2], 1.0, None, "mean", value, grad)
    logits.backward(grad)
    assert float((value - loss.detach()).abs()) <= 2 * C.CHAIN * C.U * (1 + float(value))
    for p, q in zip(by_loss, [p.grad for p in student.parameters() if p.grad is not None]):
        # the same gradient of the logits to a rounding or two, through the same layers
        assert float((p - q).norm()) <= 1e-4 * float(p.norm()) + 1e-12
    # a label of reads: their likelihood and its gradient reach the student, too
    reads = torch.randint(0, 120, (6, 2, 20), generator=g).to(dev)
    out = cb.profile_log_probs(student(X.to(dev))[0], reads, signal_groups=[1, 2])
    (-out.log_probs.sum() - 0.01 * out.entropy.sum()).backward()
    assert all(torch.isfinite(p.grad).all() for p in student.parameters() if p.grad is not None)


REFUSED = [
    ("float64", lambda d: cb.profile_log_probs(torch.zeros(2, 5, dtype=torch.float64, device=d))),
    ("at least one axis", lambda d: cb.profile_log_probs(torch.zeros((), device=d))),
    ("must be \\(N, n_outputs, W\\)",
     lambda d: cb.profile_log_probs(torch.zeros(2, 5, device=d), signal_groups=[5])),
    ("do not add up", lambda d: cb.profile_log_probs(torch.zeros(2, 5, 7, device=d),
                                                     signal_groups=[2, 2])),
    ("positive ints", lambda d: cb.profile_log_probs(torch.zeros(2, 5, 7, device=d),
                                                     signal_groups=[5, 0])),
    ("non-empty", lambda d: cb.profile_log_probs(torch.zeros(2, 5, 7, device=d),
                                                 signal_groups=[])),
    ("at most 1048576", lambda d: cb.profile_log_probs(
        torch.zeros(1, device=d).expand(1, (1 << 20) + 1))),
    ("temperature", lambda d: cb.profile_log_probs(torch.zeros(2, 5, device=d), temperature=0.0)),
    ("temperature", lambda d: cb.profile_log_probs(torch.zeros(2, 5, device=d),
                                                   temperature=float("nan"))),
    ("top_k", lambda d: cb.profile_log_probs(torch.zeros(2, 5, device=d), top_k=129)),
    ("top_k", lambda d: cb.profile_log_probs(torch.zeros(2, 5, device=d), top_k=-1)),
    ("top_k", lambda d: cb.profile_log_probs(torch.zeros(2, 5, device=d), top_k=2.0)),
    ("int64 or int32", lambda d: cb.profile_log_probs(torch.zeros(2, 5, device=d),
                                                      torch.zeros(2, 1, device=d))),
    ("must have the shape", lambda d: cb.profile_log_probs(
        torch.zeros(2, 5, device=d), torch.zeros(3, 1, dtype=torch.int64, device=d))),
    ("must have the shape", lambda d: cb.profile_log_probs(
        torch.zeros(2, 5, device=d), torch.zeros(2, dtype=torch.int64, device=d))),
    ("at most 1024", lambda d: cb.profile_log_probs(
        torch.zeros(2, 5, device=d), torch.zeros(2, 1025, dtype=torch.int64, device=d))),
    ("bool tensor", lambda d: cb.profile_log_probs(torch.zeros(2, 5, device=d),
                                                   mask=torch.zeros(2, 5, device=d))),
    ("does not broadcast", lambda d: cb.profile_log_probs(
        torch.zeros(2, 5, device=d), mask=torch.zeros(2, 4, dtype=torch.bool, device=d))),
    ("teacher_log_probs must be floating", lambda d: _distill(d, lp=torch.zeros(2, 4))),
    ("teacher_log_probs must be floating",
     lambda d: _distill(d, lp=torch.zeros(2, 3, dtype=torch.int64))),
    ("takes no gradient", lambda d: _distill(d, lp=torch.zeros(2, 3, requires_grad=True))),
    ("takes no gradient", lambda d: _distill(d, weight=torch.ones(2, requires_grad=True))),
    ("weight must be", lambda d: _distill(d, weight=torch.ones(3))),
    ("reduction", lambda d: _distill(d, reduction="batchmean")),
    ("at most 1024", lambda d: cb.distillation_loss(
        torch.zeros(2, 5, device=d), torch.zeros(2, 1025, dtype=torch.int64, device=d),
        torch.zeros(2, 1025, device=d))),
]


def _distill(d, lp=None, weight=None, **kw):
    lp = torch.zeros(2, 3) if lp is None else lp
    move = (lambda t: t if t is None else t.to(d) if not t.requires_grad
            else t.detach().to(d).requires_grad_())
    return cb.distillation_loss(torch.zeros(2, 5, device=d),
                                torch.zeros(2, 3, dtype=torch.int64, device=d), move(lp),
                                weight=move(weight), **kw)


def case_refused(dev, match, call):
    with pytest.raises((RuntimeError, ValueError), match=match):
        call(dev)


def case_no_second_derivative(dev):
    z = torch.randn(2, 30, device=dev, requires_grad=True)
    out = cb.profile_log_probs(z, top_k=2)
    g, = torch.autograd.grad(out.entropy.sum(), z, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


# ------------------------------------------------------------ rows that take the rarer ways
def case_hard_rows(dev, dtype, v, k):
    """Rows whose largest entries lie in one place, in order, or are few; rows with -inf."""
    g = torch.Generator().manual_seed(v + k)
    noise = torch.randn(9, v, generator=g)
    pos = torch.arange(v).float()
    z = torch.stack([
        pos / v * 8 + noise[0] * 1e-3,                                # ascending
        -pos / v * 8 + noise[1] * 1e-3,                               # descending
        8 * torch.exp(-((pos - v // 3) / 12) ** 2) + noise[2] * 0.1,  # a summit
        8 * torch.exp(-((pos - v // 2) / (v / 5)) ** 2) + noise[3] * 0.1,   # a broad one
        torch.where(pos % max(2, v // 7) == 3, noise[4], -INF),       # few entries at all
        torch.where(torch.rand(v, generator=g) < 0.5, noise[5], -INF),
        torch.where(pos == v - 1, 2.0, -INF),                         # one entry, at the end
        torch.full((v,), -INF),
        torch.full((v,), float(torch.finfo(dtype).min)),
    ]).to(dtype)
    t = C.make_targets((9, v), None, 3, g)
    t[:, 0] = v - 1
    z, t = z.to(dev).requires_grad_(), t.to(dev)
    out = cb.profile_log_probs(z, t, top_k=k)
    gs = dict(lp=torch.randn(t.shape, generator=g), h=torch.randn(9, generator=g),
              norm=torch.randn(9, generator=g), top=torch.randn(9, k, generator=g))
    gs = {n: x.to(dev) for n, x in gs.items()}
    grad, = torch.autograd.grad(out[:4], z, tuple(gs.values()))
    C.check_scores(z, out, t, k, None, None, 1.0, gs, grad)
    idx, lp = out.top_indices, out.top_log_probs.detach().clamp(min=-60.0) - 0.05
    for renorm in (False, True):
        loss, grad = cb.distillation_loss_and_grad(z, idx, lp, renormalize=renorm,
                                                   reduction="none")
        C.check_distill(z, idx, lp, renorm, None, None, 1.0, None, "none", loss, grad)


def case_repeats(dev, v, k, rows):
    """Lists with entries twice and more, next to lists where they only look alike (32768 apart),
    empty places and dropped entries among them."""
    z, g = C.logits((rows, v), F32, v + k)
    z[:, ::11] = -INF
    idx = torch.randint(0, v, (rows, k), generator=g)
    idx[:, 1::5] = idx[:, 0:1]
    idx[:, 2::7] = torch.where(idx[:, 3:4] >= 32768, idx[:, 3:4] - 32768,
                               (idx[:, 3:4] + 32768) % v)
    idx[:, 4::9] = -1
    lp = torch.log_softmax(torch.randn(rows, k, generator=g), -1) - 0.2
    lp[:, 5::13] = -INF
    z, idx, lp = z.to(dev), idx.to(dev), lp.to(dev)
    w = torch.ones(rows)
    if rows > 2:
        w[1] = 0.0
    w = w.to(dev)
    for renorm in (False, True):
        how = dict(renormalize=renorm, weight=w, reduction="none")
        loss, grad = cb.distillation_loss_and_grad(z, idx, lp, **how)
        C.check_distill(z, idx, lp, renorm, None, None, 1.0, w, "none", loss, grad)
        C.check_distill(z, idx, lp, renorm, None, None, 1.0, w, "none",
                        cb.distillation_loss(z, idx, lp, **how), None)


def case_many_targets(dev, v):
    """As many given entries as a call takes, most of them more than once."""
    z, g = C.logits((2, v), BF16, 3)
    t = torch.randint(0, min(v, 300), (2, 1024), generator=g)
    t[:, ::17] = -1
    z, t = z.to(dev).requires_grad_(), t.to(dev)
    out = cb.profile_log_probs(z, t)
    gs = dict(lp=torch.randn(t.shape, generator=g), h=torch.zeros(2), norm=torch.zeros(2),
              top=torch.zeros(2, 0))
    grad, = torch.autograd.grad(out.log_probs, z, gs["lp"].to(dev))
    C.check_scores(z, out, t, 0, None, None, 1.0, gs, grad)


def case_temperatures(dev, dtype, T):
    z, g = C.logits((3, 700), dtype, 41)
    z[1] = -torch.finfo(dtype).max
    z[1, 5:9] = -torch.finfo(dtype).max * 0.75
    t = C.make_targets((3, 700), None, 2, g).to(dev)
    z = z.to(dev)
    out = cb.profile_log_probs(z, t, top_k=9, temperature=T)
    C.check_scores(z, out, t, 9, None, None, T)
    idx = out.top_indices
    lp = out.top_log_probs.clamp(min=-80.0)
    loss, grad = cb.distillation_loss_and_grad(z[::2], idx[::2], lp[::2] - 0.1, temperature=T,
                                               reduction="none")
    C.check_distill(z[::2], idx[::2], lp[::2] - 0.1, False, None, None, T, None, "none", loss, grad)


def case_ends(dev, dtype, v, k, rows):
    """Some of a row's first and last entries, which no full vector holds, are listed and some not."""
    z, g = C.logits((rows, v), dtype, v + k)
    z[:, [0, 2, -1, -3]] += 4.0
    idx = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(rows)])
    ends = torch.tensor([0, 1, 4, 6, v - 1, v - 2, v - 4, v - 7])
    inner = (idx > 7) & (idx < v - 8)
    idx = torch.where(inner, idx, -1)
    at = torch.randperm(k, generator=g)[:8]
    for r in range(rows):
        idx[r, at] = ends.roll(r) if r % 3 else torch.where(ends % 2 == r % 2, ends, -1)
    lp = torch.log_softmax(torch.randn(rows, k, generator=g), -1) - 0.3
    z, idx, lp = z.to(dev), idx.to(dev), lp.to(dev)
    for renorm in (False, True):
        how = dict(renormalize=renorm, reduction="none")
        loss, grad = cb.distillation_loss_and_grad(z, idx, lp, **how)
        C.check_distill(z, idx, lp, renorm, None, None, 1.0, None, "none", loss, grad)
        C.check_distill(z, idx, lp, renorm, None, None, 1.0, None, "none",
                        cb.distillation_loss(z, idx, lp, **how), None)
