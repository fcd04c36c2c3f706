"""More cases of the likelihood and distillation tests, run on the device they are given."""

import math

import pytest
import torch

import cherimoya_b200 as cb
import likelihood_common as C
from oracle import likelihood_oracle as LO


def case_candidates(dev, dtype, v, rows):
    """Rows in which a block finds more candidates for its top entries than it ranks and has
    room for all of them: equal ones, ones that share their 16-byte vectors, and more than
    there is room for, in neighbouring rows, so that one launch takes each way."""
    g = torch.Generator().manual_seed(v + rows)
    z = -1.0 - torch.rand(rows, v, generator=g)
    for r in range(rows):
        at = torch.randperm(v // 8 - 1, generator=g)
        if r % 3 == 0:                                   # 480 equal ones, an entry to a vector
            z[r, 8 * at[:480] + 5] = 4.0
        elif r % 3 == 1:                                 # 60 vectors full of different ones
            full = (8 * at[:60, None] + torch.arange(8)).reshape(-1)
            z[r, full] = 2.0 + torch.randperm(480, generator=g).float() / 64
        else:                                            # equal ones beyond all room
            z[r, ::2] = 3.0
    z = z.to(dtype)
    t = C.make_targets((rows, v), None, 2, g)
    z, t = z.to(dev), t.to(dev)
    for k in (1, 8, 40):
        for _ in range(3):
            out = cb.profile_log_probs(z, t, top_k=k)
        C.check_scores(z, out, t, k, None, None, 1.0)


def case_small_mass(dev, dtype, v, k, rows):
    """Lists of little mass: outside the list the gradient is the entry's share of the rest times
    (list's mass under the teacher - its mass under the student), and its error is bounded by
    those two masses, not by the rest's, which are nearly 1. From the bounds of
    likelihood_common.py each mass is off by at most 2 CHAIN U of itself, and so is the share.
    Without a list the gradient is exactly 0."""
    g = torch.Generator().manual_seed(v + k)
    z = (0.5 * torch.randn(rows, v, generator=g)).to(dtype)
    q = torch.log_softmax(z.double(), -1)
    idx = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(rows)])
    lp = (q.gather(-1, idx) + 0.3 * torch.randn(rows, k, generator=g)).float()
    loss, grad = cb.distillation_loss_and_grad(z.to(dev), idx.to(dev), lp.to(dev),
                                               reduction="none")
    listed = torch.zeros(rows, v, dtype=torch.bool).scatter_(-1, idx, True)
    p_u, q_u = lp.double().exp(), q.gather(-1, idx).exp()
    p_list, q_list = p_u.sum(-1, keepdim=True), q_u.sum(-1, keepdim=True)
    assert float(p_list.max()) < 0.5 and float(q_list.max()) < 0.5
    share = torch.where(listed, 0.0, q.exp() / (1 - q_list))
    want = share * (p_list - q_list)
    want.scatter_(-1, idx, q_u - p_u)
    mag = share * (p_list + q_list)
    mag.scatter_(-1, idx, q_u + p_u)
    tol = C.HALF_STEP[dtype] * want.abs() + 2 * C.CHAIN * C.U * mag + C.TINY[dtype]
    C.same(grad, want, tol, "gradient")
    z = z.to(dev).requires_grad_()
    loss = cb.distillation_loss(z, idx.to(dev), lp.to(dev), reduction="sum")
    auto, = torch.autograd.grad(loss, z)
    C.same(auto, want, tol, "gradient through autograd")
    none = torch.empty(rows, 0, device=dev)
    loss, grad = cb.distillation_loss_and_grad(z, none.long(), none)
    assert float(loss) == 0.0 and float(grad.abs().max()) == 0.0


def _calls():
    """(what is transformed, function of it) of every public call and every differentiable-looking
    argument; the others are plain."""
    g = torch.Generator().manual_seed(2)
    z, idx = torch.randn(3, 20, generator=g), torch.randint(0, 20, (3, 4), generator=g)
    lp, w = torch.full((3, 4), -2.0), torch.ones(3)
    return {
        "scores": (z, lambda d, x: cb.profile_log_probs(x, top_k=2).entropy.sum()),
        "loss": (z, lambda d, x: cb.distillation_loss(x, idx.to(d), lp.to(d))),
        "loss and grad": (z, lambda d, x: cb.distillation_loss_and_grad(x, idx.to(d),
                                                                        lp.to(d))[0]),
        "teacher": (lp, lambda d, x: cb.distillation_loss(z.to(d), idx.to(d), x)),
        "weight": (w, lambda d, x: cb.distillation_loss(z.to(d), idx.to(d), lp.to(d), weight=x)),
    }


CALLS = sorted(_calls())


def _dual(f, x):
    from torch.autograd import forward_ad
    with forward_ad.dual_level():
        return forward_ad.unpack_dual(f(forward_ad.make_dual(x, torch.ones_like(x)))).tangent


TRANSFORMS = {
    "jvp": lambda f, x: torch.func.jvp(f, (x,), (x,)),
    "jacfwd": lambda f, x: torch.func.jacfwd(f)(x),
    "grad": lambda f, x: torch.func.grad(f)(x),
    "vmap": lambda f, x: torch.func.vmap(f)(x[None]),
    "dual": _dual,
    "dual without grad": torch.no_grad()(_dual),
    "dual that requires grad": lambda f, x: _dual(f, x.clone().requires_grad_()),
}


def case_transforms(dev, call, transform):
    """Derivatives that the calls do not form are refused, never 0."""
    x, f = _calls()[call]
    with pytest.raises(RuntimeError, match="forward-mode|takes no gradient"):
        TRANSFORMS[transform](lambda v: f(dev, v), x.to(dev))
    assert torch.isfinite(f(dev, x.to(dev))).all()           # and a plain call works behind it


def case_beside_forward_mode(dev):
    """Plain tensors, a fixed teacher's, are scored while others carry tangents."""
    z = torch.linspace(-1, 1, 20, device=dev).repeat(3, 1)
    want = cb.profile_log_probs(z).entropy.sum()
    got = _dual(lambda x: cb.profile_log_probs(z).entropy.sum() * x, torch.tensor(2.0, device=dev))
    assert torch.equal(got, want)


def case_temperature_is_a_number(dev):
    """A tensor's value counts, its gradient would be lost: it is refused."""
    z = torch.linspace(-1, 1, 20, device=dev).repeat(3, 1)
    idx, lp = torch.zeros(3, 1, dtype=torch.int64, device=dev), torch.full((3, 1), -1.0, device=dev)
    learnt = torch.tensor(2.0, device=dev, requires_grad=True)
    calls = [lambda x, T: cb.profile_log_probs(x, top_k=2, temperature=T)[1:4],
             lambda x, T: (cb.distillation_loss(x, idx, lp, temperature=T),),
             lambda x, T: cb.distillation_loss_and_grad(x, idx, lp, temperature=T)]
    for call in calls:
        for x in (z, z.clone().requires_grad_()):
            with pytest.raises(RuntimeError, match="temperature takes no gradient"):
                call(x, learnt)
            want = call(x, 2.0)
            for T in (learnt.detach(), learnt.detach().cpu().double()):
                got = call(x, T)
                assert all(torch.equal(a, b) and a.requires_grad == b.requires_grad
                           for a, b in zip(got, want))
            with torch.no_grad():
                assert all(torch.equal(a, b) for a, b in zip(call(x, learnt), want))
        with pytest.raises(RuntimeError, match="temperature must be a plain tensor"):
            _dual(lambda T: call(z, T)[0], learnt.detach())
        with pytest.raises(ValueError, match="temperature"):
            call(z, torch.tensor(0.0, device=dev))


def case_long_sums(dev, dtype, rows, every):
    """Rows of 2^20 entries that are nearly all alike, so that the roundings of a sum have one
    sign: every 509th entry, and so some that every thread has, is 0 and the others have a value
    between -0.69 and 0, different from row to row; with `every`, each entry of that multiple is
    -inf. With |x| <= 0.7 a term is off by (4 + 3 * 0.7) U of itself, the sum by 80 U more (partial
    sums of at most 64 terms in a row and 16 joins, as likelihood_common.py has it), and its
    logarithm by 2 U of itself."""
    v = 1 << 20
    c = (-0.69 * torch.rand(rows, generator=torch.Generator().manual_seed(rows))).to(dtype)
    one = torch.ones(v)
    if every:
        one[every - 1::every] = -1
    one[::509] = 0
    others, zeros = int((one > 0).sum()), int((one == 0).sum())
    one = one.to(dev)
    z = torch.where(one == 1, c.to(dev)[:, None], (one.clamp(max=0) * torch.inf).nan_to_num(
        0, neginf=-torch.inf).to(dtype))
    c = c.double()
    log_r = c + math.log(others)                               # of the others, below 0's
    norm = torch.logaddexp(log_r, torch.full((), math.log(zeros)).double())
    off = C.U * (6.1 + 80 + 2 * norm)
    out = cb.profile_log_probs(z)
    C.same(out.log_normalizer, norm, off, "normaliser")
    # sum of x e over s, x = c or 0: each term is off by one rounding more, the quotient by two
    share = torch.exp(log_r - norm)
    h = norm - c * share
    C.same(out.entropy, h, off + (6.1 + 80 + 6.1 + 80 + 4) * C.U * (c * share).abs()
           + 2 * C.U * h, "entropy")
    # half of the teacher's mass is the entry 0's: half of the normaliser's error reaches the loss
    idx = torch.zeros(rows, 1, dtype=torch.int64, device=dev)
    lp = torch.full((rows, 1), math.log(0.5), device=dev)
    p = lp[0, 0].double().exp().item()
    loss = cb.distillation_loss(z, idx, lp, reduction="none")
    rest = torch.logaddexp(log_r, torch.full((), math.log(zeros - 1)).double())
    want = p * (math.log(p) + norm) + (1 - p) * (math.log(1 - p) - (rest - norm))
    C.same(loss, want, 0.5 * (6.1 + 80) * C.U + 4 * C.U * want, "loss")


def case_one_target(dev, v):
    """1,024 targets that are one entry, with one gradient each that differs from row to row: the
    roundings of their sum G have one sign. Terms are added at most 64 in a row, with 16 joins: 80 U
    of G; the first term of the gradient, q G, is off by 2 CHAIN U of itself, as in
    likelihood_common.py."""
    rows = 64
    z, g = C.logits((rows, v), torch.float32, v)
    t = torch.full((rows, 1024), v // 3, dtype=torch.int64)
    each = 0.5 + torch.rand(rows, 1, generator=g)
    z = z.to(dev).requires_grad_()
    out = cb.profile_log_probs(z, t.to(dev))
    grad, = torch.autograd.grad(out.log_probs, z, each.expand(rows, 1024).to(dev))
    total = 1024 * each.double()
    q = torch.softmax(z.detach().double().cpu(), -1)
    want = -q * total
    tol = 2 * C.CHAIN * C.U * want.abs()
    want[:, v // 3] += total[:, 0]
    tol[:, v // 3] += 80 * C.U * total[:, 0]
    C.same(grad, want, tol + 2 * C.U * want.abs() + C.TINY[torch.float32], "gradient")


def case_compiled(dev, dynamic):
    """The public calls in compiled functions, without a graph break: the results of the plain
    calls, bit for bit, forward and backward."""
    g = torch.Generator().manual_seed(12)
    groups = [1, 2]
    t = torch.randint(0, 90, (4, 2, 5), generator=g)
    t[0] = -1
    idx = torch.stack([torch.randperm(90, generator=g)[:6] for _ in range(8)]).reshape(4, 2, 6)
    lp = torch.log_softmax(torch.randn(4, 2, 6, generator=g), -1) - 0.1
    w = 0.5 + torch.rand(4, 2, generator=g)
    mask = (torch.rand(4, 3, 90, generator=g) < 0.9).to(dev)
    t, idx, lp, w = t.to(dev), idx.to(dev), lp.to(dev), w.to(dev)
    how = dict(signal_groups=groups, temperature=1.5, mask=mask)

    def scores(z):
        out = cb.profile_log_probs(z, t, top_k=3, **how)
        return out.log_probs, out.entropy, out.log_normalizer, out.top_log_probs, out.top_indices

    def losses(z):
        return (cb.distillation_loss(z, idx, lp, weight=w, **how),
                cb.distillation_loss(z, idx, lp, reduction="none", renormalize=True, **how))

    def once(z):
        return cb.distillation_loss_and_grad(z, idx, lp, weight=w, **how)

    torch._dynamo.reset()
    for f, with_grad in ((scores, 4), (losses, 2), (once, 0)):
        compiled = torch.compile(f, backend="aot_eager", fullgraph=True, dynamic=dynamic)
        for seed in (1, 2):
            z = torch.randn(4, 3, 90, generator=torch.Generator().manual_seed(seed)).to(dev)
            with torch.no_grad():
                assert all(torch.equal(a, b) for a, b in zip(compiled(z), f(z)))
            grads = []
            for call in (f, compiled):
                x = z.clone().requires_grad_()
                out = call(x)
                if with_grad:
                    torch.manual_seed(seed)
                    up = [torch.randn(o.shape).to(dev) for o in out[:with_grad]]
                    grads.append(torch.autograd.grad(out[:with_grad], x, up)[0])
                else:
                    assert not any(o.requires_grad for o in out)
                    grads.append(out[1])
            assert torch.equal(*grads)
    torch._dynamo.reset()


def case_many_long_rows(dev, dtype, masked, copies):
    """Long rows, many of them, so that each has a block: three rows, each there `copies` times,
    with 600 listed entries, some of them twice, at both ends and not part of the mask."""
    v, k = 300001 if dtype == torch.float32 else 600001, 600
    z, g = C.logits((3, v), dtype, 77)
    idx = torch.randint(0, v, (3, k), generator=g)
    idx[:, :4] = torch.tensor([0, v - 1, 3, v - 2])
    idx[:, 4:8] = idx[:, 8:12]
    lp = torch.log_softmax(torch.randn(3, k, generator=g), -1) - 0.4
    mask = torch.rand(3, v, generator=g) < 0.8 if masked else None
    want, mags, off = [], [], []
    for r in range(3):
        m = mask[r] if masked else None
        loss, mag, _, _ = LO.distill_row(z[r], m, idx[r], lp[r], False, 1.0)
        want.append(loss)
        mags.append(2 * C.CHAIN * C.U * (mag + 1))
        s = LO.score_row(z[r], m, idx[r, :0], 0, 1.0)
        off.append((s["log_normalizer"], C.U * (4 * abs(s["log_s"]) + C.CHAIN)
                    + 4 * C.U * abs(s["log_normalizer"])))
    many = lambda t: t.to(dev).repeat(copies, *[1] * (t.dim() - 1))
    zl, ml = many(z), many(mask) if masked else None
    loss = cb.distillation_loss(zl, many(idx), many(lp), mask=ml, reduction="none")
    C.same(loss, torch.tensor(want * copies), torch.tensor(mags * copies), "losses")
    out = cb.profile_log_probs(zl, mask=ml, top_k=5)
    norm, tol = torch.tensor(off).double().unbind(-1)
    C.same(out.log_normalizer, norm.repeat(copies), tol.repeat(copies), "normaliser")
    seen = torch.where(mask, z, -torch.inf) if masked else z
    at = torch.sort(seen.float(), dim=-1, descending=True, stable=True)[1][:, :5]
    assert torch.equal(out.top_indices.cpu(), at.repeat(copies, 1))
