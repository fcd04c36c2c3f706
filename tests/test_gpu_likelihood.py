"""Likelihood and distillation kernels against the 64-bit oracle, over sizes on both sides of
each variant's limits, masks, extremes, layouts, streams and graphs."""

import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.dirname(os.path.abspath(__file__)))
import cherimoya_b200 as cb  # noqa: E402
import likelihood_cases as K  # noqa: E402
import likelihood_common as C  # noqa: E402

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)


@pytest.mark.parametrize("case", K.SCORE + K.LONG, ids=str)
def test_scores(case):
    K.case_scores(DEV, *case)


@pytest.mark.parametrize("case", K.DISTILL + K.DISTILL_LONG, ids=str)
def test_distill(case):
    K.case_distill(DEV, *case)


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("dtype", [K.F32, K.BF16, K.F16])
def test_odd_values(dtype, masked):
    K.case_odd_values(DEV, dtype, masked)


def test_bad_indices():
    K.case_bad_indices(DEV)


def test_empty():
    K.case_empty(DEV)


def test_layouts():
    K.case_layouts(DEV)


def test_differences():
    K.case_differences(DEV)


def test_teacher_and_student():
    K.case_teacher_student(DEV)


@pytest.mark.parametrize("match,call", K.REFUSED, ids=[str(i) for i in range(len(K.REFUSED))])
def test_refusals(match, call):
    K.case_refused(DEV, match, call)


def test_no_second_derivative():
    K.case_no_second_derivative(DEV)


def test_refuses_tensors_of_two_devices():
    z = torch.zeros(2, 5, device=DEV)
    with pytest.raises(RuntimeError, match="logits' device"):
        cb.profile_log_probs(z, torch.zeros(2, 1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="logits' device"):
        cb.profile_log_probs(z, mask=torch.ones(2, 5, dtype=torch.bool))
    i = torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="logits' device"):
        cb.distillation_loss(z, i, torch.zeros(2, 3))
    with pytest.raises(RuntimeError, match="logits' device"):
        cb.distillation_loss(z, i, torch.zeros(2, 3, device=DEV), weight=torch.ones(2))


# ties: far more equal logits at the border of the top entries than any list has room for
@pytest.mark.parametrize("dtype", [K.F32, K.BF16])
@pytest.mark.parametrize("v", [1000, 4097, 70001])
def test_ties(dtype, v):
    g = torch.Generator().manual_seed(v)
    rows = [torch.zeros(v), torch.randint(0, 3, (v,), generator=g).float(),
            torch.arange(v).float() / v, -torch.arange(v).float() / v,
            torch.cat([torch.ones(v // 2), torch.full((v - v // 2,), 1.5)])]
    z = torch.stack(rows).to(dtype).to(DEV)
    t = C.make_targets((5, v), None, 2, g).to(DEV)
    for k in (1, 33, 128):
        out = cb.profile_log_probs(z, t, top_k=k)
        C.check_scores(z, out, t, k, None, None, 1.0)


def test_many_groups():
    """More signal groups than one launch takes."""
    groups = [1, 2] * 45
    z, g = C.logits((2, 135, 30), K.F32, 4)
    t = C.make_targets(z.shape, groups, 2, g).to(DEV)
    z = z.to(DEV).requires_grad_()
    out = cb.profile_log_probs(z, t, top_k=3, signal_groups=groups)
    gs = dict(lp=torch.randn(t.shape, generator=g), h=torch.randn(out.entropy.shape, generator=g),
              norm=torch.randn(out.entropy.shape, generator=g),
              top=torch.randn(out.top_log_probs.shape, generator=g))
    gs = {n: v.to(DEV) for n, v in gs.items()}
    grad, = torch.autograd.grad(out[:4], z, tuple(gs.values()))
    C.check_scores(z, out, t, 3, None, groups, 1.0, gs, grad)
    lp = out.top_log_probs.detach() - 0.2
    loss, grad = cb.distillation_loss_and_grad(z, out.top_indices, lp, signal_groups=groups)
    C.check_distill(z, out.top_indices, lp, False, None, groups, 1.0, None, "mean", loss, grad)


def test_many_rows():
    """Every row of many is looked at, whichever block has it. Rows that lie alike in their
    16-byte granules (every 28th: 28 * 130 entries are a multiple of 8) are added up in the same
    order and agree bit for bit. Others are added in another order: each answer is within the
    bound B of the exact one, so two differ by at most 2B."""
    z, g = C.logits((7, 130), K.BF16, 9)
    t = C.make_targets((7, 130), None, 3, g)
    rep = 3001

    def near(many, one, bound):
        many, one = many.reshape(rep, -1).double(), one.reshape(1, -1).double()
        assert torch.equal(torch.isfinite(many), torch.isfinite(one).expand_as(many))
        off = torch.where(torch.isfinite(one), (many - one).abs(), 0.0)
        assert bool((off <= 2 * bound(one.abs())).all())
        same = many[:rep // 4 * 4].reshape(rep // 4, -1)
        assert torch.equal(same, same[:1].expand_as(same))

    zl, tl = z.repeat(rep, 1).to(DEV), t.repeat(rep, 1).to(DEV)
    out = cb.profile_log_probs(zl, tl, top_k=4)
    first = cb.profile_log_probs(z.to(DEV), t.to(DEV), top_k=4)
    C.check_scores(z, first, t, 4, None, None, 1.0)
    log_s = 5.0                                    # log of 130 entries
    for a, b in zip(out[:4], first[:4]):
        near(a, b, lambda x: 2 * C.U * (4 * log_s + C.CHAIN) * (1 + x))
    assert torch.equal(out.top_indices, first.top_indices.repeat(rep, 1))
    idx, lp = first.top_indices, first.top_log_probs - 0.3
    rows = cb.distillation_loss(zl, idx.repeat(rep, 1), lp.repeat(rep, 1), reduction="none")
    one = cb.distillation_loss(z.to(DEV), idx, lp, reduction="none")
    # |log P| + |log q| of the listed entries and the rest: below 12 here
    near(rows, one, lambda x: 2 * C.CHAIN * C.U * (1 + 12))
    loss, grad = cb.distillation_loss_and_grad(zl, idx.repeat(rep, 1), lp.repeat(rep, 1),
                                               reduction="sum")
    _, g1 = cb.distillation_loss_and_grad(z.to(DEV), idx, lp, reduction="sum")
    near(grad, g1, lambda x: C.HALF_STEP[K.BF16] * x + 2 * C.CHAIN * C.U * (x + 1))
    assert abs(float(loss) - float(rows.double().sum())) <= 2 ** -23 * float(rows.double().sum())


def test_repeats_bit_for_bit():
    z, g = C.logits((64, 9, 1000), K.F32, 13)
    groups = [1, 2, 2, 2, 2]
    t = C.make_targets(z.shape, groups, 200, g, empty=0.0).to(DEV)
    t[..., 100:] = t[..., :100]                       # every target twice
    z = z.to(DEV).requires_grad_()
    g_lp = torch.randn(t.shape, generator=g).to(DEV)
    seen = None
    for _ in range(4):
        out = cb.profile_log_probs(z, t, top_k=20, signal_groups=groups)
        grad, = torch.autograd.grad(out.log_probs, z, g_lp)
        loss, dg = cb.distillation_loss_and_grad(z, out.top_indices, out.top_log_probs.detach(),
                                                 signal_groups=groups)
        now = [x.detach().clone() for x in out] + [grad, loss, dg]
        assert seen is None or all(torch.equal(a, b) for a, b in zip(seen, now))
        seen = now


def test_neighbours_are_left_alone():
    """Rows that end inside a 16-byte vector: what lies behind the output's rows is not written,
    and what lies around the input's rows is not looked at."""
    for dtype in (K.F32, K.BF16):
        for width in (3, 61, 1003, 5001):
            buf = torch.full((4, width + 13), float("nan"), dtype=dtype)
            z, g = C.logits((4, width), dtype, width)
            buf[:, 5:5 + width] = z
            view = buf.to(DEV)[:, 5:5 + width].requires_grad_()
            t = C.make_targets((4, width), None, 3, g).to(DEV)
            out = cb.profile_log_probs(view, t, top_k=5)
            g_lp = torch.randn(t.shape, generator=g).to(DEV)
            grad, = torch.autograd.grad(out.log_probs, view, g_lp)
            ref = z.to(DEV).requires_grad_()
            want = cb.profile_log_probs(ref, t, top_k=5)
            wgrad, = torch.autograd.grad(want.log_probs, ref, g_lp)
            C.check_scores(view, out, t, 5, None, None, 1.0)
            assert torch.isfinite(grad).all()
            assert float((grad.float() - wgrad.float()).abs().max()) <= 2 * C.HALF_STEP[dtype] * \
                (1 + float(wgrad.float().abs().max()))


def test_on_another_stream():
    z, g = C.logits((32, 5000), K.BF16, 17)
    t = C.make_targets((32, 5000), None, 2, g).to(DEV)
    z = z.to(DEV).requires_grad_()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        out = cb.profile_log_probs(z, t, top_k=9)
        grad, = torch.autograd.grad(out.log_probs.sum(), z)
        loss, dg = cb.distillation_loss_and_grad(z, out.top_indices, out.top_log_probs.detach())
    side.synchronize()
    ref = cb.profile_log_probs(z, t, top_k=9)
    rgrad, = torch.autograd.grad(ref.log_probs.sum(), z)
    assert all(torch.equal(a, b) for a, b in zip(out, ref)) and torch.equal(grad, rgrad)
    rl, rg = cb.distillation_loss_and_grad(z, ref.top_indices, ref.top_log_probs.detach())
    assert torch.equal(loss, rl) and torch.equal(dg, rg)


def test_graphs():
    """Two graphs, replayed in turn with new inputs: a scoring pass, and a whole training step
    (forward and backward, and the one-call form)."""
    z, g = C.logits((16, 2, 700), K.F32, 19)
    groups = [1, 1]
    t = C.make_targets(z.shape, groups, 4, g).to(DEV)
    idx, lp = C.make_teacher(z, groups, 6, 1.0, g)
    idx, lp = idx.to(DEV), lp.to(DEV)
    static = z.to(DEV).requires_grad_()

    def score():
        with torch.no_grad():
            return cb.profile_log_probs(static, t, top_k=3, signal_groups=groups)

    def step():
        loss = cb.distillation_loss(static, idx, lp, signal_groups=groups)
        grad, = torch.autograd.grad(loss, static)
        value, once = cb.distillation_loss_and_grad(static, idx, lp, signal_groups=groups)
        return loss.detach(), grad, value, once

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            score(), step()
    torch.cuda.current_stream().wait_stream(side)
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        a = score()
    with torch.cuda.graph(gb):
        b = step()
    for seed in (23, 24, 25):
        new, _ = C.logits(z.shape, K.F32, seed)
        with torch.no_grad():
            static.copy_(new)
        gb.replay()
        ga.replay()
        gb.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in tuple(a) + tuple(b)]
        want = tuple(score()) + step()
        assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_backward_twice():
    z, g = C.logits((8, 300), K.F32, 29)
    idx, lp = C.make_teacher(z, None, 5, 1.0, g)
    z = z.to(DEV).requires_grad_()
    loss = cb.distillation_loss(z, idx.to(DEV), lp.to(DEV))
    a, = torch.autograd.grad(loss, z, retain_graph=True)
    b, = torch.autograd.grad(loss, z)
    assert torch.equal(a, b)
    loss = cb.distillation_loss(z, idx.to(DEV), lp.to(DEV))
    with torch.no_grad():
        z += 1.0                                      # the graph holds these very logits
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_custom_ops_trace():
    """The custom ops behind the calls have fake implementations of the right shapes."""
    from torch._subclasses.fake_tensor import FakeTensorMode
    from cherimoya_b200 import ops
    with FakeTensorMode():
        z = torch.empty(4, 10, device="cuda")
        t = torch.empty(4, 2, dtype=torch.int64, device="cuda")
        out = ops.log_probs(z, None, [], t, 3, 1.0, True)
        assert [tuple(o.shape) for o in out] == [(4, 2), (4,), (4,), (4, 3), (4, 3), (4, 2)]
        losses, loss, grad = ops.distill(z, None, [], t, t.float(), False, None, 0.25, None,
                                         True, True, True, 1.0)
        assert tuple(losses.shape) == (4,) and loss.dim() == 0 and grad.shape == z.shape


def test_long_strides():
    """Rows that start more than 2^31 elements into their storage."""
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB of free device memory")
    big = torch.empty((1 << 31) + 4096, dtype=torch.bfloat16, device=DEV)
    z, g = C.logits((2, 1001), K.BF16, 31)
    view = torch.as_strided(big, (2, 1001), ((1 << 31) + 7, 1))
    view.copy_(z.to(DEV))
    t = C.make_targets((2, 1001), None, 3, g).to(DEV)
    out = cb.profile_log_probs(view, t, top_k=5)
    C.check_scores(view, out, t, 5, None, None, 1.0)
    loss, grad = cb.distillation_loss_and_grad(view, out.top_indices, out.top_log_probs - 0.1)
    C.check_distill(view, out.top_indices, out.top_log_probs - 0.1, False, None, None, 1.0, None,
                    "mean", loss, grad)


# a warp, a block and a cluster to a row; below and above what a ring or a chunk holds
@pytest.mark.parametrize("dtype", [K.F32, K.BF16, K.F16])
@pytest.mark.parametrize("v,k", [(50, 7), (403, 50), (900, 40), (2000, 64), (2100, 128),
                                 (9001, 20), (70001, 64), (300001, 128)])
def test_hard_rows(dtype, v, k):
    K.case_hard_rows(DEV, dtype, v, k)


@pytest.mark.parametrize("v,k,rows", [(60, 20, 3), (1000, 128, 3), (3001, 129, 3),
                                      (12000, 400, 3), (70000, 90, 3), (70000, 1024, 2),
                                      (300000, 700, 2), (40000, 300, 300)])
def test_repeats(v, k, rows):
    K.case_repeats(DEV, v, k, rows)


@pytest.mark.parametrize("v", [2000, 40000])
def test_many_targets(v):
    K.case_many_targets(DEV, v)


@pytest.mark.parametrize("T", [1 / 1024, 1024.0])
@pytest.mark.parametrize("dtype", [K.F32, K.BF16, K.F16])
def test_temperatures(dtype, T):
    K.case_temperatures(DEV, dtype, T)


@pytest.mark.parametrize("dtype", [K.F32, K.BF16])
def test_windows_and_masks_off_their_boundaries(dtype):
    """Logits, mask and gradient whose rows start at every offset from a 16-byte boundary."""
    g = torch.Generator().manual_seed(7)
    for off in range(8):
        for width in (45, 1500, 6007):
            full = torch.randn(3, width + 16 + off % 3, generator=g).to(dtype).to(DEV)
            z = full[:, off:off + width].requires_grad_()
            m = torch.rand(3, width + 9, generator=g).to(DEV)[:, (5 * off) % 8:][:, :width] < 0.7
            t = C.make_targets(z.shape, None, 3, g).to(DEV)
            out = cb.profile_log_probs(z, t, top_k=6, mask=m)
            gs = dict(lp=torch.randn(t.shape, generator=g), h=torch.randn(3, generator=g),
                      norm=torch.randn(3, generator=g), top=torch.randn(3, 6, generator=g))
            gs = {n: v.to(DEV) for n, v in gs.items()}
            grad, = torch.autograd.grad(out[:4], z, tuple(gs.values()))
            C.check_scores(z, out, t, 6, m, None, 1.0, gs, grad)
            lp = out.top_log_probs.detach() - 0.1
            loss, grad = cb.distillation_loss_and_grad(z, out.top_indices, lp, mask=m)
            C.check_distill(z, out.top_indices, lp, False, m, None, 1.0, None, "mean", loss, grad)


@pytest.mark.parametrize("v,k,rows", [(61, 9, 9), (1003, 40, 9), (1003, 200, 9), (9005, 50, 9),
                                      (9005, 50, 600), (20011, 300, 600), (100003, 40, 5)])
@pytest.mark.parametrize("dtype", [K.F32, K.BF16, K.F16])
def test_ends(dtype, v, k, rows):
    K.case_ends(DEV, dtype, v, k, rows)
