"""Inputs, the 64-bit comparison and its error bounds, shared by the CPU and the GPU
tests of the likelihood and distillation operators.

Bounds, with u = 2^-24 (half a step of fp32), x = (z - m) / T of an entry and m the
row's maximum. z - m, 1/T and their product round once each: x is off by 3u|x|. The
hardware exp2 is off by at most 4u relative, so a term of the sum s is off by
(4 + 3|x|)u; weighted with the terms, |x| averages to at most the log of the row's
length (14 for 2^20 entries), which makes 46u. Each partial sum has at most 64 terms
in a row before partial sums of equal weight are joined (another 16 roundings), 80u.
log s is off by that and by 2u of itself, a result (x - log s) by one rounding more:
in all  u (4|x| + 4|log s| + 128).  CHAIN below is those 128, and products of a few such
factors (probability times coefficient) are within twice that.
"""

import math

import torch

import cherimoya_b200 as cb
from oracle import likelihood_oracle as LO

U = 2.0 ** -24
CHAIN = 128
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -24}


def logits(shape, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(*shape, generator=g) * scale
    return z.to(dtype), g


def lead_of(shape, groups):
    return tuple(shape[:-1]) if groups is None else (shape[0], len(groups))


def sizes_of(shape, groups):
    return [shape[-1]] if groups is None else [c * shape[2] for c in groups]


def make_targets(shape, groups, count, g, empty=0.1):
    lead, sizes = lead_of(shape, groups), sizes_of(shape, groups)
    size = torch.tensor(sizes if groups is not None else sizes[0]).expand(lead).unsqueeze(-1)
    t = (torch.rand(*lead, count, generator=g) * size).long().clamp(min=0)
    t = torch.minimum(t, (size - 1).clamp(min=0))
    t[torch.rand(t.shape, generator=g) < empty] = -1
    if min(sizes) == 0:
        t.fill_(-1)
    return t


def make_teacher(z, groups, k, T, g, noise=0.7):
    """A teacher near the student: its top k cells and log probabilities, -1 behind."""
    teach = z.double() + noise * torch.randn(z.shape, generator=g).double()
    vals, idxs = [], []
    for row in LO.split_rows(teach / T, groups):
        row = torch.where(torch.isfinite(row), row, -math.inf)
        n = min(k, row.numel())
        top, at = torch.log_softmax(row, -1).topk(n) if n else (row[:0], row[:0].long())
        top = torch.where(torch.isfinite(top), top, -50.0)
        vals.append(torch.nn.functional.pad(top, (0, k - n), value=-math.inf))
        idxs.append(torch.nn.functional.pad(at, (0, k - n), value=-1))
    lead = lead_of(z.shape, groups)
    return (torch.stack(idxs).reshape(lead + (k,)),
            torch.stack(vals).float().reshape(lead + (k,)))


def same(got, want, tol, what):
    """got (fp32 or lower) against want (64 bits): equal where not finite, else within tol."""
    got, want = got.double().cpu().reshape(-1), torch.as_tensor(want).double().reshape(-1)
    tol = torch.as_tensor(tol).double().reshape(-1).expand_as(want)
    want = torch.where(want.abs() > torch.finfo(torch.float32).max, want * math.inf, want)
    odd = ~torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), what
    inf = odd & ~torch.isnan(want)
    assert torch.equal(got[inf], want[inf]), what
    off = (got - want).abs()[~odd] - tol[~odd]
    assert off.numel() == 0 or float(off.max()) <= 0, "{}: {:.3g} beyond the bound".format(
        what, float(off.max()))


def check_scores(z, out, targets, top_k, mask, groups, T, g=None, grad=None):
    """profile_log_probs' results (and the gradient of <g, results>) against the oracle."""
    zc, tc = z.detach().cpu(), targets.cpu()
    mc = mask.cpu().expand(zc.shape) if mask is not None else None
    rows = LO.split_rows(zc, groups)
    masks = LO.split_rows(mc, groups) if mc is not None else [None] * len(rows)
    R = len(rows)
    tr = tc.reshape(R, tc.shape[-1])
    flat = {k: v.detach().cpu().reshape((R,) + v.shape[len(out.entropy.shape):])
            for k, v in out._asdict().items()}
    grads = LO.split_rows(grad.cpu(), groups) if grad is not None else None
    for r in range(R):
        gr = None
        if g is not None:
            gr = {k: v.cpu().reshape(R, -1)[r] for k, v in g.items()}
            gr["h"], gr["norm"] = gr["h"][0], gr["norm"][0]
        o = LO.score_row(rows[r], masks[r], tr[r], top_k, T, gr)
        what = "row {}".format(r)
        log_s = abs(o["log_s"])
        base = U * (4 * log_s + CHAIN)
        lp = torch.tensor(o["log_probs"], dtype=torch.float64)
        same(flat["log_probs"][r], lp, base + 4 * U * lp.abs().nan_to_num(0, 0, 0), what + " lp")
        top = torch.tensor(o["top"], dtype=torch.float64)
        same(flat["top_log_probs"][r], top, base + 4 * U * top.abs().nan_to_num(0, 0, 0),
             what + " top")
        assert flat["top_indices"][r].tolist() == o["at"], what + " indices"
        norm = o["log_normalizer"]
        same(flat["log_normalizer"][r], norm, base + (4 * U * abs(norm) if math.isfinite(norm)
                                                      else 0), what + " normaliser")
        h = o["entropy"]
        same(flat["entropy"][r], h, 2 * base * (1 + (abs(h) if math.isfinite(h) else 0)),
             what + " entropy")
        if grads is not None:
            d = o["grad"]
            tol = HALF_STEP[z.dtype] * d.abs() + 2 * CHAIN * U * o["grad_mag"] + TINY[z.dtype]
            same(grads[r], d, tol.nan_to_num(0), what + " gradient")


def check_distill(z, idx, t_lp, renorm, mask, groups, T, weight, reduction, loss, grad, upstream=1.0):
    zc = z.detach().cpu()
    rows = LO.split_rows(zc, groups)
    R = len(rows)
    mc = mask.cpu().expand(zc.shape) if mask is not None else None
    masks = LO.split_rows(mc, groups) if mc is not None else [None] * R
    ir, lr = idx.cpu().reshape(R, -1), t_lp.cpu().reshape(R, -1)
    w = weight.cpu().reshape(R).double() if weight is not None else torch.ones(R).double()
    grads = LO.split_rows(grad.cpu(), groups) if grad is not None else None
    scale = (1.0 / R if reduction == "mean" else 1.0)
    losses, mags = [], []
    up = torch.as_tensor(upstream).double().cpu().reshape(-1).expand(R)
    for r in range(R):
        l, lm, d, dm = LO.distill_row(rows[r], masks[r], ir[r], lr[r], renorm, T, float(w[r]))
        losses.append(l * scale)
        mags.append(lm * scale)
        if grads is not None:
            f = scale * float(up[r])
            d, dm = d * f, dm * abs(f)
            tol = HALF_STEP[z.dtype] * d.abs() + 2 * CHAIN * U * dm + TINY[z.dtype]
            same(grads[r], d, tol.nan_to_num(0), "row {} gradient".format(r))
    losses, mags = torch.tensor(losses).double(), torch.tensor(mags).double()
    # a row's loss is a sum of terms P (log P - log q), each log q off by the bound above;
    # the probabilities sum to 1
    tol = 2 * CHAIN * U * (mags + w.abs().nan_to_num(0) * scale * T * T)
    if reduction == "none":
        same(loss, losses, tol, "losses")
    else:
        same(loss, losses.sum(), tol.sum() + U * losses.sum().abs().nan_to_num(0), "loss")
