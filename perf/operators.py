"""Cases that measure the operators on profile logits: log probabilities of given cells with
entropy and top alternatives (``profile_log_probs``), and distillation from a teacher's top
cells (``distillation_loss``, ``distillation_loss_and_grad``).

A row is one categorical distribution: the flattened channels and positions of one signal group
of one example (``groups`` gives the channels of each group), or, where ``groups`` is empty, the
last axis of a plain (rows, entries) matrix.
"""

import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
TRIM = 557      # the default model's trimming: its training path's logits are a window of a longer row


def listed():
    return [
        # one locus scored alone: where the most likely cut sites are and one read's likelihood
        dict(name="one_locus", op="score", dtype="fp32", n=1, groups="1", w=1000, s=1, k=8,
             t=1.0, mask=False, window=False),
        # the teacher's pass over a batch of the default model: its top cells are kept
        dict(name="teacher_pass", op="score", dtype="fp32", n=1024, groups="1", w=1000, s=16,
             k=32, t=1.0, mask=False, window=False),
        # reads of five assays at 2048 loci, unmappable positions masked
        dict(name="multitask_reads", op="score", dtype="fp32", n=2048, groups="1,2,2,2,2",
             w=1000, s=64, k=16, t=1.0, mask=True, window=False),
        # a single row of a large vocabulary, as one step of decoding sees it
        dict(name="one_long_row", op="score", dtype="bf16", n=1, groups="", w=131072, s=1, k=20,
             t=1.0, mask=False, window=False),
        # scoring given entries of a large, odd-sized vocabulary
        dict(name="many_long_rows", op="score", dtype="bf16", n=4096, groups="", w=50001, s=1,
             k=8, t=1.0, mask=False, window=False),
        # a training step on the likelihood of reads: logits are the model's trimmed window
        dict(name="reads_step", op="score_grad", dtype="fp32", n=1024, groups="1", w=1000, s=64,
             k=0, t=1.0, mask=False, window=True),
        # a policy or likelihood step with an entropy term on a large vocabulary
        dict(name="long_rows_step", op="score_grad", dtype="bf16", n=2048, groups="", w=65536,
             s=1, k=0, t=1.0, mask=False, window=False),
        # distillation of the default model, the loss and its gradient in one call
        dict(name="distill_locus", op="distill_step", dtype="fp32", n=1024, groups="1", w=1000,
             k=32, t=1.0, mask=False, window=False, renorm=False),
        # a small batch of a half-precision student
        dict(name="distill_few", op="distill_autograd", dtype="fp16", n=16, groups="1", w=1000,
             k=8, t=2.0, mask=False, window=True, renorm=True),
        # a masked multi-task student under autocast, through autograd
        dict(name="distill_multitask", op="distill_autograd", dtype="bf16", n=512,
             groups="1,2,2,2,2", w=1000, k=16, t=2.0, mask=True, window=False, renorm=True),
        # the largest step: a large vocabulary and many rows
        dict(name="distill_long_rows", op="distill_step", dtype="bf16", n=8192, groups="",
             w=32768, k=64, t=1.0, mask=False, window=False, renorm=False),
        # validation loss of long fp32 rows
        dict(name="distill_eval", op="distill_eval", dtype="fp32", n=1024, groups="", w=100003,
             k=100, t=1.5, mask=False, window=False, renorm=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["score", "score", "score_grad", "distill_step", "distill_autograd",
                     "distill_eval"])
    case = dict(op=op, dtype=rng.choice(["fp32", "bf16", "fp16"]))
    if rng.random() < 0.5:
        groups = [rng.choice([1, 1, 2, 2, 3]) for _ in range(rng.choice([1, 1, 2, 4, 5]))]
        case.update(n=_log_int(rng, 1, 2048), groups=",".join(map(str, groups)),
                    w=rng.randint(400, 2000), mask=rng.random() < 0.4,
                    window=rng.random() < 0.4)
    else:
        w = _log_int(rng, 60, 200000)
        case.update(n=_log_int(rng, 1, min(8192, 110000000 // w)), groups="", w=w,
                    mask=rng.random() < 0.25, window=False)
    case["t"] = rng.choice([1.0, 1.0, 0.7, 2.0])
    if op.startswith("score"):
        case.update(s=_log_int(rng, 1, 64), k=0 if op == "score_grad" else _log_int(rng, 1, 50))
    else:
        case.update(k=_log_int(rng, 1, 50), renorm=rng.random() < 0.5)
    return case


def _groups(case):
    return [int(c) for c in case["groups"].split(",")] if case["groups"] else []


# ------------------------------------------------------------------ inputs
def _smooth(x):
    """Neighbouring positions of a profile are alike."""
    return (x + x.roll(1, -1) + x.roll(-1, -1) + x.roll(2, -1) + x.roll(-2, -1)) * 0.45


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    groups, n, w, dt = _groups(case), case["n"], case["w"], DTYPES[case["dtype"]]
    if groups:
        shape, length = (n, sum(groups), w), w + (2 * TRIM if case["window"] else 0)
        base = _smooth(torch.randn(n, sum(groups), length, device=dev, generator=gen))
        # a few summits of several times the background
        base += 4.0 * (torch.rand(base.shape, device=dev, generator=gen) < 0.004)
        full = base.to(dt)
        logits = full[:, :, TRIM:TRIM + w] if case["window"] else full
    else:
        shape = (n, w)
        base = torch.randn(n, w, device=dev, generator=gen) * 2.0
        # how sure a row is differs from row to row
        base[:, :: max(1, w // 37)] += 8.0 * torch.rand(n, 1, device=dev, generator=gen)
        logits = base.to(dt)
    state = dict(case=case, groups=groups, logits=logits)
    state["mask"] = None
    if case["mask"]:       # True where a cell takes part; one row in 50 has none
        state["mask"] = torch.rand(shape, device=dev, generator=gen) < 0.9
        dead = torch.rand(n, device=dev, generator=gen) < 0.02
        state["mask"] &= ~dead.view(-1, *([1] * (len(shape) - 1)))
    lead = (n, len(groups)) if groups else (n,)
    # half-precision gradients are scaled up, as a loss scaler does, or they would vanish
    scale = 256.0 * n * max(1, len(groups)) if dt == torch.float16 else 1.0
    sizes = [g * w for g in groups] or [w]
    if case["op"].startswith("score"):
        u = torch.rand(*lead, case["s"], device=dev, generator=gen)
        size = torch.tensor(sizes, device=dev)
        size = size.view(1, -1, 1) if groups else size.view(1, 1)
        t = (u * size).long().clamp_(max=max(sizes) - 1)
        t = torch.minimum(t, size - 1)
        # rows have fewer targets than the widest one: the places behind are empty (-1)
        if case["s"] > 1:
            t[torch.rand(t.shape, device=dev, generator=gen) < 0.1] = -1
        state["targets"] = t
        if case["op"] == "score_grad":
            state["g_lp"] = torch.randn(t.shape, device=dev, generator=gen) * (scale / n)
            state["g_h"] = torch.full(lead, 0.01 * scale / n, device=dev)
    else:
        # the teacher: a model that is near the student; its top cells, as they were stored
        k, T = case["k"], case["t"]
        noise = torch.randn(base.shape, device=dev, generator=gen).mul_(0.7)
        teach = noise.add_(base).div_(T)
        if groups and case["window"]:
            teach = teach[:, :, TRIM:TRIM + w]
        del noise
        parts = torch.split(teach, groups, dim=1) if groups else (teach,)
        vals, idxs = [], []
        for p in parts:
            top, at = p.reshape(n, -1).log_softmax(-1).topk(min(k, p[0].numel()), dim=-1)
            vals.append(torch.nn.functional.pad(top, (0, k - top.shape[1]), value=-math.inf))
            idxs.append(torch.nn.functional.pad(at, (0, k - at.shape[1]), value=-1))
        state["t_lp"] = torch.stack(vals, 1) if groups else vals[0]
        state["t_idx"] = torch.stack(idxs, 1) if groups else idxs[0]
        state["weight"] = (0.5 + torch.rand(lead, device=dev, generator=gen)) * scale
    if case["op"] in ("score_grad", "distill_autograd"):
        state["logits"] = state["logits"].detach().requires_grad_()
    return state


# ------------------------------------------------------------------ the plain form, in 32 bits
def _cells(state):
    """Which entry of the flattened logits each (group, place) is, and which places there are."""
    groups, w = state["groups"], state["case"]["w"]
    dev = state["logits"].device
    size = torch.tensor(groups, device=dev) * w
    place = torch.arange(max(groups) * w, device=dev)
    keep = place < size[:, None]
    return ((size.cumsum(0) - size)[:, None] + place).clamp_(max=sum(groups) * w - 1), keep


def _rows(state):
    """The rows' logits over the temperature, -inf where nothing is: (..., entries)."""
    z = state["logits"].detach()
    mask = state["mask"]
    if state["groups"]:
        n = z.shape[0]
        at, keep = _cells(state)
        z = z.reshape(n, -1)[:, at].float()
        if mask is not None:
            keep = keep & mask.reshape(n, -1)[:, at]
        z = torch.where(keep, z, -math.inf)
    else:
        z = z.float()
        if mask is not None:
            z = torch.where(mask, z, -math.inf)
    return z / state["case"]["t"] if state["case"]["t"] != 1.0 else z


def _back(state, grad):
    """The rows' gradient in the logits' layout and type."""
    logits = state["logits"]
    if state["groups"]:
        grad = grad[:, _cells(state)[1]].reshape(logits.shape)
    return grad.to(logits.dtype)


def _sums(z):
    m = z.amax(-1, keepdim=True)
    m = torch.where(m == -math.inf, 0.0, m)
    e = torch.exp(z - m)
    return m, e, e.sum(-1, keepdim=True)


def _top(z, k):
    """The k largest entries, ties to the lowest index, -1 and -inf where there are fewer."""
    bits = z.view(torch.int32).long()
    order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
    size = z.shape[-1]
    key = order * (1 << 31) + (size - 1 - torch.arange(size, device=z.device))
    got = key.topk(k, dim=-1).values
    at = size - 1 - (got & 0x7FFFFFFF)
    top = z.gather(-1, at)
    return top, torch.where(top == -math.inf, -1, at)


def _score(state, z):
    m, e, s = _sums(z)
    lse = (m + torch.log(s))
    x = torch.where(e > 0, z - m, 0.0)
    h = (torch.log(s) - (e * x).sum(-1, keepdim=True) / s).squeeze(-1)
    h = torch.where(s.squeeze(-1) > 0, h, 0.0)
    t = state["targets"]
    zt = z.gather(-1, t.clamp(min=0))
    lp = torch.where(t < 0, 0.0, torch.where(zt == -math.inf, zt, zt - lse))
    return lp, h, lse, e, s


def _score_grad(state, z):
    lp, h, lse, e, s = _score(state, z)
    t, temp = state["targets"], state["case"]["t"]
    g = torch.where((t < 0) | (lp == -math.inf), 0.0, state["g_lp"])
    gh = state["g_h"].unsqueeze(-1)
    q = torch.where(s > 0, e / s, 0.0)
    logq = torch.where(q > 0, z - lse, 0.0)
    d = q * (-g.sum(-1, keepdim=True) - gh * (logq + h.unsqueeze(-1)))
    d.scatter_add_(-1, t.clamp(min=0), g)
    return lp, h, _back(state, d / temp)


def _distill(state, z, want_grad):
    case, t = state["case"], state["case"]["t"]
    idx, w = state["t_idx"], state["weight"].unsqueeze(-1)
    zu = z.gather(-1, idx.clamp(min=0))
    there = (idx >= 0) & (zu > -math.inf)
    lp = torch.where(there, state["t_lp"].double(), -math.inf)   # the rest's mass is 1 minus a sum
    u = torch.zeros(z.shape, dtype=torch.int32, device=z.device)
    u.scatter_add_(-1, idx.clamp(min=0), there.int())
    rest = torch.where(u > 0, -math.inf, z)
    m, e, s = _sums(rest)
    has = s > 0
    lse_r = torch.where(has, m + torch.log(s), -math.inf)
    zu = torch.where(there, zu, -math.inf)
    both = torch.cat([zu, lse_r], -1)
    top, e_u, s_u = _sums(both)
    lse = top + torch.log(s_u)
    p = torch.exp(lp)
    mass = p.sum(-1, keepdim=True)
    whole = (mass > 1) | ~has
    if case["renorm"]:
        whole = torch.ones_like(whole)
    p = torch.where(whole & (mass > 0), p / mass, p)
    p_r = torch.where(whole, 0.0, 1 - mass)
    live = (s_u > 0) & ((mass > 0) | ~whole)
    logq = torch.where(there, zu - lse, 0.0)
    logq_r = torch.where(has, lse_r - lse, 0.0)
    loss = (torch.where(p > 0, p * (torch.log(p) - logq), 0.0).sum(-1, keepdim=True)
            + torch.where(p_r > 0, p_r * (torch.log(p_r) - logq_r), 0.0))
    loss = torch.where(live, loss, 0.0) * (t * t) * w
    loss = (loss.sum() / w.numel()).float()
    if not want_grad:
        return loss
    scale = torch.where(live, w * (t / w.numel()), 0.0)
    q_r = torch.where(has, e_u[..., -1:] / s_u, 0.0)
    d = torch.where(has, e / s, 0.0) * (scale * (q_r - p_r)).float()
    d_u = torch.where(there & live, scale * (e_u[..., :-1] / s_u - p), 0.0).float()
    d.scatter_add_(-1, idx.clamp(min=0), d_u)
    return loss, _back(state, d)


# ------------------------------------------------------------------ one pass
def run(state):
    case, op = state["case"], state["case"]["op"]
    if own:
        return _run_own(state)
    z = _rows(state)
    if op == "score":
        lp, h, lse, _, _ = _score(state, z)
        top, at = _top(z, case["k"])
        return dict(log_probs=lp, entropy=h,
                    top_log_probs=torch.where(at < 0, -math.inf, top - lse), top_indices=at)
    if op == "score_grad":
        lp, h, grad = _score_grad(state, z)
        return dict(log_probs=lp, entropy=h, grad=grad)
    if op == "distill_eval":
        return dict(loss=_distill(state, z, False))
    loss, grad = _distill(state, z, True)
    return dict(loss=loss, grad=grad)


def _run_own(state):
    import cherimoya_b200 as cherimoya

    case, op, logits = state["case"], state["case"]["op"], state["logits"]
    how = dict(mask=state["mask"], signal_groups=state["groups"] or None, temperature=case["t"])
    if op == "score":
        out = cherimoya.profile_log_probs(logits, state["targets"], top_k=case["k"], **how)
        return dict(log_probs=out.log_probs, entropy=out.entropy,
                    top_log_probs=out.top_log_probs, top_indices=out.top_indices)
    if op == "score_grad":
        out = cherimoya.profile_log_probs(logits, state["targets"], **how)
        grad, = torch.autograd.grad((out.log_probs, out.entropy), logits,
                                    (state["g_lp"], state["g_h"]))
        return dict(log_probs=out.log_probs.detach(), entropy=out.entropy.detach(), grad=grad)
    teacher = (state["t_idx"], state["t_lp"])
    how.update(weight=state["weight"], renormalize=case["renorm"])
    if op == "distill_eval":
        return dict(loss=cherimoya.distillation_loss(logits, *teacher, **how))
    if op == "distill_autograd":
        loss = cherimoya.distillation_loss(logits, *teacher, **how)
        grad, = torch.autograd.grad(loss, logits)
        return dict(loss=loss.detach(), grad=grad)
    loss, grad = cherimoya.distillation_loss_and_grad(logits, *teacher, **how)
    return dict(loss=loss, grad=grad)


def work(case):
    groups = _groups(case)
    rows = case["n"] * max(1, len(groups))
    cells = case["n"] * (sum(groups) if groups else 1) * case["w"]
    b = 4 if case["dtype"] == "fp32" else 2
    moved, flops = cells * (b + (1 if case["mask"] else 0)), 6 * cells
    if case["op"].startswith("score"):
        moved += rows * (case["s"] * 12 + 4 + case["k"] * 12)
    else:
        moved += rows * (case["k"] * 12 + 4)
    if case["op"] not in ("score", "distill_eval"):
        moved += cells * b
        flops += 4 * cells
    return {"bytes": moved, "flops": flops}


# ------------------------------------------------------------------ the definition, in 64 bits
def exact(case, seed):
    state = prepare(case, seed)
    groups, n, w, T = state["groups"], case["n"], case["w"], case["t"]
    logits = state["logits"].detach()
    mask = state["mask"] if state["mask"] is not None else None
    outs, at = [], 0
    for g, c in enumerate(groups or [None]):
        z = logits if c is None else logits[:, at:at + c].reshape(n, c * w)
        a = None if mask is None else mask if c is None else mask[:, at:at + c].reshape(n, c * w)
        at += c or 0
        pick = (lambda v: v) if c is None else (lambda v, g=g: v[:, g])
        step = max(1, (1 << 26) // z.shape[1])
        parts = []
        for r in range(0, n, step):
            sl = slice(r, r + step)
            zz = z[sl].double() / T
            if a is not None:
                zz = zz.masked_fill(~a[sl], -math.inf)
            if case["op"].startswith("score"):
                parts.append(_exact_score(state, case, zz, pick, sl))
            else:
                parts.append(_exact_distill(state, case, zz, pick, sl, n * max(1, len(groups))))
        outs.append({k: torch.cat([p[k] for p in parts]) for k in parts[0]})
    res = {}
    for k in outs[0]:
        if k == "loss":
            res[k] = sum(o[k].sum() for o in outs)
        elif k == "grad":
            res[k] = outs[0][k] if not groups else torch.cat(
                [o[k].reshape(n, c, w) for o, c in zip(outs, groups)], 1)
        else:
            res[k] = outs[0][k] if not groups else torch.stack([o[k] for o in outs], 1)
    return res


def _exact_score(state, case, z, pick, sl):
    logq = torch.log_softmax(z, -1)
    logq = torch.where(z == -math.inf, -math.inf, logq)
    q = logq.exp()
    h = -torch.special.xlogy(q, q).sum(-1)
    t = pick(state["targets"])[sl]
    lp = logq.gather(-1, t.clamp(min=0)).masked_fill(t < 0, 0.0)
    out = dict(log_probs=lp, entropy=h)
    if case["op"] == "score":
        top, at = torch.sort(logq, dim=-1, descending=True, stable=True)
        # equal logits give equal log probabilities, so a stable sort keeps their order
        top, at = top[:, :case["k"]], at[:, :case["k"]]
        out.update(top_log_probs=top.clone(), top_indices=at.masked_fill(top == -math.inf, -1))
        return out
    g = pick(state["g_lp"])[sl].double().masked_fill((t < 0) | torch.isinf(lp), 0.0)
    gh = pick(state["g_h"])[sl].double()[:, None]
    grad = -q * g.sum(-1, keepdim=True) - gh * (torch.special.xlogy(q, q) + q * h[:, None])
    grad.scatter_add_(-1, t.clamp(min=0), g)
    out["grad"] = grad / case["t"]
    return out


def _exact_distill(state, case, z, pick, sl, rows):
    idx = pick(state["t_idx"])[sl]
    lp = pick(state["t_lp"])[sl].double()
    wt = pick(state["weight"])[sl].double() / rows
    logq = torch.log_softmax(z, -1)
    logq = torch.where(z == -math.inf, -math.inf, logq)
    gone = (idx < 0) | torch.isinf(logq.gather(-1, idx.clamp(min=0)))
    lp = lp.masked_fill(gone, -math.inf)
    top = torch.zeros_like(z).scatter_add_(-1, idx.clamp(min=0), lp.exp())
    inside = torch.zeros_like(z).scatter_add_(-1, idx.clamp(min=0), (~gone).double()) > 0
    outside = (z > -math.inf) & ~inside
    some = outside.any(-1)
    mass = top.sum(-1)
    full = torch.ones_like(some) if case["renorm"] else (mass > 1) | ~some
    live = (z > -math.inf).any(-1) & ((mass > 0) | ~full)
    top = torch.where((full & (mass > 0))[:, None], top / mass[:, None], top)
    p_r = torch.where(full, 0.0, 1 - mass)
    logq_r = torch.logsumexp(logq.masked_fill(~outside, -math.inf), -1)
    safe = torch.where(inside, logq, 0.0)
    loss = (torch.special.xlogy(top, top) - top * safe).sum(-1)
    loss = loss + torch.special.xlogy(p_r, p_r) - p_r * torch.where(some, logq_r, 0.0)
    loss = torch.where(live, loss, 0.0) * case["t"] ** 2 * wt
    out = dict(loss=loss)
    if case["op"] != "distill_eval":
        share = torch.where(outside, (logq - torch.where(some, logq_r, 0.0)[:, None]).exp(), 0.0)
        grad = logq.exp() - top - share * p_r[:, None]
        out["grad"] = grad * (torch.where(live, wt, 0.0) * case["t"])[:, None]
    return out
