"""64-bit restatement of the likelihood and distillation operators, one row at
a time, from their definitions. Test oracle only.

Each function also returns a magnitude per result: the sum of the absolute
values of what is added up, which the tests' error bounds are stated in."""

import math

import torch

NAN, INF = float("nan"), float("inf")


def split_rows(x, groups):
    """List of (index in the flat row order, flat row) of a tensor laid out as the logits."""
    if groups is None:
        flat = x.reshape(-1, x.shape[-1]) if x.numel() else x.reshape(x.shape[0], -1)
        return list(flat)
    rows = []
    for n in range(x.shape[0]):
        c = 0
        for g in groups:
            rows.append(x[n, c:c + g].reshape(-1))
            c += g
    return rows


def _row(z, mask, T):
    z = z.double().clone()
    if mask is not None:
        z[~mask] = -INF
    part = z != -INF
    return z, part, bool((torch.isnan(z) | (z == INF)).any())


def score_row(z, mask, targets, top_k, T, g=None):
    """dict of log_probs, entropy, log_normalizer, top, at (+ grad with g: dict of
    lp, h, norm, top), each with a magnitude."""
    z, part, bad = _row(z, mask, T)
    V = z.numel()
    x = z / T
    nothing = not bool(part.any())
    if bad:
        lse, logq, log_s = NAN, torch.full_like(x, NAN), 0.0
    elif nothing:
        lse, logq, log_s = -INF, torch.full_like(x, -INF), 0.0
    else:
        m = float(x.max())
        log_s = math.log(float(torch.exp(x - m).sum()))
        lse, logq = m + log_s, (x - m) - log_s     # rows at 1e38 keep their log_s
    q = torch.where(part, torch.exp(logq), 0.0)
    h = NAN if bad else 0.0 if nothing else float(-(q[q > 0] * logq[q > 0]).sum())
    out = dict(entropy=h, log_normalizer=lse, log_s=log_s)
    lp = []
    for t in targets.tolist():
        if t < 0:
            lp.append(0.0)
        elif bad or t >= V:
            lp.append(NAN)
        else:
            lp.append(float(logq[t]) if bool(part[t]) else -INF)
    out["log_probs"] = lp
    order = [] if bad else sorted((int(v) for v in torch.nonzero(part).reshape(-1)),
                                  key=lambda v: (-float(z[v]), v))[:top_k] if V < 5000 else \
        [v for v in torch.sort(z, descending=True, stable=True)[1][:top_k].tolist() if part[v]]
    out["at"] = order + [-1] * (top_k - len(order))
    out["top"] = [float(logq[v]) for v in order] + [NAN if bad else -INF] * (top_k - len(order))
    if g is not None:
        d, mag = torch.zeros_like(x), torch.zeros_like(x)
        spots = [(t, float(gi), lp[i]) for i, (t, gi) in enumerate(zip(targets.tolist(), g["lp"]))]
        spots += [(t, float(gi), 0.0) for t, gi in zip(out["at"], g["top"])]
        a, amag = float(g["norm"]), abs(float(g["norm"]))
        for t, gi, value in spots:
            if t < 0:
                continue
            if t >= V:
                a = NAN
                continue
            if not bool(part[t]) and not bad:
                continue
            a -= gi
            amag += abs(gi)
            d[t] += gi
            mag[t] += abs(gi)
        lq = torch.where(q > 0, logq, 0.0)
        gh = float(g["h"])
        d = d + q * (a - gh * (lq + h))
        mag = mag + q * (amag + abs(gh) * (lq.abs() + abs(h)))
        if bad:
            d = torch.full_like(x, NAN)
        out["grad"] = torch.where(part, d / T, 0.0)
        out["grad_mag"] = torch.where(part, mag / T, 0.0)
    return out


def distill_row(z, mask, idx, t_lp, renormalize, T, weight=1.0):
    """(loss, its magnitude, gradient, its magnitude) of one row."""
    zero = torch.zeros(z.numel(), dtype=torch.float64)
    if weight == 0:
        return 0.0, 0.0, zero, zero
    z, part, bad = _row(z, mask, T)
    V = z.numel()
    mass = {}
    for i, lp in zip(idx.tolist(), t_lp.double().tolist()):
        if i < 0:
            continue
        if i >= V:
            bad = True
            continue
        if not bool(part[i]):
            continue
        if not lp < INF:
            bad = True
        mass.setdefault(i, []).append(lp)
    if bad or weight != weight:
        nan = torch.where(part, NAN, 0.0).double()
        return NAN, 0.0, nan, zero
    if not bool(part.any()):
        return 0.0, 0.0, zero, zero
    x = z / T
    m = float(x.max())
    log_s = math.log(float(torch.exp(x - m).sum()))
    listed = torch.zeros(V, dtype=torch.bool)
    listed[list(mass)] = True
    rest = part & ~listed
    shift = max((lp for lps in mass.values() for lp in lps), default=0.0) if renormalize else 0.0
    shift = 0.0 if shift == -INF else shift
    P = {i: sum(math.exp(lp - shift) for lp in lps) for i, lps in mass.items()}
    total = math.fsum(P.values())
    whole = renormalize or total > 1 or not bool(rest.any())
    if whole:
        if total <= 0:
            return 0.0, 0.0, zero, zero
        P = {i: p / total for i, p in P.items()}
        p_r = 0.0
    else:
        p_r = 1.0 - total
    logq = torch.where(part, (x - m) - log_s, -INF)
    loss = mag = 0.0
    for i, p in P.items():
        if p > 0:
            loss += p * (math.log(p) - float(logq[i]))
            mag += p * (abs(math.log(p)) + abs(float(logq[i])))
    d = torch.exp(logq)
    dmag = d.clone()
    if bool(rest.any()):
        xr = x[rest]
        mr = float(xr.max())
        s_r = float(torch.exp(xr - mr).sum())
        log_qr = (mr - m) + math.log(s_r) - log_s
        if p_r > 0:
            loss += p_r * (math.log(p_r) - log_qr)
            mag += p_r * (abs(math.log(p_r)) + abs(log_qr))
        share = torch.where(rest, torch.exp(x - mr) / s_r, 0.0)
        d = d - share * p_r
        dmag = dmag + share * p_r
    for i, p in P.items():
        d[i] = d[i] - p
        dmag[i] += p
    w = float(weight)
    return loss * T * T * w, mag * T * T * abs(w), d * T * w, dmag * T * abs(w)
