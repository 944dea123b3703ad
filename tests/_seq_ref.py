"""Plain float64 restatements of the sequence and output operators, and bounds for their rounding errors.

Rounding: a value rounded to a type is off by at most half a step, eps / 2 relative (U below for fp32, HALF[dtype] for the output).  A quantity
that is a sum of products with at most n roundings on the way of each term is off by at most n U times the same sum of absolute values
(first order; the factor 1.01 covers the higher ones)."""
import numpy as np
import torch

U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}      # half a step of the smallest numbers, at most


def fold(v, shape):
    """Sum over the axes a gate of `shape` does not have."""
    for d in range(4):
        if shape[d] == 1 and v.shape[d] != 1:
            v = v.sum(axis=d, keepdims=True)
    return v


def recurrence(u, qc, qh, z0, lengths, dz, dzT):
    """All outputs and gradients of z_t = qc_t z_{t-1} + qh_t u_t in float64 (numpy), step by step."""
    B, T, H, N = u.shape
    a = np.broadcast_to(qc, u.shape)
    q = np.ones_like(u) if qh is None else np.broadcast_to(qh, u.shape)
    live = np.arange(T)[None, :] < np.clip(np.full(B, T) if lengths is None else lengths, 0, T)[:, None]
    z, prev = np.zeros_like(u), np.zeros_like(u)
    h = np.zeros((B, H, N)) if z0 is None else z0.copy()
    for t in range(T):
        m = live[:, t][:, None, None]
        prev[:, t] = h
        with np.errstate(invalid="ignore"):
            h = np.where(m, a[:, t] * h + q[:, t] * u[:, t], h)
        z[:, t] = np.where(m, h, 0.0)
    zT = h
    r = np.zeros((B, H, N)) if dzT is None else dzT.copy()
    da, dq, du = np.zeros_like(u), np.zeros_like(u), np.zeros_like(u)
    for t in range(T - 1, -1, -1):
        m = live[:, t][:, None, None]
        with np.errstate(invalid="ignore"):
            g = r + (0.0 if dz is None else np.where(m, dz[:, t], 0.0))
            da[:, t], dq[:, t], du[:, t] = np.where(m, g * prev[:, t], 0), np.where(m, g * u[:, t], 0), np.where(m, g * q[:, t], 0)
            r = np.where(m, a[:, t] * g, r)
    return dict(z=z, zT=zT, du=du, dq_check=fold(da, qc.shape), dq_hat=None if qh is None else fold(dq, qh.shape), dz0=r)


def recurrence_bounds(u, qc, qh, z0, lengths, dz, dzT, dtype):
    """What each output may be off by: the same sums of absolute values times the number of roundings of a term (a state: at most 2 per step
    and 16 for the joins; a gradient: two such chains and the sum over the axes the gate lacks), plus the output's own rounding."""
    ab = [None if v is None else np.abs(v) for v in (u, qc, qh, z0)]
    m = recurrence(*ab, lengths, None if dz is None else np.abs(dz), None if dzT is None else np.abs(dzT))
    T = u.shape[1]
    n = dict(z=2 * T + 32, zT=2 * T + 32, du=2 * T + 32, dz0=2 * T + 32)
    for k, g in (("dq_check", qc), ("dq_hat", qh)):
        if g is not None:
            n[k] = 4 * T + 64 + u.size // max(1, g.size)
    return {k: None if m[k] is None else 1.01 * n[k] * U * m[k] + (HALF[dtype] * 1.01 * m[k] + TINY[dtype] if k in ("z", "du", "dq_check", "dq_hat") else 0.0)
            for k in m}


# ---- tokens and distillation: definitions in float64, row by row, with bounds -------------------------------------------------------
FLUSH = 2.0 ** -126  # the exponential gives zero for results below 2^-126: a probability is off by less than that, its gradient by that times its weight
NSUM = 320           # roundings of a term of a row's sums, at most: 64 in a thread, 10 in a workgroup, the tiles' joins, the exponential's own


def _row(x, c):
    """Row in float64: (y = c (x - M), log sum, p, lp); a row of nothing but -inf has p = 0, lp = -inf, log sum 0."""
    M = x.max()
    if M == -np.inf:
        return np.full_like(x, -np.inf), 0.0, np.zeros_like(x), np.full_like(x, -np.inf)
    y = c * (x - M)
    ls = np.log(np.exp(y).sum())
    return y, ls, np.exp(y - ls), y - ls


def _sum_err(y, p):
    """Relative error of a row's sum of exponentials: its roundings, and each exponent's (difference, scaled c, product: 3 of |y|)."""
    yy = np.where(p > 0, np.abs(y), 0.0)
    return U * (NSUM + 4.0 * (p * yy).sum())


def order(x):
    """Indices by descending value, equal ones ascending, NaN first."""
    key = np.where(np.isnan(x), np.inf, x)
    return np.lexsort((np.arange(x.size), -key, ~np.isnan(x)))


def tokens(x, tok, top, T, ignore, dlogp, dent, dtop, half):
    """(values, bounds) of every output and of dlogits for logits x [R, V] (float64 of the tested type's values)."""
    R, V = x.shape
    c = 1.0 / T
    out = dict(logp=np.zeros(R), entropy=np.zeros(R), top_logp=np.zeros((R, top)), top_tokens=np.zeros((R, top), dtype=np.int64), dlogits=np.zeros((R, V)))
    tol = {k: np.zeros_like(v, dtype=np.float64) for k, v in out.items()}
    for r in range(R):
        y, ls, p, lp = _row(x[r], c)
        empty = not (p > 0).any()
        ya = np.where(p > 0, np.abs(y), 0.0)
        es = _sum_err(y, p)
        dlp = U * 4 * np.where(np.isfinite(y), np.abs(y), 0.0) + es + 3 * U * abs(ls)          # of a log probability
        H = -(p * np.where(p > 0, lp, 0.0)).sum()
        dH = es + 3 * U * abs(ls) + (p * ya * (U * 4 * ya + U * NSUM)).sum() + (p * ya).sum() * es + 2 * U * abs(H)
        out["entropy"][r], tol["entropy"][r] = H, dH
        given = tok[r] != ignore
        if given:
            out["logp"][r], tol["logp"][r] = lp[tok[r]], dlp[tok[r]] + (U * abs(lp[tok[r]]) if np.isfinite(lp[tok[r]]) else 0.0)
        best = order(x[r])[:top]
        out["top_tokens"][r] = best
        out["top_logp"][r] = lp[best]
        tol["top_logp"][r] = dlp[best] + U * np.where(np.isfinite(lp[best]), np.abs(lp[best]), 0.0)
        if empty:
            continue
        w = np.zeros(V)
        wa = np.zeros(V)
        if given and dlogp is not None:
            w[tok[r]] += dlogp[r]
            wa[tok[r]] += abs(dlogp[r])
        if dtop is not None:
            w[best] += dtop[r]
            wa[best] += np.abs(dtop[r])
        gH = 0.0 if dent is None else dent[r]
        lpz = np.where(p > 0, lp, 0.0)
        d = c * (w - p * w.sum() - gH * p * (lpz + H))
        rel = dlp + 8 * U
        err = c * (p * (rel * (abs(w.sum()) + abs(gH) * np.abs(lpz + H)) + (top + 4) * U * wa.sum() + abs(gH) * (dlp + dH + 4 * U * (np.abs(lpz) + H)))
                   + 6 * U * wa + FLUSH * (abs(w.sum()) + abs(gH) * (np.abs(lpz) + H)))
        out["dlogits"][r], tol["dlogits"][r] = d, 1.05 * err + half[0] * 1.01 * np.abs(d) + half[1]
    return out, tol


def distill(x, idx, val, T, tail, dloss, half):
    R, V = x.shape
    c = 1.0 / T
    out, tol = dict(loss=np.zeros(R), dlogits=np.zeros((R, V))), dict(loss=np.zeros(R), dlogits=np.zeros((R, V)))
    for r in range(R):
        ok = (idx[r] >= 0) & (idx[r] < V)
        i, v = idx[r][ok], val[r][ok]
        if i.size == 0 or (not tail and (v == -np.inf).all()):
            continue
        y, ls, q, lq = _row(x[r], c)
        if tail:
            p, dp = np.exp(v), np.zeros_like(v)
            named = np.zeros(V, dtype=bool)
            named[i] = True
            pr, qr = max(0.0, 1.0 - p.sum()), q[~named].sum()
        else:
            dv = c * (v - v.max())
            p = np.exp(dv)
            p /= p.sum()
            da = np.where(p > 0, np.abs(dv), 0.0)
            dp = 2 * U * (da + (p * da).sum()) + 4 * U                                         # relative
            pr = 0.0
        lp = np.where(p > 0, np.log(np.where(p > 0, p, 1.0)), 0.0)
        loss = (p * (lp - np.where(p > 0, lq[i], 0.0))).sum()
        mass = np.zeros(V)
        np.add.at(mass, i, p)
        masserr = np.zeros(V)
        np.add.at(masserr, i, p * dp)
        es = _sum_err(y, q)
        dlq = U * 4 * np.abs(np.where(np.isfinite(y), y, 0.0)) + es + 3 * U * abs(ls)
        g = dloss[r] * c
        if not tail:
            d = g * (q - mass)
            err = abs(g) * (q * (dlq + 8 * U) + masserr + FLUSH) + 4 * U * np.abs(d)
            el = (p * dlq[i]).sum() + (p * dp * (np.abs(lp - np.where(p > 0, lq[i], 0.0)) + 1)).sum()
        else:
            W = 1.0 if pr > 0 else p.sum()
            if pr > 0:
                with np.errstate(divide="ignore"):
                    loss = loss + pr * (np.log(pr) - np.log(qr))
            rest = np.where(named, 0.0, q) / (qr if qr > 0 else 1.0)
            yr = np.where(named, 0.0, y - (y[~named].max() if qr > 0 else 0.0))
            esr = _sum_err(yr, rest)                                                           # of the rest's sum
            coef = W * qr - pr
            d = g * np.where(named, W * q - mass, rest * coef)
            ey = 4 * U * np.abs(np.where(np.isfinite(y), y, 0.0))
            share = qr * (1 - qr) * (esr + ey[i].max() + 4 * U * abs(ls))                      # of q_r
            err = abs(g) * np.where(named, q * (ey + esr + 8 * U), rest * (abs(coef) * (4 * U * np.abs(yr) + esr + 12 * U) + share) + FLUSH * abs(coef)) + 4 * U * np.abs(d)
            el = abs(coef) * esr + (np.abs(W * q[i] - mass[i]) * ey[i]).sum() + 1e-12
        out["loss"][r], tol["loss"][r] = loss, (1.05 * el + 3 * U * abs(loss) if np.isfinite(loss) else 0.0)
        out["dlogits"][r], tol["dlogits"][r] = d, 1.05 * err + half[0] * 1.01 * np.abs(d) + half[1]
    return out, tol
