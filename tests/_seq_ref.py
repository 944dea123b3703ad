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
