"""The gated linear recurrence (csrc/gf_recur.hip, autograd node in csrc/gf_torch.cpp): a recurrent layer that is linear in its state, parallel in time.

    z, zT = linear_recurrence(u, q_check, q_hat, z0, lengths)         z_t = q_check_t z_{t-1} + q_hat_t u_t

This is GatedGRNN's recursion (alegnn/utils/graphML.py:1421-1462) with an identity B(S) and sigma, so all T steps are one launch instead of
one filter per step; the gates are GatedGRNN's q_hat / q_check (time, node) and, beyond the reference, per feature or per element.
"""
from __future__ import annotations

import torch
import torch.autograd.forward_ad as fwAD

from . import _lib

_FLOATS = (torch.float32, torch.bfloat16, torch.float16)
_F32 = (torch.float32,)
_I32 = (torch.int32,)


def _require_cuda(who, name, t, dtypes):
    if t.device.type != "cuda":
        raise RuntimeError(f"alegnn_amd.{who}: `{name}` is on '{t.device}'. This implementation runs on MI355X (HIP) only and has no "
                           "CPU fallback; move the data to 'cuda'.")
    if t.dtype not in dtypes:
        raise TypeError(f"alegnn_amd.{who}: `{name}` has dtype {t.dtype}; supported: {', '.join(str(d) for d in dtypes)}")


def _no_tangent(who, **inputs):
    """Forward-mode derivatives are not there: a tangent is refused, not dropped."""
    for name, t in inputs.items():
        if t is not None and t.is_floating_point() and fwAD.unpack_dual(t).tangent is not None:
            raise NotImplementedError(f"alegnn_amd.{who}: `{name}` carries a tangent; forward-mode derivatives are not supported")


def _same_device(who, name, t, x):
    if t.device != x.device:
        raise RuntimeError(f"alegnn_amd.{who}: `{name}` is on '{t.device}', the other tensors on '{x.device}'")


def _check_gate(who, q, shape, name):
    have = tuple(q.shape)
    B, T, H, N = shape
    if not (len(have) == 4 and have[1] == T and have[0] in (1, B) and have[2] in (1, H) and have[3] in (1, N)):
        raise AssertionError(f"{who}: {name} has shape {have} for an input {tuple(shape)} (want [B|1, T, H|1, N|1])")


def _explain(u, q_check, q_hat, z0, lengths):
    """Why the arguments were refused."""
    who = "linear_recurrence"
    _no_tangent(who, u=u, q_check=q_check, q_hat=q_hat, z0=z0)
    assert u.dim() == 4, f"{who}: u has shape {tuple(u.shape)}, want [B, T, H, N]"
    _require_cuda(who, "u", u, _FLOATS)
    assert max(u.shape) <= 2 ** 31 - 2 ** 17, f"{who}: u has shape {tuple(u.shape)}: a side over 2^31 - 2^17"
    for name, q in (("q_check", q_check), ("q_hat", q_hat)):
        if q is not None:
            _check_gate(who, q, u.shape, name)
            _require_cuda(who, name, q, (u.dtype,))
            _same_device(who, name, q, u)
    if z0 is not None:
        assert tuple(z0.shape) == (u.shape[0], u.shape[2], u.shape[3]), f"{who}: z0 has shape {tuple(z0.shape)} for u {tuple(u.shape)}"
        _require_cuda(who, "z0", z0, _F32)
        _same_device(who, "z0", z0, u)
    if lengths is not None:
        assert tuple(lengths.shape) == (u.shape[0],), f"{who}: lengths has shape {tuple(lengths.shape)}, want [{u.shape[0]}]"
        _require_cuda(who, "lengths", lengths, _I32)
        _same_device(who, "lengths", lengths, u)
    raise RuntimeError(f"{who}: refused")


def linear_recurrence(u, q_check, q_hat=None, z0=None, lengths=None):
    """z_t = q_check_t * z_{t-1} + q_hat_t * u_t for t = 1..T, starting from z0.

    u [B,T,H,N] in float32, bfloat16 or float16; q_check and q_hat (None = 1) [B|1, T, H|1, N|1] in u's dtype: one gate per time step
    ([B,T,1,1]), node ([B,T,1,N]), feature ([B,T,H,1]) or element; z0 [B,H,N] float32 (None = 0); lengths [B] int32 on u's device: how many
    steps of each sequence count (None = all; values are clamped to [0, T]).  What padded steps hold does not matter: they give z = 0 and no
    gradient.  Returns z [B,T,H,N] in u's dtype and the last state zT [B,H,N] in float32 -- what the next call takes as z0, so a sequence can
    be fed in pieces down to single steps (T = 1) without losing the state's precision.  The state is float32 throughout; the product of
    q_check over any 64 consecutive steps must be finite (gates below 4 in magnitude always are), over longer stretches only the states have
    to stay in range.  Differentiable (once, in reverse mode) in u, q_check, q_hat and z0."""
    host = _lib.host()
    try:
        return host.linear_recurrence(u, q_check, q_hat, z0, lengths)
    except host.Refused:
        pass
    _explain(u, q_check, q_hat, z0, lengths)
