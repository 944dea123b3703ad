"""Autograd boundary of the gated linear recurrence (csrc/gf_recur.hip): a recurrent layer that is linear in its state, parallel in time.

    z, zT = linear_recurrence(u, q_check, q_hat, z0, lengths)         z_t = q_check_t z_{t-1} + q_hat_t u_t

This is GatedGRNN's recursion (alegnn/utils/graphML.py:1421-1462) with an identity B(S) and sigma, so all T steps are one launch instead of
one filter per step; the gates are GatedGRNN's q_hat / q_check (time, node) and, beyond the reference, per feature or per element.
"""
from __future__ import annotations

import contextlib
import functools

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .functional import _ptr

_DTYPES = {torch.float32: _lib.GF_F32, torch.bfloat16: _lib.GF_BF16, torch.float16: _lib.GF_F16}
_FLOATS = tuple(_DTYPES)
_F32 = (torch.float32,)
_I32 = (torch.int32,)
_HERE = contextlib.nullcontext()

# The calls below are a few microseconds of GPU work at the reference's own sizes, so the host side counts: device and stream are asked for
# without building torch's Python objects, scratch and statistics share one allocation, and double backward is refused only when asked for.


def _on(dev):
    """The tensors' device as the current one (nothing to do in the usual case)."""
    return _HERE if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev.index)


def _require_cuda(who, name, t, dtypes):
    if t.device.type != "cuda":
        raise RuntimeError(f"alegnn_amd.{who}: `{name}` is on '{t.device}'. This implementation runs on MI355X (HIP) only and has no "
                           "CPU fallback; move the data to 'cuda'.")
    if t.dtype not in dtypes:
        raise TypeError(f"alegnn_amd.{who}: `{name}` has dtype {t.dtype}; supported: {', '.join(str(d) for d in dtypes)}")


def _dense(t):
    """Contiguous and aligned to 16 bytes (the kernels' vector loads): a view that starts at an odd element is copied."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _gate_kind(q, shape, name):
    """Which axes a gate of an input [B, T, H, N] has (GF_GATE_*)."""
    have = tuple(q.shape)
    B, T, H, N = shape
    if not (len(have) == 4 and have[1] == T and have[0] in (1, B) and have[2] in (1, H) and have[3] in (1, N)):
        raise AssertionError(f"{name}: shape {have} for an input {tuple(shape)} (want [B|1, T, H|1, N|1])")
    return (_lib.GF_GATE_B if have[0] == B else 0) | (_lib.GF_GATE_H if have[2] == H else 0) | (_lib.GF_GATE_N if have[3] == N else 0)


@functools.lru_cache(maxsize=256)
def _sizes(B, T, H, N, kc, hat, kh):
    """(checkpoint floats, forward workspace bytes, backward workspace bytes) of a shape."""
    L = _lib.lib()
    return (L.gf_recurrence_checkpoint_floats(B, T, H, N, kc, hat, kh), L.gf_recurrence_workspace_bytes(B, T, H, N, kc, hat, kh, 0),
            L.gf_recurrence_workspace_bytes(B, T, H, N, kc, hat, kh, 1))


def _forward(u, qc, qh, z0, lengths, kinds, keep):
    L = _lib.lib()
    B, T, H, N = u.shape
    dev = u.device
    kc, kh, hat = kinds
    with _on(dev):
        z = torch.empty((B, T, H, N), dtype=u.dtype, device=dev)
        zT = torch.empty((B, H, N), dtype=torch.float32, device=dev)
        if B * H * N == 0:
            return z, zT, None
        nck, nb, _ = _sizes(B, T, H, N, kc, hat, kh)
        ckpt = torch.empty(nck, dtype=torch.float32, device=dev) if keep else None
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        _lib.check(L.gf_recurrence_forward(u.data_ptr(), qc.data_ptr(), kc, _ptr(qh), kh, _ptr(z0), _ptr(lengths), z.data_ptr(), zT.data_ptr(),
                                           _ptr(ckpt), _ptr(ws), nb, _DTYPES[u.dtype], B, T, H, N, _stream(dev)), "gf_recurrence_forward")
    return z, zT, ckpt


def _once(f, ctx, *grads):
    """f(ctx, *grads); under create_graph the result refuses to be differentiated again."""
    return once_differentiable(f)(ctx, *grads) if torch.is_grad_enabled() else f(ctx, *grads)


def _recurrence_backward(ctx, dz, dzT):
    L = _lib.lib()
    u, qc, qh, lengths, ckpt = ctx.saved_tensors
    kc, kh, hat = ctx.kinds
    B, T, H, N = u.shape
    dev = u.device
    need_u, need_c, need_h, need_0 = ctx.needs_input_grad[:4]
    if dz is None and dzT is None:
        return None, None, None, None, None, None
    dz, dzT = _dense(dz), _dense(dzT)
    with _on(dev):
        du = torch.empty_like(u) if need_u else None
        dqc = torch.empty_like(qc) if need_c else None
        dqh = torch.empty_like(qh) if need_h else None
        dz0 = torch.empty((B, H, N), dtype=torch.float32, device=dev) if need_0 else None
        if B * H * N == 0:
            return du, None if dqc is None else dqc.zero_(), None if dqh is None else dqh.zero_(), dz0, None, None
        nb = _sizes(B, T, H, N, kc, hat, kh)[2]
        ws = torch.empty(nb, dtype=torch.uint8, device=dev) if nb else None
        _lib.check(L.gf_recurrence_backward(u.data_ptr(), qc.data_ptr(), kc, _ptr(qh), kh, _ptr(lengths), _ptr(ckpt), _ptr(dz), _ptr(dzT),
                                            _ptr(du), _ptr(dqc), _ptr(dqh), _ptr(dz0), _ptr(ws), nb, _DTYPES[u.dtype], B, T, H, N,
                                            _stream(dev)), "gf_recurrence_backward")
    return du, dqc, dqh, dz0, None, None


class _LinearRecurrenceFunction(torch.autograd.Function):
    """gf_recurrence_forward / gf_recurrence_backward (include/gfhip.h)."""

    @staticmethod
    def forward(ctx, u, qc, qh, z0, lengths, kinds):
        u, qc, qh, z0 = _dense(u), _dense(qc), _dense(qh), _dense(z0)
        z, zT, ckpt = _forward(u, qc, qh, z0, lengths, kinds, ctx.needs_input_grad[1])
        ctx.kinds = kinds
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(u, qc, qh, lengths, ckpt)
        return z, zT

    @staticmethod
    def backward(ctx, dz, dzT):
        return _once(_recurrence_backward, ctx, dz, dzT)


def linear_recurrence(u, q_check, q_hat=None, z0=None, lengths=None):
    """z_t = q_check_t * z_{t-1} + q_hat_t * u_t for t = 1..T, starting from z0.

    u [B,T,H,N] in float32, bfloat16 or float16; q_check and q_hat (None = 1) [B|1, T, H|1, N|1] in u's dtype: one gate per time step
    ([B,T,1,1]), node ([B,T,1,N]), feature ([B,T,H,1]) or element; z0 [B,H,N] float32 (None = 0); lengths [B] int32 on u's device: how many
    steps of each sequence count (None = all; values are clamped to [0, T]).  Padded steps are not read, give z = 0 and no gradient.
    Returns z [B,T,H,N] in u's dtype and the last state zT [B,H,N] in float32 -- what the next call takes as z0, so a sequence can be fed in
    pieces down to single steps (T = 1) without losing the state's precision.  The state is float32 throughout; products of q_check
    over a few hundred steps must stay finite (gates in [-1, 1] always do).  Differentiable (once) in u, q_check, q_hat and z0."""
    who = "linear_recurrence"
    assert u.dim() == 4, f"{who}: u has shape {tuple(u.shape)}, want [B, T, H, N]"
    _require_cuda(who, "u", u, _FLOATS)
    assert max(u.shape) <= 2 ** 31 - 2 ** 17, f"{who}: u has shape {tuple(u.shape)}: a side over 2^31 - 2^17"
    kinds = [0, 0, 0 if q_hat is None else 1]
    for i, name, q in ((0, "q_check", q_check), (1, "q_hat", q_hat)):
        if q is not None:
            kinds[i] = _gate_kind(q, u.shape, name)
            _require_cuda(who, name, q, (u.dtype,))
            assert q.device == u.device, f"{who}: {name} is on {q.device}, u on {u.device}"
    kinds = tuple(kinds)
    if z0 is not None:
        assert tuple(z0.shape) == (u.shape[0], u.shape[2], u.shape[3]), f"{who}: z0 has shape {tuple(z0.shape)} for u {tuple(u.shape)}"
        _require_cuda(who, "z0", z0, _F32)
        assert z0.device == u.device, f"{who}: z0 is on {z0.device}, u on {u.device}"
    if lengths is not None:
        assert tuple(lengths.shape) == (u.shape[0],), f"{who}: lengths has shape {tuple(lengths.shape)}, want [{u.shape[0]}]"
        _require_cuda(who, "lengths", lengths, _I32)
        assert lengths.device == u.device, f"{who}: lengths is on {lengths.device}, u on {u.device}"
        lengths = lengths.contiguous()
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (u, q_check, q_hat, z0)):
        return _LinearRecurrenceFunction.apply(u, q_check, q_hat, z0, lengths, kinds)
    return _forward(_dense(u), _dense(q_check), _dense(q_hat), _dense(z0), lengths, kinds, False)[:2]
