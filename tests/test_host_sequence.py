"""Refusals of the sequence and output operators, on the CPU: the C ABI validates before any HIP call, the Python layer before it loads a kernel."""
import ctypes
import types

import numpy as np
import pytest
import torch

import _seq_ref as ref
import alegnn_amd
from alegnn_amd import _lib, distill_top, linear_recurrence, token_log_probs
from alegnn_amd.functional_seq import _check_gate
from alegnn_amd.modules.training import Trainer
from alegnn_amd.utils import graphML as gml

FULL = _lib.GF_GATE_B | _lib.GF_GATE_H | _lib.GF_GATE_N


def recurrence_args(**kw):
    """A valid argument list of gf_recurrence_forward (made-up aligned addresses: nothing is launched once an argument is refused)."""
    a = dict(u=64, qc=64, kc=FULL, qh=64, kh=FULL, z0=64, lengths=None, z=64, zT=64, ckpt=64, ws=64, nb=1 << 40, dtype=0, B=2, T=5, H=3, N=4)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=3), -2, b"dtype"), (dict(kc=8), -2, b"gate kinds"), (dict(kh=-1), -2, b"gate kinds"), (dict(B=0), -1, b"bad shape"),
    (dict(T=-1), -1, b"bad shape"), (dict(H=0), -1, b"bad shape"), (dict(N=-4), -1, b"bad shape"), (dict(H=1 << 15, N=1 << 15), -1, b"channels"),
    (dict(T=(1 << 31) - 1, H=1, N=1), -1, b"steps"),
    (dict(u=None), -2, b"NULL"), (dict(qc=None), -2, b"NULL"), (dict(z=None), -2, b"NULL"), (dict(zT=None), -2, b"NULL"), (dict(u=68), -2, b"aligned"),
    (dict(qh=72), -2, b"aligned"), (dict(z=4), -2, b"aligned"), (dict(B=1, T=70000, N=4, ws=None, nb=0), -2, b"workspace"),
    (dict(B=(1 << 31) - 1, H=1 << 10, N=1 << 10), -1, b"too many"),
])
def test_recurrence_forward_refuses(kw, code, word):
    L = _lib.lib()
    assert L.gf_recurrence_forward(*recurrence_args(**kw)) == code
    assert word in L.gf_last_error()


@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=-1), -2, b"dtype"), (dict(B=0), -1, b"bad shape"), (dict(u=None), -2, b"NULL"), (dict(ckpt=None), -2, b"checkpoints"),
    (dict(qh=None), -2, b"without q_hat"), (dict(dz=68), -2, b"aligned"), (dict(du=72), -2, b"aligned"), (dict(kc=_lib.GF_GATE_B, ws=None, nb=0), -2, b"workspace"),
    (dict(ws=72, kc=_lib.GF_GATE_B), -2, b"aligned"),
])
def test_recurrence_backward_refuses(kw, code, word):
    a = dict(u=64, qc=64, kc=FULL, qh=64, kh=FULL, lengths=None, ckpt=64, dz=64, dzT=64, du=64, dqc=64, dqh=64, dz0=64, ws=64, nb=1 << 40, dtype=0, B=2, T=5,
             H=3, N=4)
    a.update(kw)
    L = _lib.lib()
    assert L.gf_recurrence_backward(*a.values(), None) == code
    assert word in L.gf_last_error()


def test_recurrence_sizes():
    L = _lib.lib()
    for B, T, H, N in ((2, 5, 3, 4), (1, 100000, 1, 3), (32, 257, 32, 1682), (1, 1, 1, 1)):
        n = L.gf_recurrence_checkpoint_floats(B, T, H, N, FULL, 1, FULL)
        assert n % (B * H * N) == 0 and 1 <= n // (B * H * N) <= T          # whole states, at most one per step
        assert L.gf_recurrence_workspace_bytes(B, T, H, N, FULL, 1, FULL, 1) >= L.gf_recurrence_workspace_bytes(B, T, H, N, FULL, 1, FULL, 0)
        node = _lib.GF_GATE_B | _lib.GF_GATE_N                              # a gate shared by the features: its product is kept in fp32
        assert L.gf_recurrence_workspace_bytes(B, T, H, N, node, 0, 0, 1) >= 4 * B * T * H * N
    assert L.gf_recurrence_checkpoint_floats(0, 5, 3, 4, FULL, 0, 0) == 0 and L.gf_recurrence_checkpoint_floats(2, 0, 3, 4, FULL, 0, 0) == 0
    assert L.gf_recurrence_workspace_bytes(2, 5, -3, 4, FULL, 0, 0, 1) == 0


def token_args(**kw):
    a = dict(x=64, stride=10, tokens=64, temperature=1.0, ignore=-100, logp=64, entropy=64, tl=64, ti=64, top=3, stats=64, ws=64, nb=1 << 40, dtype=0, R=4,
             V=10)
    a.update(kw)
    return [*a.values(), None]


@pytest.mark.parametrize("kw,code,word", [
    (dict(dtype=7), -2, b"dtype"), (dict(R=0), -1, b"bad shape"), (dict(V=0), -1, b"bad shape"), (dict(stride=-1), -1, b"bad shape"),
    (dict(temperature=0.0), -2, b"temperature"), (dict(temperature=-1.0), -2, b"temperature"), (dict(temperature=float("inf")), -2, b"temperature"),
    (dict(temperature=float("nan")), -2, b"temperature"), (dict(top=-1), -1, b"top"), (dict(top=11), -1, b"top"), (dict(top=65, V=100), -1, b"top"),
    (dict(x=None), -2, b"NULL"), (dict(tokens=None), -2, b"NULL"), (dict(logp=None), -2, b"NULL"), (dict(tl=None), -2, b"NULL"), (dict(ti=None), -2, b"NULL"),
    (dict(ws=None), -2, b"workspace"), (dict(nb=8), -2, b"workspace"), (dict(ws=68), -2, b"workspace"),
    (dict(V=(1 << 31) - 1), -1, b"outputs"), (dict(temperature=1e-38), -2, b"temperature"),
])
def test_token_forward_refuses(kw, code, word):
    L = _lib.lib()
    assert L.gf_token_logp_forward(*token_args(**kw)) == code
    assert word in L.gf_last_error()


def test_token_backward_and_distill_refuse():
    L = _lib.lib()

    def backward(**kw):
        a = dict(x=64, stride=10, tokens=64, temperature=1.0, ignore=-100, stats=64, ti=64, top=3, dlogp=64, dent=64, dtop=64, dx=64, dtype=0, R=4, V=10)
        a.update(kw)
        return L.gf_token_logp_backward(*a.values(), None)
    for kw, code in ((dict(stats=None), -2), (dict(ti=None), -2), (dict(dx=None), -2), (dict(top=65, V=99), -1), (dict(R=0), -1), (dict(dtype=5), -2)):
        assert backward(**kw) == code, kw

    def forward(**kw):
        a = dict(x=64, stride=10, idx=64, val=64, temperature=1.0, tail=0, loss=64, stats=64, probs=64, ws=64, nb=1 << 40, dtype=0, R=4, V=10, K=3)
        a.update(kw)
        return L.gf_distill_top_forward(*a.values(), None)
    for kw, code in ((dict(K=0), -1), (dict(K=65), -1), (dict(idx=None), -2), (dict(val=None), -2), (dict(loss=None), -2), (dict(probs=None), -2), (dict(V=0), -1),
                     (dict(nb=0), -2), (dict(temperature=0.0), -2), (dict(dtype=9), -2)):
        assert forward(**kw) == code, kw

    def dback(**kw):
        a = dict(x=64, stride=10, idx=64, probs=64, stats=64, temperature=1.0, tail=0, dloss=64, dx=64, dtype=0, R=4, V=10, K=3)
        a.update(kw)
        return L.gf_distill_top_backward(*a.values(), None)
    for kw, code in ((dict(K=0), -1), (dict(K=65), -1), (dict(dloss=None), -2), (dict(dx=None), -2), (dict(R=-1), -1)):
        assert dback(**kw) == code, kw
    assert L.gf_token_logp_workspace_bytes(0, 10, 3, 0) == 0 and L.gf_token_logp_workspace_bytes(4, 10, 3, 9) == 0
    assert L.gf_distill_top_workspace_bytes(4, -1, 3, 0) == 0


def test_python_layer_refuses_what_is_not_on_the_gpu_and_wrong_shapes():
    u = torch.zeros(2, 3, 4, 5)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_recurrence(u, u)
    with pytest.raises(AssertionError, match="shape"):
        linear_recurrence(u[0], u)
    x, t = torch.zeros(3, 7), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        token_log_probs(x, t)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        distill_top(x, t[:, None], x[:, :1])
    with pytest.raises(AssertionError, match="dim"):
        token_log_probs(x, t, dim=2)
    for bad in ((2, 3, 4), (2, 2, 4, 5), (3, 3, 4, 5), (2, 3, 2, 5), (2, 3, 4, 2)):
        with pytest.raises(AssertionError, match="want"):
            _check_gate("linear_recurrence", torch.zeros(bad), u.shape, "q_check")
    for good in ((1, 3, 1, 5), (2, 3, 4, 1), (1, 3, 1, 1), (2, 3, 4, 5)):
        _check_gate("linear_recurrence", torch.zeros(good), u.shape, "q_check")


def test_trainer_refuses_a_teacher_of_another_shape():
    data = types.SimpleNamespace(nTrain=10)
    ok = (torch.zeros(10, 3, dtype=torch.int64), torch.zeros(10, 3))
    for t in ((ok[0][:9], ok[1][:9]), (ok[0], ok[1][:, :2]), (ok[0][:, 0], ok[1][:, 0])):
        with pytest.raises(ValueError, match="teacherTop"):
            Trainer(None, data, 1, 5, teacherTop=t)
    with pytest.raises(ValueError, match="distillWeight"):
        Trainer(None, data, 1, 5, teacherTop=ok, distillWeight=1.5)


def test_layer_has_its_parameters_and_checks():
    layer = gml.LinearHiddenState(3, 4, 2, E=1)
    assert {k: tuple(v.shape) for k, v in layer.state_dict().items()} == {
        "aWeights": (4, 1, 2, 3), "xBias": (4, 1), "inputGate.weight": (4, 1, 2, 3), "inputGate.bias": (4, 1), "forgetGate.weight": (4, 1, 2, 3),
        "forgetGate.bias": (4, 1)}
    assert tuple(gml.LinearHiddenState(3, 4, 2, gate='node', bias=False).forgetGate.weight.shape) == (1, 1, 2, 3)
    with pytest.raises(AssertionError):
        gml.LinearHiddenState(3, 4, 2, gate='edge')
    with pytest.raises(AssertionError):
        layer(torch.zeros(2, 5, 3, 6), None)                        # no GSO yet
    with pytest.raises(AssertionError):
        layer.addGSO(torch.zeros(2, 6, 6))


# ---- the restatement the GPU tests compare with, against torch in float64 ------------------------------------------------------------------
def test_restatement_of_the_recurrence_against_autograd():
    g = torch.Generator().manual_seed(0)
    B, T, H, N = 2, 6, 3, 4
    u, qh, z0 = torch.randn(B, T, H, N, generator=g).double(), torch.randn(B, T, 1, N, generator=g).double(), torch.randn(B, H, N, generator=g).double()
    qc, dz, dzT = torch.rand(1, T, H, 1, generator=g).double(), torch.randn(B, T, H, N, generator=g).double(), torch.randn(B, H, N, generator=g).double()
    leaves = [t.clone().requires_grad_() for t in (u, qc, qh, z0)]
    h, zs = leaves[3], []
    for t in range(T):
        h = leaves[1][:, t] * h + leaves[2][:, t] * leaves[0][:, t]
        zs.append(h)
    grads = torch.autograd.grad([torch.stack(zs, 1), h], leaves, [dz, dzT])
    r = ref.recurrence(*(t.numpy() for t in (u, qc, qh, z0)), None, dz.numpy(), dzT.numpy())
    assert np.allclose(r["z"], torch.stack(zs, 1).detach().numpy(), rtol=1e-13, atol=1e-13)
    for k, w in zip(("du", "dq_check", "dq_hat", "dz0"), grads):
        assert np.allclose(r[k], w.numpy(), rtol=1e-12, atol=1e-12), k


def test_restatement_of_tokens_and_distillation_against_autograd():
    g = torch.Generator().manual_seed(1)
    R, V, top = 4, 11, 3
    x = torch.randn(R, V, generator=g).double()
    x[1, 4:] = -torch.inf
    tok = torch.tensor([3, 2, -100, 0])
    up = [torch.randn(R, generator=g).double(), torch.randn(R, generator=g).double(), torch.randn(R, top, generator=g).double()]
    leaf = x.clone().requires_grad_()
    lp = torch.log_softmax(leaf / 1.5, 1)
    p = lp.exp()
    logp = torch.where(tok >= 0, lp.gather(1, tok.clamp(min=0)[:, None])[:, 0], 0.0)
    ent = -(p * lp.masked_fill(p == 0, 0.0)).sum(1)
    best = torch.topk(x, top, 1)
    (d,) = torch.autograd.grad([logp, ent, lp.gather(1, best.indices)], leaf, up)
    out, _ = ref.tokens(x.numpy(), tok.numpy(), top, 1.5, -100, *(t.numpy() for t in up), (0.0, 0.0))
    d[1, 4:] = 0.0                                                   # (torch gives NaN at -inf)
    for k, w in (("logp", logp), ("entropy", ent), ("dlogits", d)):
        assert np.allclose(out[k], w.detach().numpy(), rtol=1e-10, atol=1e-10), k
    assert np.array_equal(out["top_tokens"], best.indices.numpy())
    x = torch.randn(R, V, generator=g).double()
    idx = torch.tensor([[0, 5, 7], [1, 1, 2], [3, -1, 4], [-1, -1, -1]])
    val = torch.log_softmax(torch.randn(R, V, generator=g).double(), 1)[:, :3]
    for tail in (False, True):
        leaf = x.clone().requires_grad_()
        lq = torch.log_softmax(leaf / 2.0, 1)
        rows = []
        for r in range(3):
            ok = idx[r] >= 0
            i, v = idx[r][ok], val[r][ok]
            if tail:
                pk = v.exp()
                keep = torch.ones(V, dtype=torch.bool)
                keep[i] = False
                pr = 1 - pk.sum()
                rows.append((pk * (v - lq[r, i])).sum() + pr * (pr.log() - lq[r, keep].exp().sum().log()))
            else:
                pk = torch.softmax(v / 2.0, 0)
                rows.append((pk * (pk.log() - lq[r, i])).sum())
        (d,) = torch.autograd.grad(torch.stack(rows).sum(), leaf)
        out, _ = ref.distill(x.numpy(), idx.numpy(), val.numpy(), 2.0, tail, np.ones(R), (0.0, 0.0))
        assert np.allclose(out["loss"][:3], [float(v) for v in rows], rtol=1e-10) and out["loss"][3] == 0
        assert np.allclose(out["dlogits"], d.numpy(), rtol=1e-9, atol=1e-12)


def test_a_tangent_is_named_before_anything_else_is():
    import torch.autograd.forward_ad as fwAD
    u, x, t, v = torch.zeros(2, 3, 4, 5), torch.zeros(3, 7), torch.zeros(3, dtype=torch.int64), torch.zeros(3, 1)
    with fwAD.dual_level():
        def dual(a):
            return fwAD.make_dual(a, torch.ones_like(a))
        for name, call in (("u", lambda: linear_recurrence(dual(u), u)), ("q_check", lambda: linear_recurrence(u, dual(u))),
                           ("q_hat", lambda: linear_recurrence(u, u, dual(u))), ("z0", lambda: linear_recurrence(u, u, u, dual(u[:, 0]))),
                           ("logits", lambda: token_log_probs(dual(x), t)), ("logits", lambda: distill_top(dual(x), t[:, None], v)),
                           ("values", lambda: distill_top(x, t[:, None], dual(v)))):
            with pytest.raises(NotImplementedError, match=f"`{name}` carries a tangent"):
                call()
        with pytest.raises(RuntimeError, match="no CPU fallback"):
            linear_recurrence(u, u)
