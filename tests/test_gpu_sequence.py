"""linear_recurrence on the GPU against a step-by-step float64 restatement (tests/_seq_ref.py), bounds derived there."""
import numpy as np
import pytest
import torch

import _seq_ref as ref
import alegnn_amd
from alegnn_amd import linear_recurrence

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def gate_shape(kind, B, T, H, N):
    return {"full": (B, T, H, N), "node": (B, T, 1, N), "feature": (B, T, H, 1), "time": (B, T, 1, 1), "node1": (1, T, 1, N),
            "time1": (1, T, 1, 1), "full1": (1, T, H, N)}[kind]


def make(B, T, H, N, kc, kh, dtype, seed=0, signed=True):
    g = torch.Generator().manual_seed(seed)
    u = torch.randn((B, T, H, N), generator=g).to(dtype)
    qc = torch.rand(gate_shape(kc, B, T, H, N), generator=g)
    qc = (qc * 1.98 - 0.99 if signed else qc * 0.3 + 0.7).to(dtype)
    qh = None if kh is None else torch.randn(gate_shape(kh, B, T, H, N), generator=g).to(dtype)
    z0 = torch.randn((B, H, N), generator=g)
    dz = torch.randn((B, T, H, N), generator=g).to(dtype)
    dzT = torch.randn((B, H, N), generator=g)
    return u, qc, qh, z0, dz, dzT


def run(u, qc, qh, z0, lengths, dz, dzT, dev="cuda"):
    ins = [None if t is None else t.to(dev).requires_grad_() for t in (u, qc, qh, z0)]
    z, zT = linear_recurrence(*ins, lengths=None if lengths is None else lengths.to(dev))
    leaves = [t for t in ins if t is not None]
    grads = torch.autograd.grad([z, zT], leaves, [dz.to(dev), dzT.to(dev)])
    names = [k for k, t in zip(("du", "dq_check", "dq_hat", "dz0"), ins) if t is not None]
    out = dict(zip(names, grads), z=z.detach(), zT=zT.detach())
    for k, t in (("z", u), ("du", u), ("dq_check", qc), ("dq_hat", qh)):
        if t is not None:
            assert out[k].dtype == t.dtype and out[k].shape == t.shape
    assert out["zT"].dtype == torch.float32
    return {k: v.double().cpu().numpy() for k, v in out.items()}


def f64(t):
    return None if t is None else t.double().numpy()


def check(out, ins, lengths, dtype):
    u, qc, qh, z0, dz, dzT = (f64(t) for t in ins)
    n = None if lengths is None else lengths.numpy()
    want, tol = ref.recurrence(u, qc, qh, z0, n, dz, dzT), ref.recurrence_bounds(u, qc, qh, z0, n, dz, dzT, dtype)
    for k, v in out.items():
        if want[k].size == 0:
            continue
        bad = ~(np.abs(v - want[k]) <= tol[k])
        assert not bad.any(), (k, int(bad.sum()), float(np.abs(v - want[k])[bad].max()), np.argwhere(bad)[0].tolist())


SHAPES = [(1, 1, 1, 1), (2, 7, 3, 5), (3, 8, 2, 4), (2, 9, 4, 8), (1, 65, 5, 4), (3, 300, 3, 12), (1, 1030, 1, 3), (2, 520, 2, 64), (1, 5000, 2, 4),
          (2, 130, 7, 52), (4, 33, 32, 50)]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("kc,kh", [("full", "full"), ("full", None), ("time", None), ("node", "node"), ("feature", "time"), ("node", "full"),
                                   ("full1", "node1"), ("time1", "feature")])
def test_values_and_gradients(shape, kc, kh):
    ins = make(*shape, kc, kh, torch.float32, seed=sum(shape))
    check(run(*ins[:4], None, *ins[4:]), ins, None, torch.float32)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1), (2, 9, 3, 5), (2, 130, 4, 8), (1, 3000, 1, 4), (3, 70, 2, 51)], ids=str)
@pytest.mark.parametrize("kc,kh", [("full", "full"), ("time", None), ("node", "feature"), ("full", "time1")])
def test_half_types(shape, kc, kh, dtype):
    ins = make(*shape, kc, kh, DT[dtype], seed=sum(shape) + 1)
    check(run(*ins[:4], None, *ins[4:]), ins, None, DT[dtype])


@pytest.mark.parametrize("shape", [(5, 1, 2, 3), (7, 40, 3, 4), (6, 300, 1, 8), (4, 4000, 1, 4)], ids=str)
@pytest.mark.parametrize("kc,kh", [("full", "full"), ("time", "node"), ("time1", None)])
def test_lengths_with_nan_in_the_padding(shape, kc, kh):
    B, T, H, N = shape
    ins = list(make(*shape, kc, kh, torch.float32, seed=3))
    lengths = torch.tensor([0, 1, T, T // 2, max(T - 1, 0), -3, T + 5][:B], dtype=torch.int32)
    dead = torch.arange(T)[None, :] >= lengths.clamp(0, T)[:, None]
    clean = list(ins)
    for i, k in ((0, "full"), (4, "full"), (1, kc), (2, kh)):
        if ins[i] is not None and k == "full":                  # what is padding must not be read, whatever it holds
            ins[i] = ins[i].masked_fill(dead[:, :, None, None], float("nan"))
    out = run(*ins[:4], lengths, *ins[4:])
    check(out, clean, lengths, torch.float32)
    d = dead.numpy()
    assert (out["z"][d] == 0).all() and (out["du"][d] == 0).all()
    if kc == "full":
        assert (out["dq_check"][d] == 0).all() and (out["dq_hat"][d] == 0).all()


@pytest.mark.parametrize("kc,kh", [("full", "full"), ("time", None)])
def test_sequences_that_end_inside_a_split_of_the_time_axis(kc, kh):
    """One workgroup per (sequence, split): the backward walk skips 0 to 3 slabs of 64 steps behind the end before it joins the first one."""
    B, T, H, N = 12, 2048, 2, 4
    ins = make(B, T, H, N, kc, kh, torch.float32, seed=8)
    lengths = torch.tensor([257 + 53 * k for k in range(B)], dtype=torch.int32)
    out = run(*ins[:4], lengths, *ins[4:])
    check(out, ins, lengths, torch.float32)
    for _ in range(3):
        again = run(*ins[:4], lengths, *ins[4:])
        assert all(np.array_equal(out[k], again[k]) for k in out)


def test_no_steps_no_sequences_and_no_channels():
    z0 = torch.randn(2, 3, 4, device="cuda")
    for shape in ((2, 0, 3, 4), (0, 5, 3, 4), (2, 5, 0, 4), (2, 5, 3, 0)):
        u = torch.zeros(shape, device="cuda", requires_grad=True)
        q = torch.zeros(shape, device="cuda", requires_grad=True)
        s = (z0 if shape[1] == 0 else torch.zeros(shape[0], shape[2], shape[3], device="cuda")).clone().requires_grad_()
        z, zT = linear_recurrence(u, q, None, s)
        assert z.shape == shape and torch.equal(zT, s)
        w = torch.randn_like(zT)
        gu, gq, gs = torch.autograd.grad([z, zT], [u, q, s], [torch.zeros_like(z), w])
        assert gu.shape == shape and gq.shape == shape and torch.equal(gs, w)


def test_pieces_and_single_steps_continue_a_sequence():
    """Feeding a sequence in pieces through zT -> z0 gives the whole run's values: each piece within the whole run's bound."""
    B, T, H, N = 3, 37, 4, 25
    ins = make(B, T, H, N, "full", "full", torch.bfloat16, seed=5)
    u, qc, qh, z0 = (t.cuda() for t in ins[:4])
    want = ref.recurrence(*(f64(t) for t in ins[:4]), None, None, None)
    tol = ref.recurrence_bounds(*(f64(t) for t in ins[:4]), None, None, None, torch.bfloat16)
    with torch.no_grad():
        s, t = z0, 0
        for n in (1, 1, 5, 8, 1, 16, 0, 5):
            z, s = linear_recurrence(u[:, t:t + n], qc[:, t:t + n], qh[:, t:t + n], s)
            assert (np.abs(z.double().cpu().numpy() - want["z"][:, t:t + n]) <= tol["z"][:, t:t + n]).all()
            t += n
    assert t == T and (np.abs(s.double().cpu().numpy() - want["zT"]) <= tol["zT"]).all()


def test_strided_and_misaligned_inputs():
    B, T, H, N = 2, 50, 4, 12
    ins = make(B, T, H, N, "full", "node", torch.float32, seed=7)
    want = run(*ins[:4], None, *ins[4:])

    def odd(t):                                                  # the same values, one element behind an aligned address, and strided
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
        flat[1:] = t.flatten().cuda()
        return flat[1:].view(t.shape)
    a = [odd(t) for t in ins]
    b = [t.cuda().transpose(1, -1).contiguous().transpose(1, -1) if t.dim() == 4 else t.cuda() for t in ins]
    for v in (a, b):
        leaves = [t.detach().requires_grad_() for t in v[:4]]
        z, zT = linear_recurrence(*leaves)
        g = torch.autograd.grad([z, zT], leaves, [v[4], v[5]])
        got = dict(z=z, zT=zT, du=g[0], dq_check=g[1], dq_hat=g[2], dz0=g[3])
        for k, t in got.items():
            assert np.array_equal(t.detach().double().cpu().numpy(), want[k]), k


def test_only_some_gradients_and_no_state():
    B, T, H, N = 2, 90, 3, 8
    u, qc, qh, z0, dz, dzT = (t.cuda() for t in make(B, T, H, N, "time", "full", torch.float32, seed=8))
    full = [t.clone().requires_grad_() for t in (u, qc, qh, z0)]
    z, zT = linear_recurrence(*full)
    want = torch.autograd.grad([z, zT], full, [dz, dzT])
    for i in range(4):
        v = [t.clone().requires_grad_(i == j) for j, t in enumerate((u, qc, qh, z0))]
        z, zT = linear_recurrence(*v)
        assert torch.equal(torch.autograd.grad([z, zT], [v[i]], [dz, dzT])[0], want[i])
    x = u.clone().requires_grad_()                               # only one of the two outputs used
    z, _ = linear_recurrence(x, qc, qh)
    a = torch.autograd.grad(z, x, dz)[0]
    z, zT = linear_recurrence(x, qc, qh, torch.zeros_like(z0))
    assert torch.equal(a, torch.autograd.grad([z, zT], x, [dz, torch.zeros_like(zT)])[0])
    _, zT = linear_recurrence(x, qc, qh)
    b = torch.autograd.grad(zT, x, dzT)[0]
    z, zT = linear_recurrence(x, qc, qh)
    assert torch.equal(b, torch.autograd.grad([z, zT], x, [torch.zeros_like(z), dzT])[0])


def test_gradients_against_differences():
    B, T, H, N = 2, 19, 2, 4
    ins = make(B, T, H, N, "node", "feature", torch.float32, seed=9)
    out = run(*ins[:4], None, *ins[4:])
    u, qc, qh, z0, dz, dzT = (f64(t) for t in ins)

    def value(**kw):
        a = dict(u=u, qc=qc, qh=qh, z0=z0)
        a.update(kw)
        r = ref.recurrence(a["u"], a["qc"], a["qh"], a["z0"], None, None, None)
        return (r["z"] * dz).sum() + (r["zT"] * dzT).sum()
    rng = np.random.RandomState(0)
    for name, v, k in (("u", u, "du"), ("qc", qc, "dq_check"), ("qh", qh, "dq_hat"), ("z0", z0, "dz0")):
        d, e = rng.randn(*v.shape), 1e-4
        slope = (value(**{name: v + e * d}) - value(**{name: v - e * d})) / (2 * e)
        # central differences of a polynomial are off by O(e^2) of its third derivative: 1e-5 of the slope's own terms is far above both errors
        assert abs(slope - (out[k] * d).sum()) <= 1e-5 * np.abs(out[k] * d).sum()


def test_runs_agree_bitwise_and_on_another_stream():
    ins = make(2, 3000, 2, 20, "time", "node", torch.bfloat16, seed=10)
    first = run(*ins[:4], None, *ins[4:])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        second = run(*ins[:4], None, *ins[4:])
    torch.cuda.current_stream().wait_stream(side)
    for k in first:
        assert np.array_equal(first[k], second[k]), k


def test_captured_steps_replay():
    """Two captured graphs (a training pass and a single step) replayed in turn between eager calls give the eager results every time."""
    dev = "cuda"
    u, qc, qh, z0, dz, dzT = (t.to(dev) for t in make(2, 2500, 2, 20, "time", "full", torch.float32, seed=11))

    def passes(a):
        v = [t.detach().requires_grad_() for t in a[:4]]
        z, zT = linear_recurrence(*v)
        return [z.detach(), zT.detach(), *torch.autograd.grad([z, zT], v, [a[4], a[5]])]

    def step(a):
        with torch.no_grad():
            return list(linear_recurrence(a[0][:, :1], a[1][:, :1], a[2][:, :1], a[3]))
    static = [t.clone() for t in (u, qc, qh, z0, dz, dzT)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes(static), step(static)
    torch.cuda.current_stream().wait_stream(side)
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = passes(static)
    with torch.cuda.graph(g2):
        o2 = step(static)
    for i in range(4):
        fresh = [t * (0.9 ** i) for t in (u, qc, qh, z0, dz, dzT)]
        for s, f in zip(static, fresh):
            s.copy_(f)
        g1.replay()
        w2 = step(fresh)
        g2.replay()
        w1 = passes(fresh)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(o1, w1)) and all(torch.equal(a, b) for a, b in zip(o2, w2)), i


def test_more_than_two_to_the_31_elements():
    B, T, H, N = 1, 70001, 4, 7700                               # 2.16e9 elements: offsets pass 32 bits
    g = torch.Generator(device="cuda").manual_seed(1)
    u = torch.empty((B, T, H, N), dtype=torch.bfloat16, device="cuda").normal_(generator=g)
    qc = torch.rand((B, T, 1, 1), generator=g, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        z, zT = linear_recurrence(u, qc)
    pick = torch.tensor([0, 1, 7699], device="cuda")
    small = u[:, :, 3:4][..., pick].cpu()
    want = ref.recurrence(f64(small), f64(qc.cpu()), None, None, None, None, None)
    tol = ref.recurrence_bounds(f64(small), f64(qc.cpu()), None, None, None, None, None, torch.bfloat16)
    assert (np.abs(f64(z[:, :, 3:4][..., pick].cpu()) - want["z"]) <= tol["z"]).all()
    assert (np.abs(f64(zT[:, 3:4][..., pick].cpu()) - want["zT"]) <= tol["zT"]).all()


def test_many_sequences():
    ins = make(70000, 3, 1, 1, "time", None, torch.float32, seed=12)
    check(run(*ins[:4], None, *ins[4:]), ins, None, torch.float32)


def grown(B, T, H, N, kind, dtype, seed, forward):
    """Gates whose product over the whole sequence passes the largest float32, with a state (forward: z, else its adjoint) that stays in range: zero or
    tiny until the last steps of its walk."""
    g = torch.Generator().manual_seed(seed)
    q = torch.full(gate_shape(kind, B, T, H, N), 1.0)
    late = T // 3
    q[:, :300] = 1.2 + 0.01 * torch.rand(q[:, :300].shape, generator=g)
    q[:, T - late - 300:T - late] = 1.2 + 0.01 * torch.rand(q[:, T - late - 300:T - late].shape, generator=g)
    q = q.to(dtype)
    u, dz = torch.zeros((B, T, H, N)), torch.zeros((B, T, H, N))
    (u if forward else dz)[:, T - 100:] = torch.randn((B, 100, H, N), generator=g)
    z0 = torch.where(torch.rand((B, H, N), generator=g) < 0.5, 0.0, 1e-30)
    if forward:
        return u.to(dtype), q, None, z0, dz.to(dtype), torch.zeros((B, H, N))
    return u.to(dtype), q.flip(1), None, torch.zeros((B, H, N)), dz.flip(1).to(dtype), z0


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 20000, 2, 4), (3, 2048, 2, 3), (2, 1500, 1, 26)], ids=str)
@pytest.mark.parametrize("kind", ["full", "node", "feature", "time"])
@pytest.mark.parametrize("forward", [True, False])
def test_products_beyond_the_range_of_a_number(shape, kind, forward, dtype):
    """Splits of the time axis are composed without the product of all their gates having to be a float32: what the step by step walk gives in range
    is answered in range."""
    ins = grown(*shape, kind, DT[dtype], sum(shape), forward)
    check(run(*ins[:4], None, *ins[4:]), ins, None, DT[dtype])
    lengths = torch.tensor([shape[1] - 50, shape[1], 700][:shape[0]], dtype=torch.int32)
    check(run(*ins[:4], lengths, *ins[4:]), ins, lengths, DT[dtype])


def test_growth_over_the_whole_sequence():
    B, T, H, N = 1, 20000, 2, 4                                  # 1.01^20000 = 1e86
    g = torch.Generator().manual_seed(0)
    u, q, zero = torch.zeros((B, T, H, N)), torch.full((B, T, 1, 1), 1.01), torch.zeros((B, H, N))
    u[:, T - 100:] = torch.randn((B, 100, H, N), generator=g)
    dz = torch.zeros_like(u)
    dz[:, :100] = torch.randn((B, 100, H, N), generator=g)
    ins = (u, q, None, zero, dz, zero)
    out = run(*ins[:4], None, *ins[4:])
    check(out, ins, None, torch.float32)
    z, zT = linear_recurrence(u.cuda(), q.cuda())                # no initial state: the same walk from zeros
    assert np.array_equal(z.double().cpu().numpy(), out["z"]) and np.array_equal(zT.double().cpu().numpy(), out["zT"]) and (z[:, :T - 100] == 0).all()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(2, 31, 5, 52), (3, 29, 3, 51), (2, 30, 2, 130)], ids=str)
@pytest.mark.parametrize("kc,kh", [("full", "full"), ("node", "full"), ("feature", "node"), ("time", None), ("time1", "time")])
@pytest.mark.parametrize("padded", [False, True])
def test_waves_side_by_side_over_more_than_one_slab(shape, kc, kh, padded, dtype):
    """17 to 32 steps: a workgroup's waves stand side by side along the channels and walk two slabs of 16 steps (the form of many channels)."""
    ins = make(*shape, kc, kh, DT[dtype], seed=sum(shape) + 2)
    lengths = torch.tensor([shape[1] - 2, 9, 16][:shape[0]], dtype=torch.int32) if padded else None
    check(run(*ins[:4], lengths, *ins[4:]), ins, lengths, DT[dtype])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("kc,kh", [("full", "full"), ("node", "time"), ("feature", None)])
def test_many_channels_and_unlike_lengths(kc, kh, dtype):
    B, T, H, N = 16, 70, 8, 600                                  # 19200 threads' channels: five slabs, several chunks of channels
    ins = make(B, T, H, N, kc, kh, DT[dtype], seed=21)
    lengths = torch.tensor([0, 1, 15, 16, 17, 31, 32, 33, 48, 50, 63, 64, 65, 69, 70, 70], dtype=torch.int32)
    check(run(*ins[:4], lengths, *ins[4:]), ins, lengths, DT[dtype])


@pytest.mark.parametrize("shape", [(3, 1, 29, 701), (2, 7, 31, 513), (2, 40, 17, 333), (1, 700, 3, 401), (40, 3, 2, 700)], ids=str)
@pytest.mark.parametrize("kind", ["time", "time1", "node", "node1", "feature", "full1"])
def test_gate_sums_are_rounded_once(shape, kind):
    """With q_check = 0 and q_hat = 1 the gates' gradients are sums of dz_t u_{t-1} and dz_t u_t: whole numbers here, each product below 2^16 and each
    wave's sum of at most 256 of them exact in float32.  What is left is the sum of the partial ones: rounded once, it is the exact sum's float32."""
    B, T, H, N = shape
    g = torch.Generator().manual_seed(sum(shape))
    u, dz = (torch.randint(0, 256, (B, T, H, N), generator=g).float() for _ in range(2))
    z0 = torch.randint(0, 256, (B, H, N), generator=g).float()
    gate = gate_shape(kind, B, T, H, N)
    out = run(u, torch.zeros(gate), torch.ones(gate), z0, None, dz, torch.zeros(B, H, N))
    prev = np.concatenate((f64(z0)[:, None], f64(u)[:, :-1]), 1)
    for k, p in (("dq_check", f64(dz) * prev), ("dq_hat", f64(dz) * f64(u))):
        assert np.array_equal(out[k], ref.fold(p, gate).astype(np.float32).astype(np.float64)), k
