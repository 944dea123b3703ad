"""token_log_probs and distill_top on the GPU against row-by-row float64 restatements (tests/_seq_ref.py), bounds derived there."""
import numpy as np
import pytest
import torch

import _seq_ref as ref
from alegnn_amd import distill_top, token_log_probs

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
NINF = float("-inf")


def half(dtype):
    return ref.HALF[dtype], ref.TINY[dtype]


def logits_of(R, V, dtype, seed, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((R, V), generator=g) * scale + torch.randn((V,), generator=g)).to(dtype), g


def within(got, want, tol, what):
    got = got.detach().double().cpu().numpy()
    with np.errstate(invalid="ignore"):
        ok = (np.abs(got - want) <= tol) | (got == want) | (np.isnan(got) & np.isnan(want))
    assert ok.all(), (what, int((~ok).sum()), np.argwhere(~ok)[0].tolist(), got[~ok][0], want[~ok][0])


def check_tokens(x, tok, top, T=1.0, ignore=-100, seed=0, grads=("logp", "entropy", "top"), view=lambda t: t):
    R, V = x.shape
    g = torch.Generator().manual_seed(seed + 100)
    up = dict(logp=torch.randn(R, generator=g), entropy=torch.randn(R, generator=g), top=torch.randn((R, top), generator=g) if top else None)
    up = {k: v if k in grads else None for k, v in up.items()}
    leaf = view(x.cuda()).detach().requires_grad_()
    logp, ent, tl, ti = token_log_probs(leaf, tok.cuda(), top=top, temperature=T, ignore_index=ignore)
    pairs = [(o, u) for o, u in ((logp, up["logp"]), (ent, up["entropy"]), (tl, up["top"])) if u is not None]
    d = torch.autograd.grad([o for o, _ in pairs], leaf, [u.cuda() for _, u in pairs])[0]
    want, tol = ref.tokens(x.double().numpy(), tok.numpy(), top, T, ignore, *(None if up[k] is None else up[k].double().numpy() for k in ("logp", "entropy", "top")),
                           half(x.dtype))
    if top:
        assert np.array_equal(ti.cpu().numpy(), want["top_tokens"])
        within(tl, want["top_logp"], tol["top_logp"], "top_logp")
    within(logp, want["logp"], tol["logp"], "logp")
    within(ent, want["entropy"], tol["entropy"], "entropy")
    assert d.dtype == x.dtype
    within(d, want["dlogits"], tol["dlogits"], "dlogits")
    with torch.no_grad():                                          # the same answers without a gradient
        l2, e2, t2, i2 = token_log_probs(x.cuda(), tok.cuda(), top=top, temperature=T, ignore_index=ignore)
    assert torch.equal(l2.nan_to_num(), logp.detach().nan_to_num()) and torch.equal(e2.nan_to_num(), ent.detach().nan_to_num())
    assert top == 0 or torch.equal(i2, ti)
    return d


SIZES = [(1, 1), (3, 2), (100, 5), (7, 63), (5, 64), (4, 65), (3, 257), (6, 1000), (2, 1682), (3, 2049), (2, 4099), (2, 10001), (1, 33333), (2, 100000),
         (1, 262147)]


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("top", [0, 1, 20, 64])
def test_tokens(size, dtype, top):
    R, V = size
    x, g = logits_of(R, V, DT[dtype], R + V)
    tok = torch.randint(0, V, (R,), generator=g)
    check_tokens(x, tok, min(top, V), T=(1.0, 2.0, 0.7)[V % 3], seed=V)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("V", [6, 300, 5000, 20011])
def test_tokens_masked_ignored_and_tied(V, dtype):
    R, top = 12, min(V, 30)
    x, g = logits_of(R, V, DT[dtype], V)
    tok = torch.randint(0, V, (R,), generator=g)
    lowest = torch.finfo(DT[dtype]).min
    x[0] = NINF                                                     # nothing left
    x[1, 1:] = NINF                                                 # one output left
    x[2] = 0.25                                                     # all equal
    x[3] = lowest                                                   # masks of the type's lowest value, everywhere
    x[4, ::2] = lowest
    x[5] = torch.linspace(-3, 3, V).to(DT[dtype])                   # sorted, with long runs of equal values in bf16
    x[6] = torch.linspace(3, -3, V).to(DT[dtype])
    x[7] = torch.where(torch.arange(V) % 2 == 0, 0.0, -0.0).to(DT[dtype])    # zeros of both signs are equal
    x[8, torch.randperm(V, generator=g)[: V // 2 + 1]] = NINF
    tok[8] = int(x[8].float().argmax())
    tok[9] = tok[10] = -100
    tok[1] = 0
    check_tokens(x, tok, top, seed=V)
    check_tokens(x, tok, 0, seed=V, grads=("entropy",))
    check_tokens(x, tok, top, seed=V, grads=("top",))


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("V", [1100, 8192, 8201, 50001])
@pytest.mark.parametrize("top", [1, 8, 64])
def test_tokens_rows_of_equal_values(V, top, dtype):
    """More values at or above a tile's threshold than are ranked at once: the alternatives are the first ones in index order all the same."""
    g = torch.Generator().manual_seed(V + top)
    x = torch.zeros((1100, V), dtype=torch.float32)
    few = torch.randperm(V, generator=g)[:20]
    x[1] = NINF                                                     # all but twenty ruled out (some tiles have none of them)
    x[1, few] = torch.randn(20, generator=g)
    x[2, few] = 1.0                                                 # twenty above the others, ties among themselves
    x[3] = torch.finfo(DT[dtype]).min
    x[3, few[:3]] = 2.0
    x[4] = torch.randint(0, 2, (V,), generator=g).float()           # two values, three values
    x[5] = torch.randint(0, 3, (V,), generator=g).float()
    x[6, 1::2] = -0.0                                               # zeros of both signs are equal
    x[7] = NINF
    x[7, V - 1] = 0.5
    x[8] = -(torch.arange(V) // 700).float()                        # steps: ties in the first tile only
    x[9] = (torch.arange(V) // 700).float()
    lane = torch.arange(V) % 2048 // 8                              # one wave's threads hold high values, one of them none
    x[10] = torch.where(lane < 63, 5.0 + torch.rand(V, generator=g), -torch.rand(V, generator=g))
    x[11] = torch.where(lane % 64 == 5, 1.0, 0.0)
    x = x.to(DT[dtype])
    with torch.no_grad():
        logp, ent, tl, ti = token_log_probs(x.cuda(), torch.zeros(1100, dtype=torch.int64, device="cuda"), top=top)
        lone = token_log_probs(x[:12].cuda(), torch.zeros(12, dtype=torch.int64, device="cuda"), top=top)[3]      # (fewer rows: other tiles)
    y = (x[:12].float() + 0.0).cpu()
    want = torch.sort(y, dim=1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ti[:12].cpu(), want) and torch.equal(lone.cpu(), want)
    assert (ti[12:].cpu() == torch.arange(top)).all()
    lp = torch.log_softmax(y.double(), 1).gather(1, want)
    e = (tl[:12].cpu().double() - lp).nan_to_num(0.0, posinf=0.0, neginf=0.0).abs()
    # the answer is rounded three times (difference, scale, minus log of the sum), each by at most 2^-24 of about |lp|: 4 * 2^-24 |lp| where that
    # exceeds the sum's own error (f16's lowest value is -65504: up to 0.0117 of rounding, whatever the kernel)
    assert (e <= 1e-4 + 2.0 ** -22 * lp.nan_to_num(0.0, posinf=0.0, neginf=0.0).abs()).all() and torch.equal(torch.isinf(tl[:12].cpu()), torch.isinf(lp))


@pytest.mark.parametrize("V", [5, 3000, 20011])
def test_tokens_not_a_number_stays_in_its_row(V):
    x, g = logits_of(6, V, torch.float32, V)
    tok = torch.randint(0, V, (6,), generator=g)
    bad = x.clone()
    bad[1, V // 2], bad[2], bad[3, V - 1] = float("nan"), float("nan"), float("inf")
    tok[4] = V                                                      # outside: NaN, not a fault
    tok[5] = -7
    leaf = bad.cuda().requires_grad_()
    logp, ent, tl, ti = token_log_probs(leaf, tok.cuda(), top=3)
    d = torch.autograd.grad([logp, ent, tl], leaf, [torch.ones_like(logp), torch.ones_like(ent), torch.ones_like(tl)])[0].cpu()
    assert torch.isnan(logp.cpu()[1:]).all() and torch.isnan(ent.cpu()[1:4]).all() and torch.isfinite(ent.cpu()[[0, 4, 5]]).all()
    assert ti.cpu()[1, 0] == V // 2 and ti.cpu()[2].tolist() == [0, 1, 2] and ti.cpu()[3, 0] == V - 1
    assert torch.isfinite(d[0]).all() and torch.isnan(d[1]).any() and torch.isnan(d[2]).all() and torch.isnan(d[4]).any()
    tok[:] = torch.tensor([0, -100, -100, -100, 0, 0])              # a padded row's logits may hold anything: no gradient comes back
    leaf = bad.cuda().requires_grad_()
    logp, _, _, _ = token_log_probs(leaf, tok.cuda())
    d = torch.autograd.grad(logp.sum(), leaf)[0]
    assert (logp[1:4] == 0).all() and (d[1:4] == 0).all() and torch.isfinite(d).all()


def test_tokens_views_dims_and_no_rows():
    x, g = logits_of(24, 77, torch.bfloat16, 1)
    tok = torch.randint(0, 77, (24,), generator=g)
    a = check_tokens(x, tok, 5, seed=2)
    wide = torch.zeros((24, 200), dtype=x.dtype).cuda()              # rows with a stride, starting at an odd element
    wide[:, 33:110] = x.cuda()
    assert torch.equal(check_tokens(x, tok, 5, seed=2, view=lambda t: wide[:, 33:110]), a)
    back = x.cuda().t().contiguous().t()                            # unit stride along the rows
    assert torch.equal(check_tokens(x, tok, 5, seed=2, view=lambda t: back), a)
    with torch.no_grad():
        want = token_log_probs(x.cuda(), tok.cuda(), top=5)
        cube = x.view(4, 6, 77).transpose(1, 2).contiguous().cuda()  # B x C x N, classes along 1
        got = token_log_probs(cube, tok.view(4, 6).cuda(), top=5, dim=1)
        assert got[0].shape == (4, 6) and got[2].shape == (4, 6, 5)
        for w, o in zip(want, got):
            assert torch.equal(w.flatten(), o.flatten())
        one = token_log_probs(x[0].cuda(), tok[0].cuda(), top=2)
        assert one[0].shape == () and one[2].shape == (2,) and torch.equal(one[0], want[0][0])
        row = x[:1].cuda().expand(24, 77)                           # one row for many tokens
        assert torch.equal(token_log_probs(row, tok.cuda())[0][0], want[0][0])
    leaf = torch.zeros((0, 9), device="cuda", requires_grad=True)
    logp, ent, tl, ti = token_log_probs(leaf, torch.zeros(0, dtype=torch.int64, device="cuda"), top=3)
    assert logp.shape == (0,) and tl.shape == (0, 3) and torch.autograd.grad(logp.sum(), leaf)[0].shape == (0, 9)
    y = x.cuda().view(4, 6, 77).transpose(1, 2).contiguous().requires_grad_()
    logp = token_log_probs(y, tok.view(4, 6).cuda(), entropy=False, dim=1)[0]
    g1 = torch.autograd.grad(logp.sum(), y)[0]
    z = x.cuda().requires_grad_()
    g2 = torch.autograd.grad(token_log_probs(z, tok.cuda(), entropy=False)[0].sum(), z)[0]
    assert torch.equal(g1.transpose(1, 2).reshape(24, 77), g2)


def teacher(x, K, g, dtype=torch.float32):
    t = torch.log_softmax(x.double() + 0.7 * torch.randn(x.shape, generator=g).double(), 1)
    v, i = torch.topk(t, K, dim=1)
    return i, v.to(dtype)


def check_distill(x, idx, val, T, tail, seed=0, view=lambda t: t):
    g = torch.Generator().manual_seed(seed + 5)
    up = torch.randn(x.shape[0], generator=g)
    leaf = view(x.cuda()).detach().requires_grad_()
    loss = distill_top(leaf, idx.cuda(), val.cuda(), temperature=T, tail=tail)
    d = torch.autograd.grad(loss, leaf, up.cuda())[0]
    want, tol = ref.distill(x.double().numpy(), idx.numpy(), val.double().numpy(), T, tail, up.double().numpy(), half(x.dtype))
    within(loss, want["loss"], tol["loss"], "loss")
    assert d.dtype == x.dtype
    within(d, want["dlogits"], tol["dlogits"], "dlogits")
    return loss.detach(), d


@pytest.mark.parametrize("dtype", list(DT))
@pytest.mark.parametrize("size", SIZES, ids=str)
@pytest.mark.parametrize("K", [1, 20, 64])
@pytest.mark.parametrize("tail", [False, True])
def test_distill(size, dtype, K, tail):
    R, V = size
    x, g = logits_of(R, V, DT[dtype], R + V + K)
    idx, val = teacher(x, min(K, V), g)
    if tail:
        val = val - 1e-3                                            # some mass is always left, also where every output is named
        if K >= V:
            idx[:, -1] = -1                                         # (one output of the rest)
    check_distill(x, idx, val, (1.0, 2.0, 0.7)[V % 3], tail, seed=V)


@pytest.mark.parametrize("V", [8, 700, 9001])
@pytest.mark.parametrize("tail", [False, True])
def test_distill_padding_duplicates_and_masks(V, tail):
    R, K = 14, 8
    x, g = logits_of(R, V, torch.bfloat16, V)
    idx, val = teacher(x, K, g)
    val -= 0.05
    idx[0] = -1                                                     # a row without a teacher
    idx[1, 3:] = -1
    idx[2, ::2] = V                                                 # outside on the other side
    idx[3, 1] = idx[3, 0]                                           # the same output twice
    idx[4, :] = idx[4, 0]
    val[4] = -3.0
    val[5, 2:] = NINF                                               # entries without mass
    val[6] = NINF
    x[7, V // 2:] = NINF                                            # ruled out for the student, some of them the teacher's
    idx[7, :4] = torch.tensor([0, 1, 2, 3])
    idx[7, 4:] = -1
    x[8] = 1.5
    x[9, :] = torch.finfo(torch.bfloat16).min
    x[10, idx[10, 0]] = 80.0                                        # a student that is sure: the rest has next to no mass
    val[11] = torch.log(torch.full((K,), 1.0 / K)) + 0.01           # masses beyond one: nothing is left
    idx[12] = torch.arange(K)
    check_distill(x, idx, val, 1.0, tail, seed=V)
    check_distill(x.float(), idx, val, 2.0, tail, seed=V)
    y = x.clone()                                                   # a row without a teacher may hold anything
    y[0] = float("nan")
    leaf = y.cuda().requires_grad_()
    loss = distill_top(leaf, idx.cuda(), val.cuda(), tail=tail)
    d = torch.autograd.grad(loss[:1].sum(), leaf)[0]
    assert loss[0] == 0 and (d == 0).all()


def test_distill_a_teacher_that_agrees_and_named_all():
    x, g = logits_of(9, 50, torch.float32, 3, scale=1.0)
    lp = torch.log_softmax(x.double(), 1)
    v, i = torch.topk(lp, 10, dim=1)
    loss, d = check_distill(x, i, v.float(), 1.0, True)              # equal distributions: zero up to the inputs' rounding, never negative by much
    assert loss.abs().max() < 1e-6
    v, i = torch.topk(lp, 50, dim=1)
    check_distill(x, i, v.float(), 1.0, False)
    full = (v + 0.5).float()                                        # every output named, more mass than one: no rest, finite
    check_distill(x, i, full, 1.0, True)
    leaf = x.cuda().requires_grad_()                                # every output named and mass left: the loss is inf by its formula
    loss = distill_top(leaf, i.cuda(), (v - 0.5).float().cuda(), tail=True)
    assert torch.isinf(loss).all()
    assert torch.isfinite(torch.autograd.grad(loss.sum(), leaf)[0]).all()


def test_distill_views_types_and_no_rows():
    x, g = logits_of(12, 101, torch.float16, 4)
    idx, val = teacher(x, 7, g)
    loss, d = check_distill(x, idx, val, 1.0, False)
    wide = torch.zeros((12, 300), dtype=x.dtype).cuda()
    wide[:, 7:108] = x.cuda()
    l2, d2 = check_distill(x, idx, val, 1.0, False, view=lambda t: wide[:, 7:108])
    assert torch.equal(loss, l2) and torch.equal(d, d2)
    with torch.no_grad():
        cube = x.view(3, 4, 101).transpose(1, 2).contiguous().cuda()
        l3 = distill_top(cube, idx.view(3, 4, 7).cuda(), val.view(3, 4, 7).cuda(), dim=1)
    assert l3.shape == (3, 4) and torch.equal(l3.flatten(), loss)
    check_distill(x, idx, val.bfloat16(), 1.0, True)
    leaf = torch.zeros((0, 9), device="cuda", requires_grad=True)
    e = distill_top(leaf, torch.zeros((0, 3), dtype=torch.int64, device="cuda"), torch.zeros((0, 3), device="cuda"))
    assert e.shape == (0,) and torch.autograd.grad(e.sum(), leaf)[0].shape == (0, 9)


def test_gradients_against_differences():
    x, g = logits_of(3, 40, torch.float32, 6, scale=1.0)
    tok = torch.tensor([3, 17, 39])
    idx, val = teacher(x, 5, g)
    rng = np.random.RandomState(0)
    d = rng.randn(3, 40)
    e = 1e-4
    x64 = x.double().numpy()

    def along(f):
        return (f(x64 + e * d) - f(x64 - e * d)) / (2 * e)
    # central differences are off by e^2 / 6 of the third derivative (of order one here): 1e-7, against gradients of order one
    for up in range(3):
        leaf = x.cuda().requires_grad_()
        logp, ent, tl, ti = token_log_probs(leaf, tok.cuda(), top=4, temperature=1.5)
        got = torch.autograd.grad((logp, ent, tl)[up].sum(), leaf)[0].double().cpu().numpy()
        slope = along(lambda v: ref.tokens(v, tok.numpy(), 4, 1.5, -100, None, None, None, (0, 0))[0][("logp", "entropy", "top_logp")[up]].sum())
        assert abs((got * d).sum() - slope) < 1e-5 * (1 + np.abs(got * d).sum())
    for tail in (False, True):
        leaf = x.cuda().requires_grad_()
        got = torch.autograd.grad(distill_top(leaf, idx.cuda(), val.cuda(), 1.5, tail).sum(), leaf)[0].double().cpu().numpy()
        slope = along(lambda v: ref.distill(v, idx.numpy(), val.double().numpy(), 1.5, tail, np.ones(3), (0, 0))[0]["loss"].sum())
        assert abs((got * d).sum() - slope) < 1e-5 * (1 + np.abs(got * d).sum())


def test_streams_runs_and_captured_graphs():
    """Eager, on a side stream and replayed from two captured graphs in turn: the same bits."""
    R, V, K = 37, 30011, 20
    xs = [logits_of(R, V, torch.bfloat16, s)[0].cuda() for s in range(3)]
    g = torch.Generator().manual_seed(1)
    tok = torch.randint(0, V, (R,), generator=g).cuda()
    idx, val = (t.cuda() for t in teacher(xs[0].cpu(), K, g))
    one = torch.ones(R, device="cuda")

    def answer(x):
        leaf = x.detach().requires_grad_()
        logp, ent, tl, ti = token_log_probs(leaf, tok, top=8)
        return [logp.detach(), ent.detach(), tl.detach(), ti, torch.autograd.grad([logp, ent], leaf, [one, one])[0]]

    def learn(x):
        leaf = x.detach().requires_grad_()
        loss = distill_top(leaf, idx, val, 2.0, True)
        return [loss.detach(), torch.autograd.grad(loss, leaf, one)[0]]
    want = [(answer(x), learn(x)) for x in xs]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [(answer(x), learn(x)) for x in xs]
    torch.cuda.current_stream().wait_stream(side)
    static = xs[0].clone()
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1):
        o1 = answer(static)
    with torch.cuda.graph(g2):
        o2 = learn(static)
    for i in (0, 1, 2, 1):
        static.copy_(xs[i])
        g1.replay()
        mid = learn(xs[(i + 1) % 3])
        g2.replay()
        torch.cuda.synchronize()
        for a, b, c in ((o1, want[i][0], again[i][0]), (o2, want[i][1], again[i][1])):
            for p, q, s in zip(a, b, c):
                assert torch.equal(p, q) and torch.equal(q, s), i
        assert torch.equal(mid[1], want[(i + 1) % 3][1][1])


def test_more_than_two_to_the_31_elements():
    R, V = 21500, 100003                                            # 2.15e9 logits: offsets pass 32 bits
    x = torch.empty((R, V), dtype=torch.bfloat16, device="cuda").normal_(generator=torch.Generator(device="cuda").manual_seed(2))
    tok = torch.full((R,), V - 1, dtype=torch.int64, device="cuda")
    idx = torch.tensor([[5, V - 1]], device="cuda").expand(R, 2)
    leaf = x.requires_grad_()
    logp, ent, tl, ti = token_log_probs(leaf, tok, top=2)
    d = torch.autograd.grad(logp.sum(), leaf)[0]
    loss = distill_top(leaf, idx, torch.zeros((R, 2), device="cuda"))
    dd = torch.autograd.grad(loss.sum(), leaf)[0]
    rows = [0, 21474, 21475, R - 1]
    xs = x.detach()[rows].double().cpu().numpy()
    want, tol = ref.tokens(xs, np.full(4, V - 1), 2, 1.0, -100, np.ones(4), None, None, half(torch.bfloat16))
    within(logp[rows], want["logp"], tol["logp"], "logp")
    assert np.array_equal(ti[rows].cpu().numpy(), want["top_tokens"])
    within(d[rows], want["dlogits"], tol["dlogits"], "dlogits")
    want, tol = ref.distill(xs, np.array([[5, V - 1]] * 4), np.zeros((4, 2)), 1.0, False, np.ones(4), half(torch.bfloat16))
    within(loss[rows], want["loss"], tol["loss"], "loss")
    within(dd[rows], want["dlogits"], tol["dlogits"], "dlogits")


@pytest.mark.parametrize("V,dtype", [(5, "f32"), (70, "bf16")])
def test_more_rows_than_one_launch_takes(V, dtype):
    R = (1 << 22) + 1003                                            # launches hold 2^22 such rows
    g = torch.Generator(device="cuda").manual_seed(V)
    x = torch.empty((R, V), device="cuda").normal_(generator=g).to(DT[dtype])
    tok = torch.randint(0, V, (R,), generator=g, device="cuda")
    idx = torch.randint(0, V, (R, 2), generator=g, device="cuda")
    val = torch.zeros((R, 2), device="cuda")
    leaf = x.requires_grad_()
    logp, ent, tl, ti = token_log_probs(leaf, tok, top=3)
    d = torch.autograd.grad([logp, ent], leaf, [torch.ones_like(logp), torch.ones_like(ent)])[0]
    loss = distill_top(leaf, idx, val)
    dd = torch.autograd.grad(loss.sum(), leaf)[0]
    rows = [0, (1 << 22) - 1, 1 << 22, (1 << 22) + 1, R - 1]
    xs = x.detach()[rows].double().cpu().numpy()
    one = np.ones(len(rows))
    want, tol = ref.tokens(xs, tok[rows].cpu().numpy(), 3, 1.0, -100, one, one, None, half(DT[dtype]))
    within(logp[rows], want["logp"], tol["logp"], "logp")
    within(ent[rows], want["entropy"], tol["entropy"], "entropy")
    within(tl[rows], want["top_logp"], tol["top_logp"], "top_logp")
    assert np.array_equal(ti[rows].cpu().numpy(), want["top_tokens"])
    within(d[rows], want["dlogits"], tol["dlogits"], "dlogits")
    want, tol = ref.distill(xs, idx[rows].cpu().numpy(), val[rows].double().cpu().numpy(), 1.0, False, one, half(DT[dtype]))
    within(loss[rows], want["loss"], tol["loss"], "loss")
    within(dd[rows], want["dlogits"], tol["dlogits"], "dlogits")


MANY = [(1100, 4099), (700, 10001), (600, 20011)]                   # enough tiles for the largest ones: one, two and three a row in 16 bits


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", MANY, ids=str)
@pytest.mark.parametrize("top", [0, 8])
def test_tokens_many_rows(size, dtype, top):
    R, V = size
    x, g = logits_of(R, V, DT[dtype], R + V)
    x[:, torch.randperm(V, generator=g)[: V // 10]] = NINF
    x[0] = NINF
    tok = x.float().argmax(1)                                       # a given output that is not ruled out, some rows without one
    tok[5:] = torch.where(torch.isinf(x[5:].gather(1, torch.arange(5, R)[:, None])[:, 0]), tok[5:], torch.arange(5, R))
    tok[3::17] = -100
    check_tokens(x, tok, top, T=1.5, seed=V)


@pytest.mark.parametrize("dtype", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("size", MANY, ids=str)
@pytest.mark.parametrize("tail", [False, True])
def test_distill_many_rows(size, dtype, tail):
    R, V = size
    x, g = logits_of(R, V, DT[dtype], R + V + 1)
    idx, val = teacher(x, 64, g)
    idx[torch.rand((R, 64), generator=g) < 0.1] = -1
    idx[2::19] = -1
    idx[4, 7] = idx[4, 9]
    check_distill(x, idx, val, 2.0, tail, seed=V)
