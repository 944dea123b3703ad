"""The sequence and output operators as the framework uses them: the recurrent layer, the recurrent network, a classifier's answers, and a network
that learns from another one's answers.  Against torch in float64 on the CPU, with the filters' stated tolerances (tests/_util.py)."""
import copy

import numpy as np
import pytest
import torch
import torch.nn as nn

from _util import FWD_RTOL, GRAD_RTOL
from alegnn_amd import distill_top, graphgen, linear_recurrence, token_log_probs
from alegnn_amd.modules.architectures import GraphRecurrentNN, SelectionGNN
from alegnn_amd.modules.evaluation import evaluate, predictTop
from alegnn_amd.modules.model import Model
from alegnn_amd.modules.training import Trainer
from alegnn_amd.utils import graphML as gml

pytestmark = pytest.mark.gpu


def gso(N, seed=0):
    A = graphgen.sbm(N, seed=seed, directed=True)
    return np.asarray(A.toarray())[None]


def filt(w, b, S, x):
    """Graph filter in float64: x [R, F, N] -> [R, H, N]."""
    y, xs = 0.0, x
    for k in range(w.shape[2]):
        y = y + torch.einsum('hf,rfn->rhn', w[:, 0, k], xs)
        xs = xs @ S
    return y if b is None else y + b


def layer64(layer, S, x, z0, lengths=None):
    """LinearHiddenState step by step in float64; returns (z, zT, leaves by name, largest forget gate)."""
    p = {k: v.detach().double().cpu().requires_grad_() for k, v in layer.named_parameters()}
    x = x.detach().double().cpu().requires_grad_()
    B, T, F, N = x.shape
    S = torch.from_numpy(S[0]).double()
    flat = x.reshape(B * T, F, N)
    u = torch.tanh(filt(p["aWeights"], p.get("xBias"), S, flat)).reshape(B, T, -1, N)
    i = torch.sigmoid(filt(p["inputGate.weight"], p.get("inputGate.bias"), S, flat)).reshape(B, T, -1, N)
    f = torch.sigmoid(filt(p["forgetGate.weight"], p.get("forgetGate.bias"), S, flat)).reshape(B, T, -1, N)
    h = torch.zeros(u[:, 0].shape, dtype=torch.float64) if z0 is None else z0.double().cpu()
    zs = []
    for t in range(T):
        live = torch.ones(B, dtype=torch.bool) if lengths is None else lengths > t
        new = f[:, t] * h + i[:, t] * u[:, t]
        h = torch.where(live[:, None, None], new, h)
        zs.append(torch.where(live[:, None, None], h, 0.0))
    return torch.stack(zs, 1), h, dict(p, x=x), float(f.max())


@pytest.mark.parametrize("gate", ["element", "node"])
@pytest.mark.parametrize("shape", [(3, 40, 30), (2, 7, 33), (1, 1, 20)], ids=str)
@pytest.mark.parametrize("padded", [False, True])
def test_layer(gate, shape, padded):
    B, T, N = shape
    F, H, K = 3, 8, 3
    torch.manual_seed(0)
    S = gso(N)
    layer = gml.LinearHiddenState(F, H, K, gate=gate)
    layer.addGSO(torch.tensor(S))
    layer.cuda()
    x = torch.randn(B, T, F, N, device="cuda", requires_grad=True)
    z0 = torch.randn(B, H, N, device="cuda")
    lengths = torch.tensor([T, T // 2, 0][:B], dtype=torch.int32, device="cuda") if padded else None
    z, zT = layer(x, z0, lengths)
    assert z.shape == (B, T, H, N) and zT.shape == (B, 1, 1, H, N)
    w, wT = torch.randn_like(z), torch.randn_like(zT)
    ((z * w).sum() + (zT * wT).sum()).backward()
    want, wantT, leaves, fmax = layer64(layer, S, x, z0, None if lengths is None else lengths.cpu())
    ((want * w.double().cpu()).sum() + (wantT * wT.double().cpu().reshape(wantT.shape)).sum()).backward()
    # a state's error is at most (error of gate x state + of gate x input + of the input) / (1 - largest forget gate), each term FWD_RTOL of its filter
    scale = 3.0 / (1.0 - fmax)
    m = float(want.abs().max())
    assert float((z.double().cpu() - want).abs().max()) <= FWD_RTOL * scale * max(m, 1.0)
    assert float((zT.double().cpu().reshape(wantT.shape) - wantT).abs().max()) <= FWD_RTOL * scale * max(m, float(wantT.abs().max()), 1.0)
    for k, v in [*layer.named_parameters(), ("x", x)]:
        g = leaves[k].grad
        assert float((v.grad.double().cpu() - g).abs().max()) <= GRAD_RTOL * scale * max(float(g.abs().max()), 1e-30), k


def test_layer_in_pieces_and_the_network_around_it():
    torch.manual_seed(1)
    B, T, F, N, H = 2, 24, 3, 40, 8
    S = gso(N, 1)
    net = GraphRecurrentNN(F, 4, H, [3, 2], True, torch.tanh, torch.relu, nn.ReLU, [5], S, hiddenLayer=gml.LinearHiddenState).cuda()
    assert isinstance(net.hiddenState, gml.LinearHiddenState)
    x = torch.randn(B, T, F, N, device="cuda")
    z0 = torch.randn(B, H, N, device="cuda")
    with torch.no_grad():
        y = net(x, z0)
        z, zT = net.hiddenState(x, z0)
        parts, s = [], z0
        for t in range(0, T, 5):                                    # served in pieces, the last one a remainder
            zp, s = net.hiddenState(x[:, t:t + 5], s)
            s = s.reshape(B, H, N)
            parts.append(zp)
    assert y.shape == (B, T, 5, N)
    m = float(z.abs().max())
    # both are within the layer's bound of the exact states (the filters run on other batch sizes)
    assert float((torch.cat(parts, 1) - z).abs().max()) <= 2 * FWD_RTOL * 3 / (1 - 0.98) * m
    assert float((s - zT.reshape(B, H, N)).abs().max()) <= 2 * FWD_RTOL * 3 / (1 - 0.98) * m
    loss = nn.CrossEntropyLoss()(net(x, z0).reshape(B * T, 5, N), torch.randint(0, 5, (B * T, N), device="cuda"))
    loss.backward()
    assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in net.parameters())
    net.changeGSO(gso(N, 2))
    assert torch.isfinite(net(x, z0)).all()


class Data:
    def __init__(self, N, n=64, classes=5, seed=0):
        g = torch.Generator().manual_seed(seed)
        w = torch.randn(classes, N, generator=g)
        x = torch.randn(n + 40, 1, N, generator=g)
        y = (x[:, 0] @ w.T + 0.5 * torch.randn(n + 40, classes, generator=g)).argmax(1)
        self.parts = dict(train=(x[:n], y[:n]), valid=(x[n:n + 20], y[n:n + 20]), test=(x[n + 20:], y[n + 20:]))
        self.nTrain = n

    def getSamples(self, kind, *args):
        x, y = self.parts[kind]
        return (x[args[0]], y[args[0]]) if args else (x, y)

    def evaluate(self, yHat, y):
        return (yHat.argmax(1) != y).float().mean()


def model_of(S, seed, tmp_path, name, F=8):
    torch.manual_seed(seed)
    net = SelectionGNN([1, F], [3], True, nn.ReLU, [S.shape[1]], gml.NoPool, [1], [5], torch.tensor(S))
    net.float()
    return Model(net, nn.CrossEntropyLoss(), torch.optim.SGD(net.parameters(), lr=0.05), Trainer, evaluate, "cuda:0", name, str(tmp_path))


def test_a_student_learns_from_a_teachers_answers(tmp_path):
    """Teacher trained, its answers on the training split read with predictTop, the student's Trainer given them: the same steps eagerly, as a replayed
    graph, and by hand."""
    N, K = 30, 3
    S = gso(N, 3).astype(np.float32)
    data = Data(N)
    np.random.seed(0)
    teacher = model_of(S, 0, tmp_path, "teacher")
    teacher.train(data, 2, 16, doPrint=False, printInterval=0, validationInterval=100)
    ans = predictTop(teacher, data, 'train', top=K, temperature=2.0, batchSize=24)
    out = teacher.archit(data.parts['train'][0].cuda()).detach().double().cpu()
    lp = torch.log_softmax(out / 2.0, 1)
    y = data.parts['train'][1]
    want = torch.topk(lp, K, 1)
    near = 1e-4                                                     # the network's own error between batch sizes, well below the gaps looked at
    assert float((ans['logProb'].cpu() - lp.gather(1, y[:, None])[:, 0]).abs().max()) < near
    assert float((ans['entropy'].cpu() + (lp.exp() * lp).sum(1)).abs().max()) < near
    assert float((ans['topLogProb'].cpu() - want.values).abs().max()) < near
    clear = (want.values[:, :-1] - want.values[:, 1:] > near).all(1) & (want.values[:, -1] - torch.sort(lp, 1, descending=True).values[:, K] > near)
    assert torch.equal(ans['topClasses'].cpu()[clear], want.indices[clear]) and clear.any()
    top = (ans['topClasses'], ans['topLogProb'])

    losses, ends = [], []
    for graph in (False, True):
        np.random.seed(1)
        student = model_of(S, 7, tmp_path, "student%d" % graph)
        v = student.train(data, 2, 16, printInterval=0, validationInterval=100, teacherTop=top, distillWeight=0.3, distillTemperature=2.0, hipGraph=graph)
        losses.append(v['lossTrain'])
        ends.append([p.detach().clone() for p in student.archit.parameters()])
    assert np.allclose(losses[0], losses[1], rtol=1e-6) and all(torch.equal(a, b) for a, b in zip(*ends))

    np.random.seed(1)                                               # by hand, with the loss in float64 on the CPU
    student = model_of(S, 7, tmp_path, "hand")
    order = np.random.permutation(data.nTrain)
    first = order[:16]
    x, y = data.getSamples('train', first)
    with torch.no_grad():
        o = student.archit(x.cuda()).double().cpu()
    lq = torch.log_softmax(o, 1)
    ce = -lq.gather(1, y[:, None]).mean()
    l2 = torch.log_softmax(o / 2.0, 1)
    c, v = top[0].cpu()[first], top[1].double().cpu()[first]
    p, q = v.exp(), l2.exp().gather(1, c)
    pr, qr = 1 - p.sum(1), 1 - q.sum(1)
    kl = (p * (v - q.log())).sum(1) + pr * (pr / qr).log()
    assert abs(losses[0][0] - float(0.7 * ce + 0.3 * kl.mean())) < 1e-4
    plain = model_of(S, 7, tmp_path, "plain")
    np.random.seed(1)
    assert abs(plain.train(data, 1, 16, printInterval=0, validationInterval=100)['lossTrain'][0] - float(ce)) < 1e-4


@pytest.mark.parametrize("graph", [False, True])
def test_a_student_of_all_the_classes(tmp_path, graph):
    """predictTop asked for more classes than there are names them all: what rounding leaves of the teacher's mass is no further outcome."""
    S = gso(30, 3).astype(np.float32)
    data = Data(30)
    teacher = model_of(S, 0, tmp_path, "all-teacher")
    ans = predictTop(teacher, data, 'train', top=64, temperature=2.0)
    assert ans['topClasses'].shape == (data.nTrain, 5)
    np.random.seed(1)
    student = model_of(S, 7, tmp_path, "all-student")
    v = student.train(data, 2, 16, printInterval=0, validationInterval=100, teacherTop=(ans['topClasses'], ans['topLogProb']), distillWeight=1.0,
                      distillTemperature=2.0, hipGraph=graph)
    assert np.isfinite(v['lossTrain']).all() and all(torch.isfinite(q).all() for q in student.archit.parameters())
    np.random.seed(1)                                               # the first step by hand
    student = model_of(S, 7, tmp_path, "all-hand")
    first = np.random.permutation(data.nTrain)[:16]
    with torch.no_grad():
        q = torch.log_softmax(student.archit(data.parts['train'][0][first].cuda()).double().cpu() / 2.0, 1)
        p = torch.log_softmax(teacher.archit(data.parts['train'][0][first].cuda()).double().cpu() / 2.0, 1)
    assert abs(v['lossTrain'][0] - float((p.exp() * (p - q)).sum(1).mean())) < 1e-4


def test_recurrent_answers_end_to_end():
    """Recurrent net -> answers over the nodes at every step -> the student's loss on them; gradients against float64 autograd from the logits on."""
    torch.manual_seed(3)
    B, T, F, N, H = 2, 12, 2, 50, 8
    S = gso(N, 4)
    teacher = GraphRecurrentNN(F, 4, H, [3, 2], True, torch.tanh, torch.relu, nn.ReLU, [1], S, hiddenLayer=gml.LinearHiddenState).cuda()
    student = copy.deepcopy(teacher)
    with torch.no_grad():
        for p in student.parameters():
            p.add_(0.1 * torch.randn_like(p))
    x, z0 = torch.randn(B, T, F, N, device="cuda"), torch.zeros(B, H, N, device="cuda")
    where = torch.randint(0, N, (B, T), device="cuda")
    with torch.no_grad():
        logp, ent, top_logp, top_nodes = token_log_probs(teacher(x, z0)[:, :, 0], where, top=8)
    assert logp.shape == (B, T) and top_nodes.shape == (B, T, 8)
    out = student(x, z0)[:, :, 0]
    out.retain_grad()
    loss = distill_top(out, top_nodes, top_logp, tail=True).mean() - token_log_probs(out, where, entropy=False)[0].mean()
    loss.backward()
    o = out.detach().double().cpu().requires_grad_()
    lq = torch.log_softmax(o, 2)
    v, c = top_logp.double().cpu(), top_nodes.cpu()
    p = v.exp()
    pr = 1 - p.sum(2)
    rest = torch.ones(B, T, N, dtype=torch.bool).scatter(2, c, False)
    qr = torch.where(rest, lq.exp(), 0.0).sum(2)
    want = ((p * (v - lq.gather(2, c))).sum(2) + pr * (pr / qr).log()).mean() - lq.gather(2, where.cpu()[..., None]).mean()
    want.backward()
    assert abs(float(loss) - float(want)) < 1e-5 * (1 + abs(float(want)))
    assert float((out.grad.double().cpu() - o.grad).abs().max()) <= 1e-5 * float(o.grad.abs().max())
    assert all(torch.isfinite(q.grad).all() for q in student.parameters())


def test_refusals_on_the_gpu():
    u = torch.zeros(2, 3, 4, 5, device="cuda")
    with pytest.raises(TypeError, match="dtype"):
        linear_recurrence(u.double(), u.double())
    with pytest.raises(TypeError, match="q_check"):
        linear_recurrence(u, u.bfloat16())
    with pytest.raises(TypeError, match="z0"):
        linear_recurrence(u, u, None, torch.zeros(2, 4, 5, device="cuda", dtype=torch.bfloat16))
    with pytest.raises(AssertionError, match="z0"):
        linear_recurrence(u, u, None, torch.zeros(2, 4, 4, device="cuda"))
    with pytest.raises(TypeError, match="lengths"):
        linear_recurrence(u, u, lengths=torch.zeros(2, dtype=torch.int64, device="cuda"))
    with pytest.raises(AssertionError, match="lengths"):
        linear_recurrence(u, u, lengths=torch.zeros(3, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        linear_recurrence(u, u.cpu())
    x, t = torch.zeros(3, 7, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda")
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="temperature"):
            token_log_probs(x, t, temperature=bad)
        with pytest.raises(ValueError, match="temperature"):
            distill_top(x, t[:, None], x[:, :1], temperature=bad)
    for top in (-1, 8, 65):
        with pytest.raises(AssertionError, match="top"):
            token_log_probs(x, t, top=top)
    with pytest.raises(AssertionError, match="tokens"):
        token_log_probs(x, t[:2])
    with pytest.raises(TypeError, match="tokens"):
        token_log_probs(x, t.int())
    with pytest.raises(TypeError, match="logits"):
        token_log_probs(x.double(), t)
    with pytest.raises(AssertionError, match="no outputs"):
        token_log_probs(x[:, :0], t)
    with pytest.raises(RuntimeError, match="CPU"):
        token_log_probs(x, t.cpu())
    with pytest.raises(AssertionError, match="indices"):
        distill_top(x, torch.zeros(3, 65, dtype=torch.int64, device="cuda"), torch.zeros(3, 65, device="cuda"))
    with pytest.raises(AssertionError, match="values"):
        distill_top(x, t[:, None], x[:, :2])
    with pytest.raises(TypeError, match="indices"):
        distill_top(x, t[:, None].int(), x[:, :1])
    with pytest.raises(NotImplementedError, match="constants"):
        distill_top(x.requires_grad_(), t[:, None], torch.zeros(3, 1, device="cuda", requires_grad=True))
    y = torch.randn(3, 7, device="cuda", requires_grad=True)        # a second derivative is refused, not wrong
    g = torch.autograd.grad(distill_top(y, t[:, None], torch.zeros(3, 1, device="cuda")).sum(), y, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()
    v = torch.randn(1, 4, 2, 2, device="cuda", requires_grad=True)
    g = torch.autograd.grad(linear_recurrence(v, torch.ones_like(v), v)[0].sum(), v, create_graph=True)[0]
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_backward_captured_from_detached_leaves_while_an_eager_graph_lives():
    """torch ends the process when a backward pass is captured whose leaves also belong to a living eager graph (their accumulation nodes stay on the
    eager stream).  Captured from detached leaves of the same storage it is sound: every replay gives the eager results, and the eager graph is
    still there afterwards."""
    g = torch.Generator(device="cuda").manual_seed(0)
    u = torch.randn(2, 50, 3, 8, device="cuda", generator=g, requires_grad=True)
    q = torch.rand(2, 50, 1, 8, device="cuda", generator=g).requires_grad_()
    x = torch.randn(9, 300, device="cuda", generator=g, requires_grad=True)
    tok = torch.randint(0, 300, (9,), device="cuda", generator=g)
    zero = torch.zeros(9, 1, device="cuda")

    def body():
        a, b, c = (t.detach().requires_grad_() for t in (u, q, x))
        z, zT = linear_recurrence(a, b)
        logp, ent, _, _ = token_log_probs(c, tok)
        loss = distill_top(c, tok[:, None], zero)
        ends = [z, zT, logp, ent, loss]
        grads = torch.autograd.grad(ends, [a, b, c], [torch.ones_like(e) for e in ends])
        return [e.detach() for e in ends], grads
    z, _ = linear_recurrence(u, q)
    alive = z.sum() + token_log_probs(x, tok)[0].sum()              # not yet differentiated
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ends, grads = body()
    first = torch.autograd.grad(alive, [u, q, x])
    assert all(torch.isfinite(t).all() for t in first)
    for i in range(3):
        with torch.no_grad():
            u.mul_(0.9), x.mul_(1.1)
        graph.replay()
        wends, wgrads = body()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip([*ends, *grads], [*wends, *wgrads])), i


def test_forward_mode_derivatives_are_refused():
    """A tangent is not dropped without a word, whichever input carries it."""
    import torch.autograd.forward_ad as fwAD
    u, q = torch.randn(2, 5, 3, 4, device="cuda"), torch.rand(2, 5, 3, 4, device="cuda")
    z0, x, t, v = torch.randn(2, 3, 4, device="cuda"), torch.randn(3, 7, device="cuda"), torch.tensor([0, 3, 6], device="cuda"), torch.zeros(3, 1, device="cuda")
    with fwAD.dual_level():
        def dual(a):
            return fwAD.make_dual(a, torch.ones_like(a))
        for grad in (False, True):
            u, x = u.detach().requires_grad_(grad), x.detach().requires_grad_(grad)
            for call in (lambda: linear_recurrence(dual(u), q), lambda: linear_recurrence(u, dual(q)), lambda: linear_recurrence(u, q, dual(q)),
                         lambda: linear_recurrence(u, q, q, dual(z0)), lambda: token_log_probs(dual(x), t), lambda: distill_top(dual(x), t[:, None], v),
                         lambda: distill_top(x, t[:, None], dual(v)), lambda: token_log_probs(dual(x).t(), t, dim=0)):
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call()
        linear_recurrence(u, q, q, z0), token_log_probs(x, t), distill_top(x, t[:, None], v)      # no tangent: served as ever
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda a: token_log_probs(a, t)[0], (x.detach(),), (torch.ones_like(x),))
    with pytest.raises(RuntimeError):
        torch.func.vmap(lambda a: linear_recurrence(a[None], q[:1])[0])(u.detach())
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: distill_top(a, t[:, None], v).sum())(x.detach())


def test_a_student_of_padded_entries(tmp_path):
    """As many entries as classes or more, some of them padding: a row that names every class has no further outcome, one that does not keeps it."""
    S = gso(30, 3).astype(np.float32)
    data = Data(30)
    teacher = model_of(S, 0, tmp_path, "pad-teacher")
    ans = predictTop(teacher, data, 'train', top=5, temperature=2.0)
    classes = torch.cat((ans['topClasses'], torch.full((data.nTrain, 2), -1, device="cuda")), 1)
    values = torch.cat((ans['topLogProb'], torch.zeros(data.nTrain, 2, device="cuda")), 1)
    classes[::3, 2:5] = -1                                          # two named classes
    classes[1::9] = -1                                              # no teacher at all
    classes[2, 5], values[2, 5] = 99, 0.5                           # padding on the other side
    losses, ends = [], []
    for graph in (False, True):                                     # eagerly, and eight replays of a graph
        np.random.seed(1)
        student = model_of(S, 7, tmp_path, "pad-student%d" % graph)
        v = student.train(data, 2, 16, printInterval=0, validationInterval=100, teacherTop=(classes, values), distillWeight=1.0, distillTemperature=2.0,
                          hipGraph=graph)
        losses.append(v['lossTrain'])
        ends.append([p.detach().clone() for p in student.archit.parameters()])
        assert np.isfinite(v['lossTrain']).all() and all(torch.isfinite(q).all() for q in ends[-1])
    assert np.allclose(losses[0], losses[1], rtol=1e-6) and all(torch.equal(a, b) for a, b in zip(*ends))
    np.random.seed(1)                                               # the first step by hand
    student = model_of(S, 7, tmp_path, "pad-hand")
    first = np.random.permutation(data.nTrain)[:16]
    with torch.no_grad():
        lq = torch.log_softmax(student.archit(data.parts['train'][0][first].cuda()).double().cpu() / 2.0, 1)
        lp = torch.log_softmax(teacher.archit(data.parts['train'][0][first].cuda()).double().cpu() / 2.0, 1)
    want = 0.0
    for r, c in enumerate(classes.cpu()[first]):
        c = c[(c >= 0) & (c < 5)]
        if len(c):
            want += float((lp[r, c].exp() * (lp[r, c] - lq[r, c])).sum())
            rest = torch.ones(5, dtype=torch.bool)
            rest[c] = False
            if rest.any():
                pr, qr = lp[r, rest].exp().sum(), lq[r, rest].exp().sum()
                want += float(pr * (pr / qr).log())
    assert abs(losses[0][0] - want / 16) < 1e-4


@pytest.mark.parametrize("gate", ["element", "node"])
def test_what_padded_steps_of_a_layer_hold_does_not_matter(gate):
    """Padding of NaN and inf gives the states and the gradients of zero padding, bit for bit: the filters never see it."""
    torch.manual_seed(0)
    B, T, F, N, H = 3, 20, 3, 30, 8
    layer = gml.LinearHiddenState(F, H, 3, gate=gate)
    layer.addGSO(torch.tensor(gso(N)))
    layer.cuda()
    lengths = torch.tensor([T, 7, 0], dtype=torch.int32, device="cuda")
    dead = (torch.arange(T, device="cuda")[None, :] >= lengths[:, None])[:, :, None, None]
    x, z0 = torch.randn(B, T, F, N, device="cuda"), torch.randn(B, H, N, device="cuda")
    w, wT = torch.randn(B, T, H, N, device="cuda"), torch.randn(B, 1, 1, H, N, device="cuda")
    a, S = torch.randn(H, 1, 2, F, device="cuda", requires_grad=True), layer._gso
    f = torch.rand(B, T, 1, N, device="cuda")

    def passes(padding):
        leaf = torch.where(dead, padding, x).requires_grad_()
        z, zT = layer(leaf, z0, lengths)
        grads = torch.autograd.grad([z, zT], [leaf, *layer.parameters()], [w, wT])
        y, yT = gml.LinearGRNN(a, S, leaf, z0, torch.tanh, None, f, lengths=lengths)
        return [z, zT, *grads, y, yT, *torch.autograd.grad([y, yT], [leaf, a], [w, wT[:, 0, 0]])]
    want = passes(torch.zeros_like(x))
    bad = torch.full_like(x, float("nan"))
    bad[:, ::2] = float("inf")
    assert all(torch.isfinite(t).all() for t in want)
    for i, (p, q) in enumerate(zip(passes(bad), want)):
        assert torch.equal(p, q), i


def test_lengths_of_a_layer_are_refused_as_the_recurrences_own():
    layer = gml.LinearHiddenState(2, 4, 2)
    layer.addGSO(torch.tensor(gso(30)))
    layer.cuda()
    x = torch.randn(3, 5, 2, 30, device="cuda")
    for lengths, kind, word in ((torch.zeros(2, dtype=torch.int32, device="cuda"), AssertionError, "lengths"),
                                (torch.zeros(3, 1, dtype=torch.int32, device="cuda"), AssertionError, "lengths"),
                                (torch.zeros(3, dtype=torch.int64, device="cuda"), TypeError, "lengths"),
                                (torch.zeros(3, dtype=torch.int32), RuntimeError, "no CPU fallback")):
        with pytest.raises(kind, match=word):
            layer(x, None, lengths)
        with pytest.raises(kind, match=word):
            gml.LinearGRNN(layer.aWeights, layer._gso, x, None, None, None, torch.ones(3, 5, 1, 1, device="cuda"), lengths=lengths)
