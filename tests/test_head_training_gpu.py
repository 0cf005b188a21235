"""The loss, the gradients' norm and the optimiser's step together, as a training program calls them: a head over a large
vocabulary (half-precision copy of the weights, fp32 master weights) and the layer in front of it."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
F8 = torch.float8_e4m3fn


@pytest.fixture(scope='module')
def ops():
    from dp_cgans_amd import ops as o
    return o


class Head(object):
    """One head: master weights, their copy in the products' type, gradients and states; every buffer stays where it is."""

    def __init__(self, ops, T, D, V, dtype, eight, seed=0, max_norm=0.05, lr=1e-2, eps=1e-4):
        g = torch.Generator(device=DEV).manual_seed(seed)
        self.ops, self.max_norm, self.lr, self.eps = ops, max_norm, lr, eps
        self.master = torch.randn(V, D, device=DEV, generator=g) / math.sqrt(D)
        self.w = self.master.to(dtype)
        self.h, self.target = torch.empty(T, D, dtype=dtype, device=DEV), torch.empty(T, dtype=torch.int64, device=DEV)
        self.dh, self.dw = torch.empty_like(self.h), torch.empty_like(self.w)
        self.loss, self.total, self.out = (torch.empty(n, device=DEV) for n in (T, 1, 2))
        self.ws = torch.empty(ops.linear_cross_entropy_ws(T, D, V, dtype), dtype=torch.uint8, device=DEV)
        self.t, self.rng = torch.zeros(1, dtype=torch.int32, device=DEV), ops.new_rng(seed, DEV)
        more = {}
        if eight:
            (m, ms), (v, vs) = ops.adamw_state8(self.master), ops.adamw_state8(self.master)
            more = dict(m_scale=[ms], v_scale=[vs])
        else:
            m, v = torch.zeros_like(self.master), torch.zeros_like(self.master)
        self.state = [m, v] + [x[0] for x in more.values()]
        copies = None if dtype == torch.float32 else [self.w]
        self.plan = ops.adamw_plan([self.master if copies else self.w], [self.dw], [m], [v], wd=0.1, copies=copies, **more)

    def batch(self, seed):
        g = torch.Generator(device=DEV).manual_seed(1000 + seed)
        self.h.copy_(torch.randn(self.h.shape, device=DEV, generator=g))
        self.target.copy_(torch.randint(0, self.w.shape[0], self.target.shape, device=DEV, generator=g))
        self.target[::9] = -100

    def step(self):
        o = self.ops
        o.linear_cross_entropy(self.h, self.w, self.target, self.loss, self.ws, dh=self.dh, dw=self.dw, total=self.total)
        o.grad_clip(self.plan, self.max_norm, self.out, t_dev=self.t)
        o.adamw_step(self.plan, self.lr, eps=self.eps, coef=self.out[1:], t_dev=self.t, t_host=0, rng=self.rng)
        o.state_advance(self.rng)

    def tensors(self):
        return [x.view(torch.uint8) if x.dtype == F8 else x
                for x in [self.master, self.w, self.dh, self.dw, self.loss, self.total, self.out, self.t] + self.state]


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16, torch.float32])
def test_one_step_against_the_formulas(ops, dtype):
    """dW, its norm and the first step, each from the operator's own inputs in fp64.  The first step moves a weight by
    lr g' / (|g'| + eps): an error of g' comes through divided by eps at most."""
    T, D, V = 500, 256, 276
    a = Head(ops, T, D, V, dtype, False)
    a.batch(0)
    h, w, w0 = a.h.double(), a.w.double(), (a.master if dtype != torch.float32 else a.w).double().clone()
    live = a.target != -100
    at = torch.where(live, a.target, 0)
    p = torch.softmax(h @ w.t(), 1)
    p[torch.arange(T, device=DEV), at] -= 1
    p *= live[:, None] / live.sum()
    a.step()
    got = a.dw.double()
    u = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}[dtype]
    # softmax - onehot and dW rounded to the type once each, 2^-11 for the probabilities' first form, fp32 sums of T and D
    bound = (2 * u + (2.0 ** -11 if dtype != torch.float32 else 0) + (T + 4 * D) * 2.0 ** -24) * (p.abs().t() @ h.abs()) + 2.0 ** -25
    assert ((got - p.t() @ h).abs() <= bound).all()
    assert ((a.dh.double() - p @ w).abs() <= (2 * u + 2.0 ** -11 + (V + 4 * D) * 2.0 ** -24) * (p.abs() @ w.abs()) + 2.0 ** -25).all()
    norm = got.square().sum().sqrt().item()
    assert abs(a.out[0].item() - norm) <= 4 * 2.0 ** -24 * norm
    coef = min(1.0, a.max_norm / norm)
    assert abs(a.out[1].item() - coef) <= 4 * 2.0 ** -24 * coef
    g = coef * got
    want = w0 * (1 - a.lr * 0.1) - a.lr * g / (g.abs() + a.eps)
    new = (a.master if dtype != torch.float32 else a.w).double()
    assert ((new - want).abs() <= 8 * 2.0 ** -24 * (w0.abs() + want.abs()) + 32 * 2.0 ** -24 * a.lr + a.lr * 16 * 2.0 ** -24 * g.abs() / a.eps).all()
    if dtype != torch.float32:
        assert torch.equal(a.w, a.master.to(dtype))
    assert a.t.item() == 1


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_steps_replayed_from_a_graph_equal_eager_steps(ops, dtype, eight):
    """Several steps on changing batches, one of which overflows (an infinity in a row that counts): that step leaves
    weights, states and the step count alone, and the next one goes on."""
    a, b = (Head(ops, 300, 128, 1800, dtype, eight) for _ in range(2))
    st = torch.cuda.Stream()
    a.batch(0)
    keep = [x.clone() for x in a.tensors()]
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        a.step()                                               # warm-up, undone
    st.synchronize()
    for x, y in zip(a.tensors(), keep):
        x.copy_(y)
    a.rng[1] = 0
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        a.step()
    count = 0
    for i in range(5):
        a.batch(i)
        b.batch(i)
        if i == 2:
            a.h[1, 3] = b.h[1, 3] = float('inf')
        torch.cuda.synchronize()
        before = [x.clone() for x in (a.master, a.w, *[s.view(torch.uint8) if s.dtype == F8 else s for s in a.state])]
        graph.replay()
        torch.cuda.synchronize()
        b.step()
        torch.cuda.synchronize()
        for k, (x, y) in enumerate(zip(a.tensors(), b.tensors())):
            assert torch.equal(torch.nan_to_num(x) if x.is_floating_point() else x, torch.nan_to_num(y) if y.is_floating_point() else y), (i, k)
        if i == 2:
            assert not math.isfinite(a.total.item()) and a.out[1].item() == 0
            for x, y in zip((a.master, a.w, *[s.view(torch.uint8) if s.dtype == F8 else s for s in a.state]), before):
                assert torch.equal(x, y)
        else:
            count += 1
        assert a.t.item() == count


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_two_heads_at_once_on_two_streams(ops, dtype):
    """Overlapping calls with a workspace and a plan each give what they give one after the other."""
    a, b = Head(ops, 700, 256, 5000, dtype, True, seed=1), Head(ops, 400, 512, 9001, dtype, False, seed=2)
    c, d = Head(ops, 700, 256, 5000, dtype, True, seed=1), Head(ops, 400, 512, 9001, dtype, False, seed=2)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for i in range(3):
        for x in (a, b, c, d):
            x.batch(i)
        torch.cuda.synchronize()
        for x, st in ((a, streams[0]), (b, streams[1])):
            with torch.cuda.stream(st):
                x.step()
        torch.cuda.synchronize()
        for x in (c, d):
            x.step()
            torch.cuda.synchronize()
        for x, y in ((a, c), (b, d)):
            for k, (s, t) in enumerate(zip(x.tensors(), y.tensors())):
                assert torch.equal(s, t), (i, k)
