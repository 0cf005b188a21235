"""grad_clip and adamw_step (many tensors, 32- and 8-bit states) against plain fp64 arithmetic.

Tolerances: a value held in a type of eps e is off by at most e/2 relative (fp32 2^-24, bf16 2^-8, fp16 2^-11).  The step's
fp32 chain has fewer than 16 roundings, each at most 2^-24 of its largest operand, plus the 1-ulp rounding of the
hyper-parameters to fp32 (each 2^-24 relative)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
F8 = torch.float8_e4m3fn
SIZES = [1, 7, 8, 127, 128, 129, 2047, 2049, 10007]


@pytest.fixture(scope='module')
def ops():
    from dp_cgans_amd import ops as o
    return o


def gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def randn(g, n):
    return torch.randn(n, device=DEV, generator=g)


def make(sizes, p_t, g_t, seed, eight=False, offset=0):
    """Tensors at ``offset`` elements past an aligned address."""
    g = gen(seed)
    cut = lambda x: torch.cat([x.new_zeros(16), x])[16:] if not offset else torch.cat([x.new_zeros(offset), x])[offset:]  # noqa: E731
    s = dict(p=[cut(randn(g, n).to(p_t)) for n in sizes], g=[cut((1e-3 * randn(g, n)).to(g_t)) for n in sizes])
    if eight:
        s['m'] = [cut((100 * randn(g, n)).clamp(-448, 448).to(F8).view(torch.uint8)).view(F8) for n in sizes]
        s['v'] = [cut((150 * randn(g, n)).abs().clamp(0, 448).to(F8).view(torch.uint8)).view(F8) for n in sizes]
        nb = lambda n: -(-n // 128)  # noqa: E731
        s['m_scale'] = [1e-5 * (0.5 + torch.rand(nb(n), device=DEV, generator=g)) for n in sizes]
        s['v_scale'] = [1e-5 * (0.5 + torch.rand(nb(n), device=DEV, generator=g)) for n in sizes]
        s['dither'] = [cut(torch.randint(-32768, 32768, (n,), device=DEV, generator=g, dtype=torch.int16)) for n in sizes]
    else:
        s['m'] = [cut(3e-4 * randn(g, n)) for n in sizes]
        s['v'] = [cut((1e-3 * randn(g, n)) ** 2) for n in sizes]
    return s


def plan_of(ops, s, **kw):
    more = {k: s[k] for k in ('m_scale', 'v_scale', 'dither') if k in s}
    more.update(kw)
    return ops.adamw_plan(s['p'], s['g'], s['m'], s['v'], **more)


def clone(s):
    return {k: [t.clone() for t in v] for k, v in s.items()}


def wide(codes, scales):
    return codes.float().double() * scales.double().repeat_interleave(128)[:codes.numel()]


def oracle(s, k, lr, wd, b1, b2, eps, t, coef=1.0):
    """(p, m, v, bound of what fp32 arithmetic may differ in p / m / v) of tensor k after one step, in fp64."""
    g = s['g'][k].double() * coef
    if 'm_scale' in s:
        m0, r0 = wide(s['m'][k], s['m_scale'][k]), wide(s['v'][k], s['v_scale'][k])
        v0 = r0 * r0
    else:
        m0, v0 = s['m'][k].double(), s['v'][k].double()
    m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
    root = (v / (1 - b2 ** t)).sqrt()
    p0 = s['p'][k].double()
    up = lr / (1 - b1 ** t) * m / (root + eps)
    p = p0 * (1 - lr * wd) - up
    em = 8 * 2.0 ** -24 * ((b1 * m0).abs() + ((1 - b1) * g).abs())
    ev = 8 * 2.0 ** -24 * v
    ep = 8 * 2.0 ** -24 * (p0.abs() + p.abs()) + 16 * 2.0 ** -24 * up.abs() + lr / (1 - b1 ** t) * em / (root + eps)
    return p, m, v, ep, em, ev


HYPER = dict(lr=1e-2, b1=0.9, b2=0.99, eps=1e-8)


def run_case(ops, s, wds, t=3, copies=None, coef=None, **kw):
    before = clone(s)
    plan = plan_of(ops, s, wd=wds, copies=copies)
    c = None if coef is None else torch.tensor([coef], device=DEV)
    ops.adamw_step(plan, t_host=t, coef=c, **HYPER, **kw)
    torch.cuda.synchronize()
    return before


@pytest.mark.parametrize('p_t,g_t', [(torch.float32, torch.float32), (torch.float32, torch.bfloat16),
                                     (torch.bfloat16, torch.bfloat16), (torch.float16, torch.float16),
                                     (torch.bfloat16, torch.float32)])
@pytest.mark.parametrize('offset', [0, 1])
def test_adamw_32_bit_states(ops, p_t, g_t, offset):
    s = make(SIZES, p_t, g_t, 3, offset=offset)
    wds = [0.1 * (k % 3) for k in range(len(SIZES))]
    copies = [torch.full((n,), 7.0, dtype=torch.bfloat16, device=DEV) for n in SIZES]
    before = run_case(ops, s, wds, copies=copies, coef=0.25)
    for k in range(len(SIZES)):
        p, m, v, ep, em, ev = oracle(before, k, wd=wds[k], t=3, coef=0.25, **HYPER)
        assert ((s['m'][k].double() - m).abs() <= em + 1e-40).all()
        assert ((s['v'][k].double() - v).abs() <= ev + 1e-44).all()
        tiny = 2.0 ** -25 if p_t == torch.float16 else 0.0               # half a step of fp16 below 2^-14
        assert ((s['p'][k].double() - p).abs() <= ep + (HALF[p_t] * (p.abs() + ep) + tiny if p_t != torch.float32 else 0)).all(), k
        assert ((copies[k].double() - p).abs() <= ep + HALF[torch.bfloat16] * (p.abs() + ep)).all()
        assert torch.equal(s['g'][k], before['g'][k])


def check_held(codes, scales, x, ex, dither, up):
    """x [n] fp64 (known to within ex) against its 8-bit form: the block's largest on 448, every code one of the two
    grid neighbours, the one the random bits choose unless x is within its error of the border."""
    n = x.numel()
    pad = -n % 128
    blocks = lambda y: torch.cat([y, y.new_zeros(pad)]).view(-1, 128)  # noqa: E731
    top = blocks(x.abs()).amax(1).clamp(min=2.0 ** -100)
    etop = blocks(ex).amax(1)
    assert ((scales.double() * 448 - top).abs() <= etop + 4 * 2.0 ** -24 * top).all()
    sc = scales.double().repeat_interleave(128)[:n]
    y = (x.abs() / sc).clamp(max=448)
    low = y.clamp(min=2.0 ** -6)
    step = low / torch.frexp(low)[0] / 16                              # exact powers of two (the GPU's pow is not)
    u = (dither.int() & 0xffff).double() / 65536
    want = torch.floor(y / step + u) * step
    if up:
        want = torch.where((x > 0) & (want == 0), torch.full_like(want, 2.0 ** -9), want)
    got = codes.float().double()
    assert torch.equal(torch.signbit(got) | (got == 0), torch.signbit(x) | (got == 0))
    got = got.abs()
    # error of y in steps: that of x, of the scale (1 division) and of one multiplication; 2^-21 for the sum with u
    slack = (ex / sc + 4 * 2.0 ** -24 * y) / step + 2.0 ** -21
    frac = y / step + u
    near = (frac - torch.round(frac)).abs() <= slack
    assert ((got - want).abs() <= 2 * step * near).all()
    return float((got != want).double().mean())


@pytest.mark.parametrize('p_t,g_t,offset', [(torch.float32, torch.float32, 0), (torch.bfloat16, torch.bfloat16, 0),
                                            (torch.float32, torch.bfloat16, 1), (torch.float16, torch.float16, 3)])
def test_adamw_8_bit_states(ops, p_t, g_t, offset):
    s = make(SIZES, p_t, g_t, 5, eight=True, offset=offset)
    before = run_case(ops, s, [0.1] * len(SIZES), coef=0.5)
    for k in range(len(SIZES)):
        p, m, v, ep, em, ev = oracle(before, k, wd=0.1, t=3, coef=0.5, **HYPER)
        tiny = 2.0 ** -25 if p_t == torch.float16 else 0.0
        assert ((s['p'][k].double() - p).abs() <= ep + (HALF[p_t] * (p.abs() + ep) + tiny if p_t != torch.float32 else 0)).all(), k
        check_held(s['m'][k], s['m_scale'][k], m, em, before['dither'][k], False)
        check_held(s['v'][k], s['v_scale'][k], v.sqrt(), 0.5 * ev / v.sqrt().clamp(min=1e-30) + 2.0 ** -24 * v.sqrt(),
                   before['dither'][k], True)


@pytest.mark.parametrize('eight', [False, True])
def test_adamw_unaligned_tensors_give_the_aligned_bits(ops, eight):
    a = make(SIZES, torch.float32, torch.bfloat16, 7, eight=eight)
    b = make(SIZES, torch.float32, torch.bfloat16, 7, eight=eight, offset=1)
    for s in (a, b):
        run_case(ops, s, 0.1)
    for name in a:
        for x, y in zip(a[name], b[name]):
            assert torch.equal(x.view(torch.uint8) if x.dtype == F8 else x, y.view(torch.uint8) if y.dtype == F8 else y), name


def test_adamw_8_bit_draws_are_the_documented_ones(ops):
    sizes = [5, 130, 2100]
    a = make(sizes, torch.float32, torch.float32, 9, eight=True)
    b = clone(a)
    del a['dither']
    rng = ops.new_rng(77, DEV)
    run_case(ops, a, 0.0, rng=rng)
    words = torch.empty(sum(-(-n // 8) for n in sizes) * 4, dtype=torch.int32, device=DEV)
    ops.fill(words, ops.FILL_U32, rng, ops.SITE_DITHER)
    at = 0
    for k, n in enumerate(sizes):
        w = words[at:at + -(-n // 8) * 4]
        b['dither'][k] = w.view(torch.int16)[:n].clone()              # little-endian: low half first
        at += -(-n // 8) * 4
    run_case(ops, b, 0.0)
    for name in a:
        for x, y in zip(a[name], b[name]):
            assert torch.equal(x.view(torch.uint8) if x.dtype == F8 else x, y.view(torch.uint8) if y.dtype == F8 else y), name


def test_adamw_8_bit_rounding_is_unbiased_over_all_random_bits(ops):
    """65536 elements of one value, one for each setting of the 16 bits: the mean of what is held is the value, to the
    resolution of the bits (1/65536 of a grid step, and the one element per border case)."""
    n, lanes = 65536 * 2, torch.arange(65536, device=DEV)
    for value in (0.3, 0.0111, 1.7e-5, 0.9):
        m = torch.zeros(n, dtype=torch.uint8, device=DEV).view(F8)
        v = torch.zeros(n, dtype=torch.uint8, device=DEV).view(F8)
        z = lambda: torch.zeros(n // 128, device=DEV)  # noqa: E731
        g = torch.zeros(n, device=DEV)
        g.view(-1, 128)[:, :64] = value
        g.view(-1, 128)[:, 64:] = 1.0                                 # the block's largest
        d = torch.zeros(n, dtype=torch.int16, device=DEV)
        d.view(-1, 128)[:, :64] = lanes.to(torch.int32).to(torch.int16).view(-1, 64)
        ms, vs = z(), z()
        plan = ops.adamw_plan([torch.zeros(n, device=DEV)], [g], [m], [v], m_scale=[ms], v_scale=[vs], dither=[d])
        ops.adamw_step(plan, lr=0.0, b1=0.0, b2=0.0, t_host=1)
        for c, sc in ((m, ms), (v, vs)):
            held = wide(c, sc).view(-1, 128)[:, :64].mean().item()
            x = g[0].item()
            y = x * 448
            step = 2.0 ** -9 if y < 2.0 ** -6 else 2.0 ** (math.floor(math.log2(y)) - 3)
            assert abs(held - x) <= 3 / 65536 * step / 448 + 4 * 2.0 ** -24 * x, (value, held)


def test_adamw_8_bit_second_moment_decays_without_gradients(ops):
    """500 steps at b2 = 0.999 and g = 0: the root falls by 0.999^250.  Each rounding moves an element by less than a
    grid step (1/8 relative), independently: the mean over 2^17 elements is within 5 * sqrt(500) / 8 / 2^8.5 = 4 %
    (with rounding to the nearest, nothing but the block's largest would ever move: 28 % too high)."""
    n = 1 << 17
    g = torch.zeros(n, device=DEV)
    r = torch.rand(n, device=DEV, generator=gen(2)) * 100 + 100
    v = r.to(F8)
    vs = torch.full((n // 128,), 1e-4, device=DEV)
    m, ms = ops.adamw_state8(g)
    start = wide(v, vs).mean().item()
    plan = ops.adamw_plan([torch.zeros(n, device=DEV)], [g], [m], [v], m_scale=[ms], v_scale=[vs])
    rng = ops.new_rng(5, DEV)
    t = torch.zeros(1, dtype=torch.int32, device=DEV)
    for _ in range(500):
        ops.adamw_step(plan, lr=1e-3, t_dev=t, t_host=1, rng=rng)
        ops.state_advance(rng, t_a=t)
    assert abs(wide(v, vs).mean().item() / start / 0.999 ** 250 - 1) < 0.04


@pytest.mark.parametrize('eight', [False, True])
def test_adamw_non_finite_gradients_stay_where_they_are(ops, eight):
    s = make([300], torch.float32, torch.float32, 11, eight=eight)
    s['g'][0][5], s['g'][0][200] = float('nan'), float('inf')
    before = run_case(ops, s, 0.0)
    bad = torch.zeros(300, dtype=torch.bool, device=DEV)
    bad[5] = bad[200] = True
    m = s['m'][0].float()
    assert torch.equal(torch.isnan(s['p'][0]), bad)                   # inf / sqrt(inf) = NaN
    assert torch.equal(~torch.isfinite(m), bad)
    before['g'][0][5] = before['g'][0][200] = 0
    p, mm, v, ep, em, ev = oracle(before, 0, wd=0.0, t=3, **HYPER)
    assert ((s['p'][0].double() - p).abs() <= ep)[~bad].all()
    if eight:
        assert torch.isfinite(s['m_scale'][0]).all() and torch.isfinite(s['v_scale'][0]).all()


def test_adamw_zero_blocks_and_fresh_states(ops):
    p = torch.ones(500, device=DEV)
    g = torch.zeros(500, device=DEV)
    g[300] = 1e-3
    (m, ms), (v, vs) = ops.adamw_state8(p), ops.adamw_state8(p)
    plan = ops.adamw_plan([p], [g], [m], [v], m_scale=[ms], v_scale=[vs])
    ops.adamw_step(plan, lr=0.1, rng=ops.new_rng(1, DEV))
    want = torch.ones(500, device=DEV)
    want[300] = 0.9                                                   # first step: lr * sign(g)
    assert torch.allclose(p, want, rtol=0, atol=1e-5)                 # eps / |g| = 1e-5 of lr, fp32 below it
    assert (m.float()[g == 0] == 0).all() and (v.float()[g == 0] == 0).all()


@pytest.mark.parametrize('g_t', [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize('offset', [0, 1])
def test_grad_clip_norm_and_factor(ops, g_t, offset):
    s = make(SIZES, torch.float32, g_t, 13, offset=offset)
    want = math.sqrt(sum(float(x.double().square().sum()) for x in s['g']))
    out = torch.empty(2, device=DEV)
    for top, gscale in ((want / 3, 1.0), (want * 3, 1.0), (want, 0.125)):
        ops.grad_clip(ops.grad_plan(s['g']), top, out, gscale=gscale)
        norm, coef = out.tolist()
        assert abs(norm - gscale * want) <= 2 * 2.0 ** -24 * norm
        assert abs(coef - gscale * min(1.0, top / (gscale * want))) <= 2 * 2.0 ** -24 * coef


def test_grad_clip_extremes(ops):
    out = torch.empty(2, device=DEV)
    t = torch.zeros(1, dtype=torch.int32, device=DEV)
    for value, norm in ((1e30, 1e32), (1e-30, 1e-28), (0.0, 0.0)):
        g = torch.full((10000,), value, device=DEV)
        ops.grad_clip(ops.grad_plan([g]), 1.0, out, t_dev=t)
        assert abs(out[0].item() - norm) <= 1e-6 * norm
        assert abs(out[1].item() - min(1.0, 1 / norm if norm else 1.0)) <= 1e-6 * out[1].item()
    assert t.item() == 3
    for bad in (float('nan'), float('inf'), -float('inf')):
        g = torch.ones(10000, device=DEV)
        g[7777] = bad
        ops.grad_clip(ops.grad_plan([torch.ones(3, device=DEV), g]), 1.0, out, t_dev=t)
        assert out[1].item() == 0.0 and not math.isfinite(out[0].item())
    assert t.item() == 3
    for empty in ([], [torch.empty(0, device=DEV)]):
        ops.grad_clip(ops.grad_plan(empty), 1.0, out)
        assert out.tolist() == [0.0, 1.0]


@pytest.mark.parametrize('eight', [False, True])
def test_a_factor_of_zero_skips_the_step(ops, eight):
    s = make(SIZES, torch.float32, torch.float32, 17, eight=eight)
    before = run_case(ops, s, 0.1, coef=0.0)
    for name in s:
        for x, y in zip(s[name], before[name]):
            assert torch.equal(x.view(torch.uint8) if x.dtype == F8 else x, y.view(torch.uint8) if y.dtype == F8 else y), name


@pytest.mark.parametrize('eight', [False, True])
def test_clip_and_step_replayed_from_a_graph_equal_eager_steps(ops, eight):
    """norm -> factor -> step on a stream of their own, captured once and replayed with other gradients (one of them
    not finite: that step is not taken and not counted), against the same calls issued one by one."""
    sizes = [4099, 64, 128 * 300]
    a = make(sizes, torch.float32, torch.bfloat16, 19, eight=eight)
    b = clone(a)
    grads = [[(1e-3 * randn(gen(100 + i), n)).to(torch.bfloat16) for n in sizes] for i in range(4)]
    grads[2][1][3] = float('inf')
    side = {}
    for s in (a, b):
        s.pop('dither', None)
        d = dict(plan=plan_of(ops, s, wd=0.01), out=torch.empty(2, device=DEV), t=torch.zeros(1, dtype=torch.int32, device=DEV),
                 rng=ops.new_rng(3, DEV))
        side[id(s)] = d

    def step(s):
        d = side[id(s)]
        ops.grad_clip(d['plan'], 0.05, d['out'], t_dev=d['t'])
        ops.adamw_step(d['plan'], lr=1e-2, coef=d['out'][1:], t_dev=d['t'], t_host=0, rng=d['rng'])
        ops.state_advance(d['rng'])

    st = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    keep = clone(a)
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        step(a)
    st.synchronize()
    for name in a:                                                    # undo the warm-up
        for x, y in zip(a[name], keep[name]):
            x.copy_(y)
    side[id(a)]['t'].zero_()
    side[id(a)]['rng'][1] = 0
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        step(a)
    for i in range(4):
        for s in (a, b):
            for x, y in zip(s['g'], grads[i]):
                x.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        step(b)
        torch.cuda.synchronize()
        for name in a:
            for x, y in zip(a[name], b[name]):
                assert torch.equal(x.view(torch.uint8) if x.dtype == F8 else x, y.view(torch.uint8) if y.dtype == F8 else y), (i, name)
    assert side[id(a)]['t'].item() == side[id(b)]['t'].item() == 3


def test_adamw_many_chunks_and_the_norm_of_them(ops):
    """20 million elements in one tensor beside a small one: more chunks than norm blocks, chunks of several passes."""
    n = 20_000_003
    g = (1e-3 * randn(gen(23), n)).to(torch.bfloat16)
    h = (1e-3 * randn(gen(24), 1000)).to(torch.bfloat16)
    ps, ms, vs = ([torch.zeros(k, device=DEV) for k in (1000, n)] for _ in range(3))
    plan = ops.adamw_plan(ps, [h, g], ms, vs)
    out = torch.empty(2, device=DEV)
    ops.grad_clip(plan, 1e9, out)
    want = math.sqrt(float(g.double().square().sum()) + float(h.double().square().sum()))
    assert abs(out[0].item() - want) <= 2 * 2.0 ** -24 * want
    ops.adamw_step(plan, lr=1e-2, b1=0.5, b2=0.5, eps=1e-3)
    for p, m, v, x in zip(ps, ms, vs, (h, g)):
        x = x.double()
        assert ((m.double() - 0.5 * x).abs() <= 2.0 ** -23 * x.abs()).all()
        assert ((p.double() + 1e-2 * x / (x.abs() + 1e-3)).abs() <= 16 * 2.0 ** -24 * 1e-2).all()


@pytest.mark.parametrize('quads', [0.3, 1, 15, 16, 17, 33, 255, 2047, 2048, 2049, 4100])
def test_norm_of_any_number_of_blocks(ops, quads):
    """A block works on 4 x 2048 elements at a time; the one that ends last finishes the call and leaves the plan as it was:
    the same bits time after time, whatever the other plan did in between."""
    n = int(quads * 8192)
    g = torch.randn(n, device=DEV, generator=torch.Generator(device=DEV).manual_seed(n))
    plan, other = ops.grad_plan([g]), ops.grad_plan([g[:n // 2], g[n // 2:]])
    before = plan.table.clone()
    want = g.double().square().sum().sqrt().item()
    outs = []
    for _ in range(4):
        out = torch.full((2,), float('nan'), device=DEV)
        ops.grad_clip(plan, 0.5, out)
        ops.grad_clip(other, 0.5, torch.empty(2, device=DEV))
        outs.append(out)
    # fp64 sums: the result is rounded to fp32 once
    assert abs(outs[0][0].item() - want) <= 2.0 ** -23 * want and abs(outs[0][1].item() * want - 0.5) <= 2.0 ** -23
    assert all(torch.equal(o, outs[0]) for o in outs)
    at = plan.info.part_off
    assert torch.equal(plan.table[:at], before[:at])


def test_small_buffers_are_refused(ops):
    f = lambda n, t=torch.float32: torch.zeros(n, dtype=t, device=DEV)  # noqa: E731
    plan = ops.adamw_plan([f(8)], [f(8)], [f(8)], [f(8)])
    for bad in (dict(coef=f(0)), dict(t_dev=f(0, torch.int32)), dict(rng=f(1, torch.int64))):
        with pytest.raises(ValueError, match='entries'):
            ops.adamw_step(plan, 1e-3, **bad)
    with pytest.raises(ValueError, match='t_dev'):
        ops.grad_clip(plan, 1.0, f(2), t_dev=f(0, torch.int32))


def test_adamw_refusals(ops):
    f = lambda n=256, t=torch.float32: torch.zeros(n, dtype=t, device=DEV)  # noqa: E731
    ok = ops.adamw_plan([f()], [f()], [f()], [f()])
    with pytest.raises(ValueError, match='GPU'):
        ops.adamw_plan([f()], [torch.zeros(256)], [f()], [f()])
    with pytest.raises(TypeError):
        ops.adamw_plan([f(t=torch.float64)], [f()], [f()], [f()])
    with pytest.raises(TypeError):
        ops.adamw_plan([f()], [f()], [f(t=torch.bfloat16)], [f()])
    with pytest.raises(ValueError, match='contiguous'):
        ops.adamw_plan([f(512)[::2]], [f()], [f()], [f()])
    with pytest.raises(ValueError, match='elements'):
        ops.adamw_plan([f(255)], [f()], [f()], [f()])
    with pytest.raises(ValueError, match='tensors for'):
        ops.adamw_plan([f(), f()], [f()], [f()], [f()])
    x = f()
    with pytest.raises(ValueError, match='overlap'):
        ops.adamw_plan([x, x], [f(), f()], [f(), f()], [f(), f()])
    with pytest.raises(ValueError, match='overlap'):
        ops.adamw_plan([x], [x], [f()], [f()])
    shared = f()
    ops.adamw_plan([f(), f()], [shared, shared], [f(), f()], [f(), f()])      # gradients are only read
    with pytest.raises(ValueError, match='m_scale'):
        ops.adamw_plan([f()], [f()], [f(t=torch.uint8).view(F8)], [f(t=torch.uint8).view(F8)], m_scale=[f(2)])
    with pytest.raises(RuntimeError, match='weight decay'):
        ops.adamw_plan([f()], [f()], [f()], [f()], wd=-1.0)
    (m, ms), (v, vs) = ops.adamw_state8(x), ops.adamw_state8(x)
    eight = ops.adamw_plan([x], [f()], [m], [v], m_scale=[ms], v_scale=[vs])
    with pytest.raises(RuntimeError, match='random bits'):
        ops.adamw_step(eight, lr=1e-3)
    for bad in (dict(b1=1.0), dict(b2=-0.1), dict(lr=-1.0), dict(lr=float('nan')), dict(t_host=0), dict(eps=-1.0)):
        with pytest.raises(RuntimeError, match='adamw'):
            ops.adamw_step(ok, **dict(dict(lr=1e-3), **bad))
    with pytest.raises(RuntimeError, match='gradients only'):
        ops.adamw_step(ops.grad_plan([f()]), lr=1e-3)
    for bad in (0.0, -1.0, float('nan')):
        with pytest.raises(RuntimeError, match='grad_clip'):
            ops.grad_clip(ok, bad, f(2))
    with pytest.raises(ValueError):
        ops.grad_clip(ok, 1.0, f(1))
