"""linear_cross_entropy (loss of a Linear layer over a large vocabulary, with its gradients) against the formulas in fp64.

Tolerances, per element, from the roundings on the way (u = 2^-24, e = half a step of the operands' type: bf16 2^-8, fp16
2^-11, fp32 u):
* a logit: D products summed in fp32, D u sum |h||w|;
* lse: the largest logit error of the row, the exponents' and the logarithm's last bits (16 u of their size), and the sum
  of V terms in runs of at most 64 + 8 + V / 1024;
* d = softmax - onehot: twice the logit error relative, 2^-11 for e^(l - max) held in fp16 (half precision only; below
  2^-14 of the slab's largest, 2^-25 absolute), e for d itself;
* dh, dW: those errors weighted with the other operand's sizes, K u for the fp32 sum, e for the result, and half the smallest
  step of fp16 where that is the type."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
U = 2.0 ** -24
E = {torch.float32: U, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 0.0, torch.bfloat16: 0.0, torch.float16: 2.0 ** -25}
TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.fixture(scope='module')
def ops():
    from dp_cgans_amd import ops as o
    return o


def inputs(T, D, V, dtype, seed, ignored=0.1, scale=1.5):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = (torch.randn(V, D, device=DEV, generator=g) * scale / math.sqrt(D)).to(dtype)
    target = torch.randint(0, V, (T,), device=DEV, generator=g)
    lift = 12 * torch.rand(T, 1, device=DEV, generator=g)
    h = (torch.randn(T, D, device=DEV, generator=g) + lift / scale ** 2 * w[target].float()).to(dtype)
    target[torch.rand(T, device=DEV, generator=g) < ignored] = -100
    return h, w, target


class Oracle(object):
    """Values and error bounds in fp64."""

    def __init__(self, h, w, target, gscale=1.0, mean=True, ignore=-100):
        T, D = h.shape
        V, dt = w.shape[0], h.dtype
        live = target != ignore
        h64, w64 = torch.where(live[:, None], h.double(), 0.0), w.double()
        l = h.double() @ w64.t()
        el = D * U * (h.double().abs() @ w64.abs().t()).amax(1)
        self.lse = torch.logsumexp(l, 1)
        at = torch.where(live, target, 0)
        self.loss = torch.where(live, self.lse - l.gather(1, at[:, None])[:, 0], 0.0)
        n = max(1, int(live.sum())) if mean else 1
        self.total = self.loss.sum() / n
        self.el = 2 * el + 16 * U * (self.lse.abs() + l.abs().amax(1)) + (72 + 8 + V / 1024) * U
        p = torch.exp(l - self.lse[:, None])
        d = p.clone()
        d.scatter_(1, at[:, None], torch.expm1(-self.loss)[:, None])
        d[~live] = 0
        a = gscale / n
        self.dh, self.dw = a * (d @ w64), a * (d.t() @ h64)
        rel = E[dt] + 2 * torch.where(live, self.el, 0.0)[:, None] + (2.0 ** -11 if dt != torch.float32 else 8 * U)
        # the target's p_t - 1 follows the loss: its error is the loss's, absolute
        ed = d.abs() * rel + (2.0 ** -25 if dt != torch.float32 else 0.0) * live[:, None]
        ed.scatter_add_(1, at[:, None], torch.where(live, 2 * self.el, 0.0)[:, None])
        self.edh = a * (ed + V * U * d.abs()) @ w64.abs()
        self.edw = a * (ed + T * U * d.abs()).t() @ h64.abs()
        self.edh += E[dt] * (self.dh.abs() + self.edh) + TINY[dt]
        self.edw32 = self.edw + 4 * U * self.dw.abs()
        self.edw = self.edw + E[dt] * (self.dw.abs() + self.edw) + TINY[dt]
        self.etotal = (self.el * live).sum() / n + 2 * U * self.total.abs()


def within(got, want, bound, what):
    bad = ~((got.double() - want).abs() <= bound)
    assert not bad.any(), '%s: %d of %d off, worst %.3g of its bound' % (
        what, int(bad.sum()), bad.numel(), float(((got.double() - want).abs() / bound.clamp(min=1e-300)).max()))


def call(ops, h, w, target, grads=True, dw=None, dh=None, piece_rows=0, **kw):
    T, D = h.shape
    V = w.shape[0]
    f = lambda *s, t=torch.float32: torch.full(s, float('nan'), dtype=t, device=DEV)  # noqa: E731
    o = dict(loss=f(T), lse=f(T), total=f(1))
    if grads:
        o['dh'] = f(T, D, t=h.dtype) if dh is None else dh
        o['dw'] = f(V, D, t=w.dtype) if dw is None else dw
    n = ops.linear_cross_entropy_ws(T, D, V, h.dtype, grads, grads and o['dw'].dtype == torch.float32, piece_rows)
    ws = torch.full((n,), 0xff, dtype=torch.uint8, device=DEV)                    # (NaN in every type)
    ops.linear_cross_entropy(h, w, target, o['loss'], ws, dh=o.get('dh'), dw=o.get('dw'), lse=o['lse'], total=o['total'],
                             piece_rows=piece_rows, **kw)
    return o


SHAPES = [(1, 8, 1), (1, 64, 300), (3, 72, 129), (257, 128, 1000), (300, 200, 2049), (700, 264, 511), (513, 1024, 777),
          (31, 2048, 257), (256, 64, 256), (1000, 136, 130), (40, 512, 9001),
          (64, 128, 700), (65, 128, 700), (128, 64, 25000), (3500, 72, 3500), (2, 1024, 30011)]


def check(o, ref, grads=True):
    within(o['loss'], ref.loss, ref.el, 'loss')
    within(o['lse'], ref.lse, ref.el, 'lse')
    within(o['total'][0], ref.total, ref.etotal, 'total')
    if grads:
        within(o['dh'], ref.dh, ref.edh, 'dh')
        within(o['dw'], ref.dw, ref.edw32 if o['dw'].dtype == torch.float32 else ref.edw, 'dw')


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('T,D,V', SHAPES)
def test_loss_and_gradients(ops, T, D, V, dtype):
    h, w, target = inputs(T, D, V, dtype, T + D + V)
    o = call(ops, h, w, target)
    check(o, Oracle(h, w, target))
    only = call(ops, h, w, target, grads=False)
    for k in ('loss', 'lse', 'total'):
        assert torch.equal(only[k], o[k]), k


@pytest.mark.parametrize('D,V', [(1, 1), (3, 50), (63, 1001), (257, 129)])
def test_fp32_takes_any_width(ops, D, V):
    h, w, target = inputs(77, D, V, torch.float32, D)
    check(call(ops, h, w, target), Oracle(h, w, target))


@pytest.mark.parametrize('T', [1, 4, 5, 16, 17])
@pytest.mark.parametrize('D,V', [(1, 1), (4, 31), (3, 33), (64, 700), (100, 129), (257, 5000), (260, 64), (1000, 4097), (1024, 20000)])
def test_few_rows_in_fp32(ops, T, D, V):
    """Up to 16 rows, in whole 16 bytes or not; in rows that start anywhere; in pieces of 16; dW added to what is there."""
    h, w, target = inputs(T, D, V, torch.float32, T + D + V)
    ref = Oracle(h, w, target)
    check(call(ops, h, w, target), ref)
    apart = lambda x: torch.full((x.shape[0], D + 3), 7.0, device=DEV)[:, 1:1 + D].copy_(x)  # noqa: E731
    check(call(ops, apart(h), apart(w), target, dh=apart(h), dw=apart(w)), ref)
    big = torch.cat([h] * 3 + [h[:1]]), torch.cat([target] * 3 + [target[:1]])
    more = Oracle(big[0], w, big[1])
    dw = torch.randn(V, D, device=DEV, generator=torch.Generator(device=DEV).manual_seed(1))
    more.dw = more.dw + dw.double()
    more.edw32 = more.edw32 + 8 * U * (more.dw.abs() + dw.double().abs())          # (each of at most four pieces adds with one rounding)
    check(call(ops, big[0], w, big[1], dw=dw, accumulate=True, piece_rows=16), more)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('T', [1, 5, 16, 17])
@pytest.mark.parametrize('D,V', [(8, 1), (8, 63), (40, 65), (256, 129), (264, 5000), (1032, 700)])
def test_few_rows_in_half_precision(ops, T, D, V, dtype):
    """Up to 16 rows, also as pieces of a longer call."""
    h, w, target = inputs(T, D, V, dtype, T + D + V)
    ref = Oracle(h, w, target)
    o = call(ops, h, w, target)
    check(o, ref)
    alone = call(ops, h, w, target, grads=False)
    assert torch.equal(alone['loss'], o['loss']) and torch.equal(alone['lse'], o['lse']) and torch.equal(alone['total'], o['total'])
    big = torch.cat([h] * 2 + [h[:1]]), torch.cat([target] * 2 + [target[:1]])
    check(call(ops, big[0], w, big[1], piece_rows=16), Oracle(big[0], w, big[1]))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('T,D,V', [(1, 64, 233), (2, 64, 233), (5, 1032, 5000), (16, 256, 18000)])
def test_gradients_of_few_rows_are_rounded_once(ops, T, D, V, dtype):
    """d is within 2^-11 (its first form in fp16) and e^2 (two numbers of the type) here: what is left is the result's rounding e."""
    for seed in range(8):
        h, w, target = inputs(T, D, V, dtype, seed, ignored=0.0)
        ref = Oracle(h, w, target)
        o = call(ops, h, w, target)
        p = torch.softmax(h.double() @ w.double().t(), 1)
        d = p.clone()
        d.scatter_(1, target[:, None], torch.expm1(-ref.loss)[:, None])
        e = E[dtype]
        ed = d.abs() * (2.0 ** -11 + e * e + 2 * ref.el[:, None]) + 2.0 ** -25
        ed.scatter_add_(1, target[:, None], 2 * ref.el[:, None])
        for name, want, other, terms in (('dh', ref.dh, lambda x: x @ w.double().abs(), V), ('dw', ref.dw, lambda x: x.t() @ h.double().abs(), T)):
            err = other(ed + 2 * terms * U * d.abs()) / T
            within(o[name], want, err + e * (want.abs() + err) + TINY[dtype], name)


@pytest.mark.parametrize('dtype', TYPES)
def test_strided_rows_and_what_lies_between_them(ops, dtype):
    """Rows inside wider buffers; everything outside the outputs' own columns keeps its bits."""
    h0, w0, target = inputs(130, 72, 300, dtype, 1)
    wide = lambda x, t=None: torch.full((x.shape[0] + 2, x.shape[1] + 24), float('nan'), dtype=t or x.dtype, device=DEV)  # noqa: E731
    hb, wb, dhb, dwb = wide(h0), wide(w0), wide(h0), wide(w0)
    cut = lambda b: b[1:-1, 8:8 + 72]  # noqa: E731
    cut(hb).copy_(h0)
    cut(wb).copy_(w0)
    o = call(ops, cut(hb), cut(wb), target, dh=cut(dhb), dw=cut(dwb))
    check(o, Oracle(h0, w0, target))
    for b in (dhb, dwb):
        edge = torch.ones_like(b, dtype=torch.bool)
        edge[1:-1, 8:80] = False
        assert torch.isnan(b[edge]).all() and not torch.isnan(b[~edge]).any()


@pytest.mark.parametrize('dtype', TYPES)
def test_ignored_rows_hold_anything(ops, dtype):
    """NaN, infinities and the type's extremes in rows that are ignored reach neither gradient."""
    h, w, target = inputs(300, 128, 500, dtype, 2, ignored=0.0)
    target[::7] = -100
    clean = call(ops, h, w, target)
    h2 = h.clone()
    for k, x in enumerate((float('nan'), float('inf'), -float('inf'), torch.finfo(dtype).max, torch.finfo(dtype).min)):
        h2[7 * k::35] = x
    o = call(ops, h2, w, target)
    live = target != -100
    for k in ('loss', 'total', 'dh', 'dw'):
        assert torch.equal(o[k], clean[k]), k
    assert torch.equal(o['lse'][live], clean['lse'][live])
    assert (o['dh'][~live] == 0).all()
    check(clean, Oracle(h, w, target))


@pytest.mark.parametrize('dtype', TYPES)
def test_all_rows_ignored(ops, dtype):
    h, w, target = inputs(70, 64, 200, dtype, 3)
    target[:] = 5
    o = call(ops, h, w, target, ignore_index=5)
    for k in ('loss', 'total', 'dh', 'dw'):
        assert (o[k] == 0).all(), k
    assert torch.isfinite(o['lse']).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_no_rows(ops, dtype):
    h, w = torch.empty(0, 64, dtype=dtype, device=DEV), torch.ones(30, 64, dtype=dtype, device=DEV)
    o = call(ops, h, w, torch.empty(0, dtype=torch.int64, device=DEV))
    assert (o['dw'] == 0).all() and o['total'].item() == 0.0
    keep = torch.ones(30, 64, device=DEV)
    call(ops, h, w, torch.empty(0, dtype=torch.int64, device=DEV), dw=keep, accumulate=True)
    assert (keep == 1).all()


@pytest.mark.parametrize('dtype', TYPES)
def test_targets_outside_the_vocabulary(ops, dtype):
    h, w, target = inputs(100, 64, 300, dtype, 4, ignored=0.0)
    bad = torch.zeros(100, dtype=torch.bool, device=DEV)
    for r, t in ((3, 300), (50, -1), (97, 2 ** 40), (98, -2 ** 40), (99, 511), (10, 2 ** 32 + 5)):
        target[r] = t
        bad[r] = True
    o = call(ops, h, w, target, mean=False)
    assert torch.equal(torch.isnan(o['loss']), bad) and torch.isnan(o['total']).all()
    assert (o['dh'][bad] == 0).all()
    ref = Oracle(h, w, torch.where(bad, -100, target), mean=False)
    within(o['dh'], ref.dh, ref.edh, 'dh')
    within(o['dw'], ref.dw, ref.edw, 'dw')


@pytest.mark.parametrize('dtype', TYPES)
def test_logits_far_apart(ops, dtype):
    """Logits of hundreds, of either sign: sure rows, hopeless rows, and slabs that vanish beside another."""
    h, w, target = inputs(200, 64, 700, dtype, 5, scale=1.0)
    h = (h.float() * torch.linspace(-150, 150, 200, device=DEV)[:, None]).to(dtype)
    check(call(ops, h, w, target), Oracle(h, w, target))


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
@pytest.mark.parametrize('offset', [-400, 400])
def test_entries_whose_logits_are_all_minus_infinity(ops, dtype, offset):
    """256 entries (whole slabs) whose logits overflow to -inf take no part, however far from 0 the others lie."""
    T, D, V = 150, 64, 700
    h, w, target = inputs(T, D, V, dtype, 6, scale=0.5)
    h[:, 0], w[:, 0] = 4, offset / 4
    off = torch.zeros(256, D, dtype=dtype, device=DEV)
    off[:, 0] = -2.0 ** 127
    ref = Oracle(h, w, target)
    o = call(ops, h, torch.cat([off, w]), torch.where(target < 0, target, target + 256))
    assert (o['dw'][:256] == 0).all()
    o['dw'] = o['dw'][256:]
    check(o, ref)


@pytest.mark.parametrize('dtype', TYPES)
def test_a_nan_row_stays_a_row(ops, dtype):
    h, w, target = inputs(100, 64, 300, dtype, 6, ignored=0.0)
    h[41, 3] = float('nan')
    o = call(ops, h, w, target)
    rows = torch.arange(100, device=DEV) == 41
    assert torch.equal(torch.isnan(o['loss']), rows)
    assert torch.equal(torch.isnan(o['dh']).any(1), rows)
    assert torch.isnan(o['dw']).all()


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('mean,gscale', [(True, 3.0), (False, 0.01)])
def test_scale_and_sum(ops, dtype, mean, gscale):
    h, w, target = inputs(300, 96, 400, dtype, 7)
    check(call(ops, h, w, target, mean=mean, gscale=gscale), Oracle(h, w, target, gscale=gscale, mean=mean))


@pytest.mark.parametrize('dtype', TYPES)
def test_pieces_of_rows(ops, dtype):
    h, w, target = inputs(1100, 136, 700, dtype, 8)
    whole = call(ops, h, w, target, piece_rows=2048)
    for rows in (256, 300, 1024):
        o = call(ops, h, w, target, piece_rows=rows)
        check(o, Oracle(h, w, target))
        for k in ('loss', 'lse', 'total'):
            assert torch.equal(o[k], whole[k]), (rows, k)


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('rows', [0, 256])
def test_fp32_weight_gradient_accumulates(ops, dtype, rows):
    h, w, target = inputs(600, 72, 500, dtype, 9)
    ref = Oracle(h, w, target)
    dw = torch.full((500, 72), float('nan'), device=DEV)
    o = call(ops, h, w, target, dw=dw, piece_rows=rows)
    within(dw, ref.dw, ref.edw32, 'dw')
    base = torch.randn(500, 72, device=DEV)
    dw.copy_(base)
    o = call(ops, h, w, target, dw=dw, accumulate=True, piece_rows=rows)
    within(dw, ref.dw + base.double(), ref.edw32 + 8 * U * (base.double().abs() + ref.dw.abs()), 'accumulated dw')
    check(dict(o, dw=None), ref, grads=False)


@pytest.mark.parametrize('dtype', TYPES)
def test_one_gradient_alone(ops, dtype):
    h, w, target = inputs(300, 128, 600, dtype, 10)
    both = call(ops, h, w, target)
    loss = torch.empty(300, device=DEV)
    ws = torch.empty(ops.linear_cross_entropy_ws(300, 128, 600, dtype), dtype=torch.uint8, device=DEV)
    dh, dw = torch.empty_like(h), torch.empty_like(w)
    ops.linear_cross_entropy(h, w, target, loss, ws, dh=dh)
    ops.linear_cross_entropy(h, w, target, loss, ws, dw=dw)
    assert torch.equal(dh, both['dh']) and torch.equal(dw, both['dw'])


@pytest.mark.parametrize('dtype', TYPES)
def test_gradients_against_differences(ops, dtype):
    """total along a direction of h and of w: (total(x + t) - total(x - t)) / 2 from the operator's own losses in fp32
    against the gradients' inner product; second differences bound the truncation, the losses' bounds the rounding."""
    h, w, target = (x.float() if x.is_floating_point() else x for x in inputs(60, 64, 200, torch.float32, 11))
    h, w = h.to(dtype).float(), w.to(dtype).float()
    o = call(ops, h.to(dtype), w.to(dtype), target)
    ref = Oracle(h, w, target)
    g = torch.Generator(device=DEV).manual_seed(12)
    t = 2.0 ** -7
    for x, grad, bound in ((h, o['dh'], ref.edh if dtype == torch.float32 else Oracle(h.to(dtype), w.to(dtype), target).edh),
                           (w, o['dw'], ref.edw if dtype == torch.float32 else Oracle(h.to(dtype), w.to(dtype), target).edw)):
        v = torch.randn(x.shape, device=DEV, generator=g) / 8
        f = lambda s: call(ops, h + s * t * v if x is h else h, w + s * t * v if x is w else w, target, grads=False)['total'].double()  # noqa: E731
        lo, mid, hi = f(-1), f(0), f(1)
        slope = (grad.double() * v.double()).sum()
        curve = (hi + lo - 2 * mid).abs() / t                     # |f''| t; the odd remainder is a further t smaller
        noise = 4 * ref.etotal / t + (bound * v.double().abs()).sum()
        assert ((hi - lo) / (2 * t) - slope).abs() <= curve + noise


@pytest.mark.parametrize('dtype', TYPES)
def test_captured_and_replayed_on_another_stream(ops, dtype):
    """A training call captured on a side stream and replayed with other contents, eager calls in between; two graphs
    with workspaces of their own; the same call twice gives the same bits."""
    T, D, V = 300, 128, 900
    st = torch.cuda.Stream()
    sets = []
    for k in range(2):
        h, w, target = inputs(T, D, V, dtype, 20 + k)
        o = dict(loss=torch.empty(T, device=DEV), dh=torch.empty_like(h), dw=torch.empty_like(w), total=torch.empty(1, device=DEV))
        ws = torch.empty(ops.linear_cross_entropy_ws(T, D, V, dtype), dtype=torch.uint8, device=DEV)
        sets.append((h, w, target, o, ws))
    run = lambda h, w, target, o, ws: ops.linear_cross_entropy(h, w, target, o['loss'], ws, dh=o['dh'], dw=o['dw'], total=o['total'])  # noqa: E731
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        for s in sets:
            run(*s)
    st.synchronize()
    graphs = []
    for s in sets:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=st):
            run(*s)
    for i in range(3):
        for k, s in enumerate(sets):
            h, w, target = inputs(T, D, V, dtype, 30 + 2 * i + k)
            for x, y in zip(s[:3], (h, w, target)):
                x.copy_(y)
        torch.cuda.synchronize()
        for gr in graphs:
            gr.replay()
        torch.cuda.synchronize()
        for s in sets:
            e = call(ops, *s[:3])
            for k in s[3]:
                assert torch.equal(s[3][k], e[k]), (i, k)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_wide_rows_that_start_inside_a_line(ops, dtype):
    """2^36 multiplications and more on rows of 2000 bytes: the same bits as on rows of 2048, whatever lies between those."""
    T, D, V = 2048, 1000, 34000
    h, w, target = inputs(T, D, V, dtype, 9)
    apart = torch.full((T, 1024), float('nan'), dtype=dtype, device=DEV)
    apart[:, :D] = h
    a, b = call(ops, h, w, target), call(ops, apart[:, :D], w, target)
    check(a, Oracle(h, w, target))
    assert all(torch.equal(a[k], b[k]) for k in a)


def test_a_vocabulary_of_many_tiles(ops):
    """Rows of several tiles, tails in every direction, against fp64 on samples of the gradients."""
    T, D, V = 1300, 320, 40009
    h, w, target = inputs(T, D, V, torch.bfloat16, 13)
    check(call(ops, h, w, target), Oracle(h, w, target))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('ignore', [0, 3, 2 ** 32 + 3])
def test_an_ignored_class_and_odd_pieces(ops, dtype, ignore):
    """ignore_index may be a class, or share its low half with one; pieces need not be whole tiles."""
    T, D, V = 330, 64, 40
    h, w, target = inputs(T, D, V, dtype, 31, ignored=0.0)
    target[::7] = ignore
    ref = Oracle(h, w, target, ignore=ignore)
    for rows in (0, 100, 33, 16):
        check(call(ops, h, w, target, ignore_index=ignore, piece_rows=rows), ref)


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float32])
def test_millions_of_rows(ops, dtype):
    """More rows than a piece holds, few classes."""
    T, D, V = (1 << 21) + 300, 8, 40
    h, w, target = inputs(T, D, V, dtype, 21)
    check(call(ops, h, w, target), Oracle(h, w, target))
    check(call(ops, h, w, target, grads=False), Oracle(h, w, target), grads=False)


def test_a_vocabulary_of_millions(ops):
    """More slabs than a grid's second dimension holds; three rows."""
    T, D, V = 3, 8, 4200011
    h, w, target = inputs(T, D, V, torch.bfloat16, 14, ignored=0.0)
    target[1] = V - 1
    check(call(ops, h, w, target), Oracle(h, w, target))
    check(call(ops, h.float(), w.float(), target), Oracle(h.float(), w.float(), target))


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('offset', [0, 200])
def test_sure_rows_keep_a_small_loss(ops, dtype, offset):
    """Rows whose target leads by 13 to 21: the small loss comes from the sum and not from the difference of two numbers of
    the logits' size.  The logits are exact here.  The sum is 1 and little beside it: a rounding of at most u each for
    the leading term's exponential (its hardware's last bit: 2), up to 8 additions in a thread's run, 2 that join four
    runs, 2 across the lanes of a row or 8 across a block, 6 that join the slabs with 2 factors each, the logarithm and
    the last product (4): 40 u in all.  The others' exponents are off by at most 2 * 32 u of their own: u of the loss
    times 64.  (The difference of two logarithms near 221 is off by up to 221 u, which the second offset would show.)"""
    T, D, V = 64, 64, 1000
    g = torch.Generator(device=DEV).manual_seed(15)
    w = torch.zeros(V, D, device=DEV)
    w[:D] = 4 * torch.eye(D, device=DEV)                     # logits 4 h, exact in every type
    target = torch.arange(T, device=DEV)
    h = torch.zeros(T, D, device=DEV)
    lead = torch.linspace(13, 21, T, device=DEV).round(decimals=0)
    h[target, target] = lead / 4
    if offset:
        h, w = torch.cat([h, torch.zeros(T, 8, device=DEV)], 1), torch.cat([w, torch.zeros(V, 8, device=DEV)], 1)
        h[:, D], w[:, D] = offset, 1
    h, w = h.to(dtype), w.to(dtype)
    o = call(ops, h, w, target)
    l = h.double() @ w.double().t()
    loss = torch.logsumexp(l, 1) - l[target, target]
    assert float(loss.min()) < 1e-5 * 1000
    assert ((o['loss'].double() - loss).abs() <= 40 * U + 64 * U * loss).all()
    d = torch.softmax(l, 1)
    pm1 = torch.expm1(-loss) / T
    got = o['dw'][target].double() if dtype == torch.float32 else None
    if got is not None:                                       # dW's row t, column t: (p_t - 1) h, and the other rows' share
        want = (d.t() @ h.double() / T)[:T]
        want += (pm1 - d[target, target] / T)[:, None] * h.double()
        # (the loss's own error in p_t - 1, and the softmax's)
        assert ((got - want).abs() <= (40 * U + 64 * U * loss)[:, None] * h.double().abs() / T + 128 * U * (d.t() @ h.double().abs() / T)[:T]).all()


def test_refusals(ops):
    z = lambda *s, t=torch.bfloat16: torch.zeros(*s, dtype=t, device=DEV)  # noqa: E731
    T, D, V = 16, 64, 100
    good = dict(h=z(T, D), w=z(V, D), target=z(T, t=torch.int64), loss=z(T, t=torch.float32), dh=z(T, D), dw=z(V, D))
    ws = z(ops.linear_cross_entropy_ws(T, D, V, torch.bfloat16), t=torch.uint8)

    def run(exc, match, ws=ws, **kw):
        a = dict(good, **kw)
        with pytest.raises(exc, match=match):
            ops.linear_cross_entropy(a.pop('h'), a.pop('w'), a.pop('target'), a.pop('loss'), ws, **a)

    run(RuntimeError, 'workspace', ws=ws[:-256])
    run(RuntimeError, '256', ws=z(ws.numel() + 256, t=torch.uint8)[16:])
    run(ValueError, 'must be', w=z(V, 72))
    run(TypeError, 'fp32, bf16', h=z(T, D, t=torch.float64))
    run(TypeError, 'w must be', w=z(V, D, t=torch.float16))
    run(TypeError, 'target', target=z(T, t=torch.int32))
    run(ValueError, 'target', target=z(T + 1, t=torch.int64))
    run(ValueError, 'loss', loss=z(2 * T, t=torch.float32)[::2])
    run(ValueError, 'dh', dh=z(T + 1, D))
    run(TypeError, 'dw', dw=z(V, D, t=torch.float16))
    run(ValueError, 'strides', h=z(D, T).t())
    run(RuntimeError, 'accumulation', accumulate=True)
    run(RuntimeError, 'aligned', h=z(T, D + 8)[:, 4:4 + D])
    run(RuntimeError, 'aligned', h=z(T, D + 4)[:, :D])
    run(RuntimeError, 'aligned', dh=z(T, D + 4)[:, :D])
    with pytest.raises(RuntimeError, match='multiple of 8'):
        ops.linear_cross_entropy_ws(T, 60, V, torch.bfloat16)
    run(RuntimeError, 'multiple of 8', h=z(T, 60), w=z(V, 60), dh=z(T, 60), dw=z(V, 60))
    with pytest.raises(TypeError):
        ops.linear_cross_entropy_ws(T, D, V, torch.float64)
    run(ValueError, 'GPU', h=torch.zeros(T, D, dtype=torch.bfloat16))
