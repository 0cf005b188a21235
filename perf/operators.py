"""Cases over which the operators of a categorical head's training tail are timed and compared:

* ``lce``    linear cross entropy: logits = h w^T over a large vocabulary, the loss of every row and, for training,
             the gradients of h and w - the logits never reach memory as a whole;
* ``clip``   the global norm of the gradients of many tensors and the factor that clips it;
* ``adamw``  a decoupled-weight-decay Adam step over many tensors, with states in 32 or in 8 bits.

``own`` false: the plain form, elementary torch operations in 32 bits (64 for long sums and next to the borders of the
8-bit grid).  ``own`` true: the calls of ``dp_cgans_amd.ops`` a training program makes.
"""
import math

import torch

own = False

TYPES = {'f32': torch.float32, 'bf16': torch.bfloat16, 'f16': torch.float16}
IGNORE = -100
BLOCK = 128                      # elements that share one scale of an 8-bit state
LR, WD, B1, B2, EPS, T_STEP = 2e-5, 0.1, 0.9, 0.999, 1e-8, 100
MAX_NORM = 1.0


def _dev():
    return torch.device('cuda:0' if torch.cuda.is_available() else 'cpu')


def listed():
    return [
        # scoring a handful of rows against all category values of the wide synthetic table: latency
        dict(name='lce_score_few', op='lce', T=4, D=256, V=18000, dtype='bf16', grads=False),
        # evaluation pass over a validation batch with a subword-sized vocabulary
        dict(name='lce_eval', op='lce', T=4096, D=2048, V=131072, dtype='bf16', grads=False),
        # training batch at the wide table's 18 000 category values, width of the wide networks
        dict(name='lce_train_columns', op='lce', T=8192, D=1024, V=18000, dtype='bf16', grads=True),
        # the same with a subword-sized vocabulary: the largest product
        dict(name='lce_train_large', op='lce', T=8192, D=2048, V=131072, dtype='bf16', grads=True),
        # last, ragged batch of an epoch; no size a multiple of a tile
        dict(name='lce_train_ragged', op='lce', T=1531, D=1160, V=50021, dtype='f16', grads=True),
        # the networks' own type at the default batch and width
        dict(name='lce_train_f32', op='lce', T=500, D=256, V=18000, dtype='f32', grads=True),
        # gradients of a network of the default width: a few thousand to a hundred thousand elements per tensor
        dict(name='clip_small', op='clip', width=256, layers=2, vocab=276, g='f32'),
        # gradients of a model of 0.4 billion parameters, half precision
        dict(name='clip_large', op='clip', width=2048, layers=6, vocab=50021, g='bf16'),
        # the default networks, all in 32 bits
        dict(name='adamw_small', op='adamw', width=256, layers=2, vocab=276, p='f32', g='f32', state=32, copy=False),
        # 0.4 billion parameters with 32-bit master weights, half-precision gradients and working copy
        dict(name='adamw_large', op='adamw', width=2048, layers=6, vocab=50021, p='f32', g='bf16', state=32, copy=True),
        # half-precision parameters, 8-bit states, odd widths
        dict(name='adamw8_odd', op='adamw', width=999, layers=4, vocab=18000, p='bf16', g='bf16', state=8, copy=False),
        # 32-bit parameters with 8-bit states at the largest size
        dict(name='adamw8_large', op='adamw', width=2048, layers=6, vocab=50021, p='f32', g='f32', state=8, copy=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(['lce', 'lce', 'clip', 'adamw', 'adamw'])
    if op == 'lce':
        dtype = rng.choice(['bf16', 'bf16', 'f16', 'f32'])
        while True:
            T, D, V = _log(rng, 1, 8192), 8 * _log(rng, 8, 512), _log(rng, 200, 131072)
            if T * D * V <= (2.2e12 if dtype != 'f32' else 2e11) and T * V <= 8192 * 131072:
                return dict(op=op, T=T, D=D, V=V, dtype=dtype, grads=rng.random() < 0.7)
    width, layers, vocab = _log(rng, 64, 2048), rng.randint(1, 6), _log(rng, 200, 50021)
    if op == 'clip':
        return dict(op=op, width=width, layers=layers, vocab=vocab, g=rng.choice(['f32', 'bf16', 'f16']))
    return dict(op=op, width=width, layers=layers, vocab=vocab, p=rng.choice(['f32', 'f32', 'bf16']),
                g=rng.choice(['f32', 'bf16']), state=rng.choice([32, 8]), copy=rng.random() < 0.5)


def _shapes(case):
    """Parameter tensors of a network of ``layers`` blocks: an embedding / head matrix, per block two vectors, four
    square matrices, two wide ones and their biases."""
    w = case['width']
    block = [(w,), (w, w), (w, w), (w, w), (w, w), (w,), (4 * w, w), (4 * w,), (w, 4 * w), (w,)]
    return [(case['vocab'], w)] + block * case['layers'] + [(w,)]


def _layout(case):
    """[(offset, shape)] of the tensors in one flat buffer, each on a multiple of BLOCK, and the buffer's length."""
    at, out = 0, []
    for s in _shapes(case):
        out.append((at, s))
        at += -(-math.prod(s) // BLOCK) * BLOCK
    return out, at


def _views(flat, layout):
    return [flat[o:o + math.prod(s)].view(s) for o, s in layout]


def _live(layout, total, dev):
    """1 inside the tensors, 0 in the gaps between them."""
    n = [math.prod(s) for _, s in layout]
    ends = [o for o, _ in layout[1:]] + [total]
    runs = torch.tensor([r for (o, _), k, e in zip(layout, n, ends) for r in (k, e - o - k)], device=dev)
    ones = torch.tensor([1.0, 0.0] * len(n), device=dev)
    return torch.repeat_interleave(ones, runs, output_size=total)


def _per_block(per_tensor, layout, total, dev):
    ends = [o for o, _ in layout[1:]] + [total]
    runs = torch.tensor([(e - o) // BLOCK for (o, _), e in zip(layout, ends)], device=dev)
    return torch.repeat_interleave(torch.tensor(per_tensor, device=dev), runs, output_size=total // BLOCK)


def _hold8(x, u):
    """x [blocks, BLOCK] in 8 bits (4 exponent, 3 mantissa bits) times one scale per block, which puts the block's
    largest value on 448, rounded up where the fraction plus u reaches 1: (signed codes, scales)."""
    scale = x.abs().amax(1).clamp(min=2.0 ** -100) / 448
    y = (x.abs() / scale[:, None]).clamp(max=448)
    step = torch.ldexp(torch.ones_like(y), (torch.frexp(y)[1] - 4).clamp(min=-9))
    return torch.sign(x) * torch.floor(y / step + u) * step, scale


def prepare(case, seed):
    dev = _dev()
    g = torch.Generator(device=dev).manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, device=dev, generator=g)  # noqa: E731
    if case['op'] == 'lce':
        T, D, V, dt = case['T'], case['D'], case['V'], TYPES[case['dtype']]
        w = (randn(V, D) * (1.5 / math.sqrt(D))).to(dt)
        # category values and subwords come Zipf-distributed; a few rows are padding
        target = (torch.exp(torch.rand(T, device=dev, generator=g) * math.log(V)) - 1).long().clamp(0, V - 1)
        lift = 16 * torch.rand(T, 1, device=dev, generator=g)          # from unsure rows to confident ones
        h = (randn(T, D) + lift / 2.25 * w[target].float()).to(dt)
        target = torch.where(torch.rand(T, device=dev, generator=g) < 0.03, IGNORE, target)
        s = dict(case=case, h=h, w=w, target=target)
        if own:
            from dp_cgans_amd import ops
            s['loss'], s['lse'] = torch.empty(T, device=dev), torch.empty(T, device=dev)
            s['total'] = torch.empty(1, device=dev)
            s['dh'], s['dw'] = (torch.empty_like(h), torch.empty_like(w)) if case['grads'] else (None, None)
            s['ws'] = torch.empty(ops.linear_cross_entropy_ws(T, D, V, dt, grads=case['grads']), dtype=torch.uint8, device=dev)
        return s
    layout, total = _layout(case)
    live = _live(layout, total, dev)
    big = _per_block([10.0 ** (-3 - i % 3) for i in range(len(layout))], layout, total, dev).repeat_interleave(BLOCK)
    s = dict(case=case, layout=layout, g=(randn(total) * big * live).to(TYPES[case['g']]))
    if case['op'] == 'clip':
        if own:
            from dp_cgans_amd import ops
            s['plan'] = ops.grad_plan(_views(s['g'], layout))
            s['out'] = torch.empty(2, device=dev)
        return s
    s['p'] = (0.02 * randn(total) * live).to(TYPES[case['p']])
    s['wd'] = [WD if len(sh) == 2 else 0.0 for _, sh in layout]
    s['coef'] = 0.5 + 0.5 * torch.rand(1, device=dev, generator=g)
    s['copy'] = torch.zeros(total, dtype=torch.bfloat16, device=dev) if case['copy'] else None
    s['t'] = T_STEP
    m = 0.3 * randn(total) * big * live
    r = big * live * (0.5 + torch.rand(total, device=dev, generator=g))
    if case['state'] == 32:
        s['m'], s['v'] = m, r * r
    else:
        for k, x in (('m', m), ('r', r)):
            q, scale = _hold8(x.view(-1, BLOCK), 0.5)
            s[k], s[k + '_scale'] = q.view(-1).to(torch.float8_e4m3fn), scale
        s['dither'] = torch.randint(-32768, 32768, (total,), device=dev, generator=g, dtype=torch.int16)
    if own:
        from dp_cgans_amd import ops
        v = lambda k: _views(s[k], layout)  # noqa: E731
        more = {}
        if case['state'] == 8:
            cut = lambda k: [s[k][o // BLOCK:o // BLOCK + -(-math.prod(sh) // BLOCK)] for o, sh in layout]  # noqa: E731
            more = dict(m_scale=cut('m_scale'), v_scale=cut('r_scale'), dither=v('dither'))
        s['plan'] = ops.adamw_plan(v('p'), v('g'), v('m'), v('v' if case['state'] == 32 else 'r'), wd=s['wd'],
                                   copies=v('copy') if case['copy'] else None, **more)
    return s


def _lce_own(s):
    from dp_cgans_amd import ops
    ops.linear_cross_entropy(s['h'], s['w'], s['target'], s['loss'], s['ws'], dh=s['dh'], dw=s['dw'], lse=s['lse'],
                             total=s['total'], ignore_index=IGNORE)
    return {k: s[k] for k in ('loss', 'lse', 'total', 'dh', 'dw')}


def _lce(s):
    h, w, target, dt = s['h'].float(), s['w'].float(), s['target'], s['h'].dtype
    valid = target != IGNORE
    at = torch.where(valid, target, 0)[:, None]
    logits = h @ w.t()
    top = logits.amax(1, keepdim=True)
    lt = logits.gather(1, at)
    p = torch.exp(logits - top)
    del logits
    total = p.sum(1, keepdim=True)
    lse = top + torch.log(total)
    loss = torch.where(valid, (lse - lt)[:, 0], 0.0)
    count = valid.sum().clamp(min=1)
    out = dict(loss=loss, lse=lse[:, 0], total=(loss.double().sum() / count).float().view(1), dh=None, dw=None)
    if s['case']['grads']:
        p /= total
        p.scatter_add_(1, at, torch.full_like(lt, -1.0))
        p *= torch.where(valid, 1.0 / count, 0.0).float()[:, None]
        out['dh'], out['dw'] = (p @ w).to(dt), (p.t() @ h).to(dt)
    return out


def _clip_own(s):
    from dp_cgans_amd import ops
    ops.grad_clip(s['plan'], MAX_NORM, s['out'])
    return s['out']


def _clip(s):
    norm = s['g'].double().square().sum().sqrt()
    return torch.stack([norm, (MAX_NORM / norm).clamp(max=1.0)]).float()


def _adamw_own(s):
    from dp_cgans_amd import ops
    s['t'] += 1
    ops.adamw_step(s['plan'], lr=LR, b1=B1, b2=B2, eps=EPS, coef=s['coef'], t_host=s['t'])


def _adamw(s):
    """The flat buffers hold zeros between the tensors, where a step leaves zeros."""
    s['t'] += 1
    wd = _per_block(s['wd'], s['layout'], s['p'].numel(), s['p'].device).repeat_interleave(BLOCK)
    if s['case']['state'] == 32:
        g = s['g'].float() * s['coef']
        m = B1 * s['m'] + (1 - B1) * g
        v = B2 * s['v'] + (1 - B2) * g * g
        r = v.sqrt()
        s['m'].copy_(m)
        s['v'].copy_(v)
    else:
        g = s['g'].double() * s['coef']
        held = lambda k: (s[k].double().view(-1, BLOCK) * s[k + '_scale'][:, None]).view(-1)  # noqa: E731
        m = B1 * held('m') + (1 - B1) * g
        r = (B2 * held('r').square() + (1 - B2) * g * g).sqrt()
        u = ((s['dither'].int() & 0xffff).double() / 65536).view(-1, BLOCK)
        for k, x in (('m', m), ('r', r)):
            q, scale = _hold8(x.view(-1, BLOCK), u)
            if k == 'r':                                 # a root that is not zero is not held as zero
                q = torch.where(x.view(-1, BLOCK) > 0, q.clamp(min=2.0 ** -9), q)
            s[k].copy_(q.view(-1).float().to(torch.float8_e4m3fn))
            s[k + '_scale'].copy_(scale)
        m, r = m.float(), r.float()
    step = LR / (1 - B1 ** s['t'])
    p = s['p'].float() * (1 - LR * wd) - step * (m / (r / math.sqrt(1 - B2 ** s['t']) + EPS))
    s['p'].copy_(p)
    if s['copy'] is not None:
        s['copy'].copy_(p)


def run(state):
    op = state['case']['op']
    if op == 'lce':
        return _lce_own(state) if own else _lce(state)
    if op == 'clip':
        return _clip_own(state) if own else _clip(state)
    (_adamw_own if own else _adamw)(state)
    # the program's own buffers; an 8-bit state is its codes, as numbers, and the scales of their blocks
    return {k: state[k] for k in ('p', 'copy', 'm', 'v', 'r', 'm_scale', 'r_scale') if k in state}


def work(case):
    size = lambda k: 4 if case[k] == 'f32' else 2  # noqa: E731
    if case['op'] == 'lce':
        T, D, V = case['T'], case['D'], case['V']
        b = (4 if case['dtype'] == 'f32' else 2) * D * (T + V) * (2 if case['grads'] else 1) + 16 * T
        return dict(bytes=b, flops=(6 if case['grads'] else 2) * T * D * V)
    n = sum(math.prod(s) for s in _shapes(case))
    if case['op'] == 'clip':
        return dict(bytes=n * size('g'), flops=2 * n)
    b = 2 * size('p') + size('g') + (2 if case['copy'] else 0)
    # 8 bits: both states and their scales in and out, and the 16 random bits of each element
    b += 16 if case['state'] == 32 else 4 + 16 / BLOCK + 2
    return dict(bytes=n * b, flops=16 * n)


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case['op'] == 'lce':
        h, w, target = s['h'].double(), s['w'].double(), s['target']
        rows = (target != IGNORE).nonzero()[:, 0]
        logp = torch.mm(h, w.t())
        lse = torch.logsumexp(logp, 1)
        logp -= lse[:, None]
        loss = torch.zeros_like(lse)
        loss[rows] = -logp[rows, target[rows]]
        n = max(1, rows.numel())
        out = dict(loss=loss, lse=lse, total=(loss.sum() / n).view(1), dh=None, dw=None)
        if case['grads']:
            d = torch.zeros_like(logp)
            d[rows] = logp[rows].exp_()
            del logp
            d[rows, target[rows]] = torch.expm1(-loss[rows])
            d /= n
            out['dh'], out['dw'] = torch.mm(d, w), torch.mm(d.t(), h)
        return out
    if case['op'] == 'clip':
        norm = torch.linalg.vector_norm(s['g'].double())
        return torch.stack([norm, torch.where(norm > MAX_NORM, MAX_NORM / norm, 1.0)])
    return _exact_adamw(s)


def _exact_adamw(s):
    layout, dev = s['layout'], s['p'].device
    total, t = s['p'].numel(), T_STEP + 1
    grad = s['g'].double() * s['coef'].double()
    if s['case']['state'] == 32:
        m0, v0 = s['m'].double(), s['v'].double()
    else:
        wide = lambda k: s[k].float().double() * s[k + '_scale'].double().repeat_interleave(BLOCK)  # noqa: E731
        m0, v0 = wide('m'), wide('r') ** 2
    m = torch.lerp(grad, m0, B1)
    v = torch.lerp(grad * grad, v0, B2)
    decay = _per_block(s['wd'], layout, total, dev).double().repeat_interleave(BLOCK)
    p = s['p'].double()
    p = p - LR * decay * p - LR * (m / (1 - B1 ** t)) / ((v / (1 - B2 ** t)).sqrt() + EPS)
    out = dict(p=p, copy=p if s['copy'] is not None else None)
    if s['case']['state'] == 32:
        out.update(m=m, v=v)
    else:                                    # (the codes follow the random bits: only their scales have a value here)
        top = lambda x: torch.maximum(x.abs().view(-1, BLOCK).amax(1), torch.tensor(2.0 ** -100, device=dev)) / 448  # noqa: E731
        out.update(m=None, r=None, m_scale=top(m), r_scale=top(v.sqrt()))
    return out
