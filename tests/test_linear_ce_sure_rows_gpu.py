"""Half-precision gradients of linear_cross_entropy in rows whose target leads by far, entry by entry against the formulas in
fp64.  The logits are exact in both types here, so what is off is the operator's own.

u = 2^-24, e = half a step of the operands' type (bf16 2^-8, fp16 2^-11)."""
import pytest
import torch

from test_linear_ce_gpu import DEV, E, TINY, U, call, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from dp_cgans_amd import ops as o
    return o


def sure_rows(T, V, dtype):
    """h, w, target, logits: row r's target is class r of 64; its logit leads by 13 to 21, all others are 0.  dh's column c is
    4 d[r][c], dW's column r is h[r][r] d[r][v]: one entry of d each."""
    D = 64
    w = torch.zeros(V, D, device=DEV)
    w[:D] = 4 * torch.eye(D, device=DEV)
    target = torch.arange(T, device=DEV)
    lead = torch.linspace(13, 21, max(T, 2), device=DEV).round(decimals=0)[-T:]
    h = torch.zeros(T, D, device=DEV)
    h[target, target] = lead / 4
    h, w = h.to(dtype), w.to(dtype)
    return h, w, target, h.double() @ w.double().t()


@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
@pytest.mark.parametrize('V', [64, 1000, 40000])
@pytest.mark.parametrize('T', [1, 2, 16, 17, 64])
def test_gradients_of_sure_rows(ops, T, V, dtype):
    """Every entry of dh and dW, relative to itself: what stands beside a sure target in its slab is small and counts.

    e^(l - max) is held in fp16 times 2^15: 2^-11 relative, and half a step of fp16's smallest, 2^-25, below it: 2^-40 of the slab's
    largest.  d: e relative, in fp16 times 2^14 and so 2^-39 absolute; 192 u for the exponents (a difference up to 31 in
    powers of two: two roundings of it, three factors).  The target's p_t - 1 follows the loss (40 u + 64 u of it).  The
    result: e, and half of fp16's smallest step, far below what gscale lifts it to."""
    h, w, target, l = sure_rows(T, V, dtype)
    gscale = T * 2.0 ** 16
    o = call(ops, h, w, target, gscale=gscale)
    loss = torch.logsumexp(l, 1) - l[target, target]
    d = torch.softmax(l, 1)
    e = E[dtype]
    ed = d * (2.0 ** -11 + e + 192 * U) + 2.0 ** -40 + (2.0 ** -39 if dtype == torch.float16 else 0.0)
    d[target, target] = torch.expm1(-loss)
    ed[target, target] = loss * e + 2 * (40 * U + 64 * U * loss)
    a = gscale / T
    for name, want, err in (('dh', d @ w.double(), ed @ w.double().abs()), ('dw', d.t() @ h.double(), ed.t() @ h.double().abs())):
        want, err = a * want, a * err
        within(o[name], want, err + e * (want.abs() + err) + TINY[dtype], name)
