"""linear_cross_entropy where the logits leave the usual range, against the formulas in fp64.  The logits are exact in every type
here, so what is off is the operator's own.

u = 2^-24, e = half a step of the operands' type (bf16 2^-8, fp16 2^-11, fp32 u)."""
import pytest
import torch

from test_linear_ce_gpu import DEV, E, TINY, TYPES, U, call, within

pytestmark = pytest.mark.gpu


@pytest.fixture(scope='module')
def ops():
    from dp_cgans_amd import ops as o
    return o


@pytest.mark.parametrize('dtype', TYPES)
@pytest.mark.parametrize('V', [50, 700, 34000])
@pytest.mark.parametrize('T', [3, 40, 300])
def test_logits_of_any_finite_size(ops, T, V, dtype):
    """Logits +-c 2^k, c up to 15 and k up to 100 (27 in fp16), and 7/8 of that in every third class.  Differences of a row's logits
    are exact in fp32, whatever their size: each term is e^0 or 0, the loss log(number of the largest) or that and 1/8 of a
    logit.  Roundings: the difference and the logarithm, 4 of the loss; the sum of V terms in runs of at most 64 + 8 + V / 1024;
    16 for the exponential, the joins and the logarithm's last bits.  p_t - 1 = expm1(-loss) is off by p_t times what the loss is,
    p_t loss <= 1/e.  d: 2^-11 for what is held in fp16, e."""
    hs, ws = (2.0 ** 12, 2.0 ** 15) if dtype == torch.float16 else (2.0 ** 50, 2.0 ** 50)
    g = torch.Generator(device=DEV).manual_seed(T + V)
    c = (1 + torch.arange(T, device=DEV) % 15).float() * (1 - 2 * (torch.arange(T, device=DEV) // 15 % 2))
    h, w = torch.zeros(T, 8, device=DEV), torch.zeros(V, 8, device=DEV)
    h[:, 0], h[:, 1] = c * hs, c * hs / 8
    w[:, 0], w[:, 1] = ws, torch.where(torch.arange(V, device=DEV) % 3 == 1, -ws, 0.0)
    h, w = h.to(dtype), w.to(dtype)
    target = torch.randint(0, V, (T,), device=DEV, generator=g)
    o = call(ops, h, w, target)
    h64, w64 = h.double(), w.double()
    l = h64 @ w64.t()
    top = l.amax(1)
    x = torch.exp(l - top[:, None])
    log = torch.log(x.sum(1))
    loss = (top - l.gather(1, target[:, None])[:, 0]) + log
    el = (64 + 8 + V / 1024 + 16) * U
    within(o['loss'], loss, el + 4 * U * loss, 'loss')
    within(o['lse'], top + log, el + 4 * U * top.abs(), 'lse')
    within(o['total'][0], loss.mean(), el + 6 * U * loss.mean(), 'total')
    d = x / x.sum(1, keepdim=True)
    d.scatter_(1, target[:, None], torch.expm1(-loss)[:, None])
    e = E[dtype]
    ed = d.abs() * (2.0 ** -11 * (dtype != torch.float32) + e + 2 * el)
    ed.scatter_add_(1, target[:, None], torch.full_like(loss, 2 * el + 4 * U)[:, None])
    for name, want, err in (('dh', d @ w64 / T, (ed + V * U * d.abs()) @ w64.abs() / T), ('dw', d.t() @ h64 / T, (ed + T * U * d.abs()).t() @ h64.abs() / T)):
        within(o[name], want, err + e * (want.abs() + err) + TINY[dtype], name)
