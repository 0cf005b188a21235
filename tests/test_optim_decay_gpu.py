"""adamw_step's weight decay where lr * wd is small beside 1."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'
N = 1 << 20


@pytest.fixture(scope='module')
def ops():
    from dp_cgans_amd import ops as o
    return o


def state(ops, eight, p, g):
    if eight:
        (m, ms), (v, vs) = ops.adamw_state8(p), ops.adamw_state8(p)
        return dict(exp_avg=[m], exp_avg_sq=[v], m_scale=[ms], v_scale=[vs], dither=[torch.zeros_like(p, dtype=torch.int16)])
    return dict(exp_avg=[torch.zeros_like(p)], exp_avg_sq=[torch.zeros_like(p)])


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('decay', [2e-6, 1e-7, 2e-8])
@pytest.mark.parametrize('cut', [0, 1])
def test_a_small_decay_is_not_lost_or_doubled(ops, decay, eight, cut):
    """Mean drift of 2^20 parameters of size 1 to 2 against fp64, in their steps of 2^-23.

    The update spreads over +-64 steps, so the one rounding of p is off by a half at most, 0.29 in the mean square: 5 * 0.29 /
    2^10 = 0.0015 of the mean.  The update's and the decay's own roundings, 2^-24 of each, at most 8: 2^-14.  (1 - decay in
    fp32 is off by up to half a step: 0.24 of them at 1e-7, all of the 0.25 at 2e-8.)"""
    gen = torch.Generator(device=DEV).manual_seed(3)
    sign = 1 - 2 * torch.randint(0, 2, (N,), device=DEV, generator=gen).float()
    p = ((1 + torch.rand(N, device=DEV, generator=gen)) * sign)[cut:].clone()
    g = torch.randn(N, device=DEV, generator=gen)[cut:].clone()
    lr = 2.0 ** -17
    wd = float(torch.tensor(decay / lr, dtype=torch.float32))
    p0 = p.double()
    shift = lambda x: torch.cat([x.new_zeros(cut), x])[cut:]  # noqa: E731  (cut: element-wise accesses)
    p, g = shift(p), shift(g)
    s = state(ops, eight, p, g)
    ops.adamw_step(ops.adamw_plan([p], [g], wd=wd, **s), lr, b1=0.5, b2=0.5, eps=1.0, t_host=1)
    g64 = g.double()
    want = p0 - lr * wd * p0 - lr * g64 / (g64.abs() + 1.0)
    drift = float(((p.double() - want) * torch.sign(p0)).mean()) * 2.0 ** 23
    assert abs(drift) <= 0.0015 + 2.0 ** -14


@pytest.mark.parametrize('eight', [False, True])
@pytest.mark.parametrize('wd', [0.0, 0.1])
def test_an_infinite_parameter_stays_one(ops, wd, eight):
    """p (1 - lr wd) less a finite update is infinite, not NaN."""
    p = torch.ones(4096, device=DEV)
    p[5], p[700] = float('inf'), -float('inf')
    g = torch.zeros_like(p)
    ops.adamw_step(ops.adamw_plan([p], [g], wd=wd, **state(ops, eight, p, g)), 1e-3, t_host=1)
    assert p[5] == float('inf') and p[700] == -float('inf')
    assert torch.isfinite(p).sum() == 4094
