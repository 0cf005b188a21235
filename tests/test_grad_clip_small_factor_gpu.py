"""grad_clip's factor where it is smaller than fp32 holds: 0 stands for a gradient that is not finite, and for nothing else."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


@pytest.fixture(scope='module')
def ops():
    from dp_cgans_amd import ops as o
    return o


@pytest.mark.parametrize('max_norm,gscale', [(1e-30, 1.0), (1.0, 1e-60), (1e-25, 1e-30)])
def test_a_finite_gradient_is_never_skipped(ops, max_norm, gscale):
    """A factor of 1e-50 or less: the smallest normal number instead, so the step decays, counts and moves by its momentum."""
    n = 3000
    p, g = torch.ones(n, device=DEV), torch.full((n,), 1e20, device=DEV)
    m, v = torch.full((n,), 0.5, device=DEV), torch.ones(n, device=DEV)
    out, t = torch.empty(2, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    plan = ops.adamw_plan([p], [g], [m], [v], wd=0.5)
    ops.grad_clip(plan, max_norm, out, gscale=gscale, t_dev=t)
    assert out[1] == 2.0 ** -126 and t.item() == 1
    ops.adamw_step(plan, 0.25, b1=0.5, b2=0.5, coef=out[1:], t_dev=t, t_host=0)
    # m = 0.25 + 0.5 g', v = 0.5 + 0.5 g'^2, g' = 2^-126 1e20 < 2e-18: corrected moments 0.5 and 1
    want = 1 - 0.25 * 0.5 - 0.25 * 0.5
    assert ((p.double() - want).abs() <= 8 * 2.0 ** -24).all() and (m == 0.25).all()


@pytest.mark.parametrize('bad', [float('nan'), float('inf')])
def test_a_gradient_that_is_not_finite_still_gives_0(ops, bad):
    g = torch.ones(3000, device=DEV)
    g[7] = bad
    out, t = torch.empty(2, device=DEV), torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.grad_clip(ops.grad_plan([g]), 1e-30, out, t_dev=t)
    assert out[1] == 0 and t.item() == 0
