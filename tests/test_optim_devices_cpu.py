"""grad_clip and adamw_step take tensors of the plan's GPU only.  Without a GPU: stand-ins for tensors of two of them, and a
library that launches nothing."""
import types

import pytest
import torch

from dp_cgans_amd import ops


class Standin(object):
    """What the wrappers ask of a tensor."""

    def __init__(self, device, dtype, n, contiguous=True):
        self.device, self.dtype, self.n, self.contiguous = torch.device(device), dtype, n, contiguous
        self.is_cuda = self.device.type == 'cuda'

    def get_device(self):
        return self.device.index if self.is_cuda else -1

    def numel(self):
        return self.n

    def is_contiguous(self):
        return self.contiguous

    def data_ptr(self):
        return 0x1000


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(ops, 'lib', lambda: types.SimpleNamespace(call=lambda *a: seen.append(a)))
    monkeypatch.setattr(ops, '_raw_stream', lambda device: 0)
    monkeypatch.setattr(ops.torch.cuda, 'current_device', lambda: 0)
    return seen


def plan(device='cuda:0'):
    return ops.MultiPlan(ops.MultiInfo(), Standin(device, torch.uint8, 4096), None)


def f32(device='cuda:0', n=2, **kw):
    return Standin(device, torch.float32, n, **kw)


def i32(device='cuda:0'):
    return Standin(device, torch.int32, 1)


def i64(device='cuda:0', **kw):
    return Standin(device, torch.int64, 2, **kw)


def test_tensors_of_the_plans_gpu_are_taken(calls):
    ops.grad_clip(plan(), 1.0, f32(), t_dev=i32())
    ops.adamw_step(plan(), 1e-3, coef=f32(n=1), t_dev=i32(), t_host=0, rng=i64())
    assert [c[0] for c in calls] == ['dpc_grad_clip', 'dpc_adamw_step']


@pytest.mark.parametrize('other', ['cuda:1', 'cpu'])
@pytest.mark.parametrize('name', ['out', 't_dev', 'plan'])
def test_grad_clip_refuses_another_gpus(calls, name, other):
    a = dict(plan=plan(), max_norm=1.0, out=f32(), t_dev=i32())
    a[name] = dict(plan=plan, out=f32, t_dev=i32)[name](other)
    with pytest.raises((ValueError, RuntimeError), match='GPU|device'):
        ops.grad_clip(**a)
    assert not calls


@pytest.mark.parametrize('other', ['cuda:1', 'cpu'])
@pytest.mark.parametrize('name', ['coef', 't_dev', 'rng', 'plan'])
def test_adamw_step_refuses_another_gpus(calls, name, other):
    a = dict(plan=plan(), lr=1e-3, coef=f32(n=1), t_dev=i32(), rng=i64())
    a[name] = dict(plan=plan, coef=f32, t_dev=i32, rng=i64)[name](other)
    with pytest.raises((ValueError, RuntimeError), match='GPU|device'):
        ops.adamw_step(**a)
    assert not calls


def test_two_words_that_are_apart_are_refused(calls):
    with pytest.raises(ValueError, match='rng'):
        ops.adamw_step(plan(), 1e-3, rng=i64(contiguous=False))
    assert not calls
