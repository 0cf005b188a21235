"""Plans of the multi-tensor optimiser: what the library refuses and lays out, without a GPU (nothing is launched)."""
import ctypes

import pytest

from dp_cgans_amd import ops
from dp_cgans_amd._lib import lib


def tensors(*ns, **kw):
    arr = (ops.MultiTensor * max(len(ns), 1))()
    for k, n in enumerate(ns):
        base = 0x10000 * (k + 1)
        arr[k].p, arr[k].g, arr[k].m, arr[k].v, arr[k].n = base, base + 0x1000, base + 0x2000, base + 0x3000, n
        for name, x in kw.items():
            setattr(arr[k], name, x)
    return arr


def size(arr, n):
    info = ops.MultiInfo()
    lib().call('dpc_multi_plan_size', arr, n, ctypes.byref(info))
    return info


def test_chunks_cover_every_tensor_once():
    ns = (1, 0, 2048, 2049, 5000)
    arr = tensors(*ns)
    info = size(arr, len(ns))
    assert (info.kind, info.count, info.blocks) == (1, 5, 1 + 0 + 1 + 2 + 3)
    host = (ctypes.c_uint8 * info.bytes)()
    lib().call('dpc_multi_plan', arr, len(ns), ctypes.byref(info), host, info.bytes)

    class Chunk(ctypes.Structure):
        _fields_ = [('t', ctypes.c_int32), ('pad', ctypes.c_int32), ('start', ctypes.c_int64)]

    chunks = (Chunk * info.blocks).from_buffer(host, info.chunk_off)
    got = {}
    for c in chunks:
        got.setdefault(c.t, []).append(c.start)
    assert got == {k: list(range(0, n, 2048)) for k, n in enumerate(ns) if n}
    assert info.part_off + 2048 * 8 == info.bytes and info.chunk_off + 16 * info.blocks <= info.part_off


@pytest.mark.parametrize('change,match', [
    (dict(n=-1), 'size'), (dict(g=None), 'gradient'), (dict(m=None), 'moments'), (dict(g=0x10001), 'misaligned'),
    (dict(m=0x20002), 'misaligned'), (dict(p_type=3), 'type'), (dict(g_type=-1), 'type'), (dict(wd=-0.5), 'decay'),
    (dict(wd=float('nan')), 'decay'), (dict(m_scale=0x40000), 'scales'), (dict(dither=0x40000), '8-bit'),
    (dict(p=None), 'without a parameter')])
def test_a_plan_refuses_what_no_step_could_take(change, match):
    with pytest.raises(RuntimeError, match=match):
        size(tensors(100, **change), 1)


def test_a_plan_holds_tensors_of_one_kind():
    arr = tensors(100, 100)
    arr[1].m_scale, arr[1].v_scale = 0x50000, 0x60000
    with pytest.raises(RuntimeError, match='one kind'):
        size(arr, 2)
    assert size(tensors(100, m_scale=0x50000, v_scale=0x60000), 1).kind == 2
    assert size(tensors(100, m_scale=0x50000, v_scale=0x60000, dither=0x70000), 1).kind == 4


def test_a_plan_is_written_only_where_it_fits():
    arr = tensors(5000)
    info = size(arr, 1)
    host = (ctypes.c_uint8 * info.bytes)()
    with pytest.raises(RuntimeError, match='sizes'):
        lib().call('dpc_multi_plan', arr, 1, ctypes.byref(info), host, info.bytes - 1)
    with pytest.raises(RuntimeError, match='sizes'):
        lib().call('dpc_multi_plan', tensors(9000), 1, ctypes.byref(info), host, info.bytes)
    with pytest.raises(RuntimeError, match='null'):
        lib().call('dpc_multi_plan', arr, 1, ctypes.byref(info), None, info.bytes)


def test_steps_refuse_bad_numbers_before_any_launch():
    info = size(tensors(100), 1)
    step = lambda *a: lib().call('dpc_adamw_step', ctypes.byref(info), 0x1000, *a)  # noqa: E731
    for a in ((1e-3, 1.0, 0.9, 1e-8, None, 1.0, None, 1, None, 0, None), (1e-3, 0.9, 0.9, 1e-8, None, 1.0, None, 0, None, 0, None),
              (float('nan'), 0.9, 0.9, 1e-8, None, 1.0, None, 1, None, 0, None)):
        with pytest.raises(RuntimeError, match='adamw'):
            step(*a)
    for top, gs in ((0.0, 1.0), (1.0, 0.0), (float('nan'), 1.0)):
        with pytest.raises(RuntimeError, match='grad_clip'):
            lib().call('dpc_grad_clip', ctypes.byref(info), 0x1000, top, gs, 0x2000, None, None)


def test_tensors_must_live_on_the_gpu():
    import torch
    x = torch.zeros(8)
    with pytest.raises(ValueError, match='GPU'):
        ops.grad_plan([x])
    with pytest.raises(ValueError, match='GPU'):
        ops.adamw_plan([x], [x], [x], [x])
