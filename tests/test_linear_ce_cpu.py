"""linear_cross_entropy's sizes and refusals through the C-ABI, without a GPU (nothing is launched)."""
import pytest

from dp_cgans_amd._lib import lib


def ws(*a):
    return lib().cdll.dpc_linear_cross_entropy_ws(*a)


def test_workspace_sizes():
    half, full = ws(8192, 1024, 18000, 1, 1, 0, 0), ws(8192, 1024, 18000, 0, 1, 0, 0)
    assert 8192 * 18000 * 2 < half < 8192 * 18000 * 2 * 1.4 and full > 8192 * 18000 * 4
    assert ws(8192, 1024, 18000, 1, 0, 0, 0) < half / 8                      # the loss alone keeps no logits
    assert ws(8192, 1024, 18000, 1, 1, 0, 256) < half / 2                    # smaller pieces, less of them
    assert ws(8192, 1024, 18000, 1, 1, 1, 256) < ws(8192, 1024, 18000, 1, 1, 0, 256)      # fp32 dw holds its own sums
    assert ws(1 << 20, 64, 131072, 1, 1, 1, 0) < 1.3 * 2 ** 30


@pytest.mark.parametrize('a', [(-1, 64, 10, 1, 1, 0, 0), (4, 0, 10, 0, 1, 0, 0), (4, 64, 0, 1, 1, 0, 0), (4, 60, 10, 2, 1, 0, 0),
                               (4, 64, 10, 3, 1, 0, 0), (1 << 31, 64, 10, 1, 1, 0, 0)])
def test_refused_sizes(a):
    assert ws(*a) == -1 and b'linear_cross_entropy' in lib().cdll.dpc_last_error()


@pytest.mark.parametrize('change,match', [
    (dict(h=None), 'null'), (dict(w=None), 'null'), (dict(target=None), 'null'), (dict(loss=None), 'null'), (dict(ws=None), 'null'),
    (dict(ldh=56), 'leading'), (dict(lddw=56), 'leading'), (dict(h=0x10008), 'aligned'), (dict(ldw=68), 'aligned'),
    (dict(dw=0x70008), 'aligned'), (dict(lddh=68), 'aligned'), (dict(ws=0x80010), '256'), (dict(ws_bytes=1000), 'smaller'),
    (dict(accumulate=1), 'accumulation'), (dict(D=60), 'multiple of 8'), (dict(dtype=7), 'type'), (dict(T=-1), 'size')])
def test_refused_arguments(change, match):
    a = dict(h=0x10000, ldh=64, w=0x20000, ldw=64, dtype=1, target=0x30000, ignore=-100, T=16, D=64, V=100, loss=0x40000, lse=None,
             total=None, dh=0x60000, lddh=64, dw=0x70000, lddw=64, dw_f32=0, accumulate=0, gscale=1.0, mean=1, piece=0, ws=0x80000,
             ws_bytes=1 << 30, stream=None)
    assert set(change) <= set(a)
    a.update(change)
    with pytest.raises(RuntimeError, match=match):
        lib().call('dpc_linear_cross_entropy', *a.values())


@pytest.mark.parametrize('change', [dict(dh=0x10000), dict(dh=0x20000), dict(dw=0x10000), dict(dw=0x20000), dict(dw=0x60000)])
def test_a_gradient_over_an_operand_is_refused(change):
    test_refused_arguments(change, 'must not lie')


@pytest.mark.parametrize('change', [dict(T=(1 << 21) + 1, V=8, piece=1 << 30), dict(dtype=0, T=(1 << 23) + 1, V=1, piece=1 << 30, D=1),
                                    dict(T=1 << 20, V=1 << 26, D=8, piece=1 << 20)])
def test_pieces_past_a_launch_are_refused(change):
    test_refused_arguments(dict(change, ws_bytes=1 << 62), 'piece is too large')
