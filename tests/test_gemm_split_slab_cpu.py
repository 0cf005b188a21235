"""The partial products of a split K side by side (dpc_gemm_desc.split_slab): what is refused, before anything is launched."""
import ctypes

import pytest

from dp_cgans_amd import ops


def desc(M=70, N=90, K=640, splitk=4, tile=64, slab=70 * 90, **more):
    d = ops.GemmDesc()
    d.M, d.N, d.K, d.alpha = M, N, K, 1.0
    d.A, d.a_rs, d.a_cs, d.B, d.b_rs, d.b_cs, d.C, d.ldc = 0x10000, K, 1, 0x20000, N, 1, 0x30000, N
    d.splitk, d.tile, d.split_slab = splitk, tile, slab
    for k, v in more.items():
        setattr(d, k, v)
    return d


@pytest.mark.parametrize('change', [dict(splitk=1), dict(splitk=0), dict(tile=0), dict(tile=128), dict(beta=1.0), dict(epi=1, aux_out=0x40000, ld_aux_out=90),
                                    dict(bias=0x40000), dict(slab=70 * 90 - 1), dict(slab=-1), dict(ldc=100), dict(atomic=1)])
def test_refused(change):
    d = desc(**change)
    with pytest.raises(RuntimeError, match='gemm: '):
        ops.lib().call('dpc_gemm_f32_ex', ctypes.byref(d), 1, None)


def test_refused_in_a_group():
    two = (ops.GemmDesc * 2)(desc(), desc())
    with pytest.raises(RuntimeError, match='slabs'):
        ops.lib().call('dpc_gemm_f32_group', ctypes.byref(two), 2, None)
