"""The partial products of a split K side by side (dpc_gemm_desc.split_slab) against each K range's product in fp64."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda:0'


@pytest.mark.parametrize('trans_a,trans_b', [(False, False), (False, True), (True, False), (True, True)])
@pytest.mark.parametrize('M,N,K,splits,gap', [(70, 90, 640, 4, 0), (1, 1, 33, 2, 3), (64, 64, 1024, 32, 0), (129, 200, 100, 3, 56), (5, 67, 20, 2, 0)])
def test_each_range_has_its_slab(trans_a, trans_b, M, N, K, splits, gap):
    """K ranges are whole tiles of 32, dealt out evenly; one that has nothing left is a slab of zeros.  The gap between two
    slabs, and between two rows, stays as it was."""
    from dp_cgans_amd import ops
    g = torch.Generator(device=DEV).manual_seed(M + N + K)
    A = torch.randn(*((K, M) if trans_a else (M, K)), device=DEV, generator=g)
    B = torch.randn(*((N, K) if trans_b else (K, N)), device=DEV, generator=g)
    ldc = N + gap
    out = torch.full((splits, M * ldc + gap), 7.0, device=DEV)
    d = ops.gemm_desc(A, B, out[0, :M * ldc].view(M, ldc)[:, :N], trans_a=trans_a, trans_b=trans_b, alpha=0.5, splitk=splits, tile=64)
    d.split_slab = out.shape[1]
    ops.gemm_run([d])
    a, b = (A.t() if trans_a else A).double(), (B.t() if trans_b else B).double()
    step = -(-(-(-K // 32)) // splits) * 32
    for s in range(splits):
        x, y = a[:, s * step:(s + 1) * step], b[s * step:(s + 1) * step]
        got = out[s, :M * ldc].view(M, ldc)
        # fp32 sums of at most `step` products, one rounding for alpha
        assert ((got[:, :N].double() - 0.5 * (x @ y)).abs() <= (step + 2) * 2.0 ** -24 * 0.5 * (x.abs() @ y.abs())).all()
        assert (got[:, N:] == 7).all() and (out[s, M * ldc:] == 7).all()
