"""linear_cross_entropy: which pieces of rows a launch takes, without a GPU (nothing is launched)."""
import pytest

from dp_cgans_amd._lib import lib
from test_linear_ce_cpu import test_refused_arguments as refused, ws

BF16, F32 = 1, 0


def test_rows_past_a_launch_are_refused():
    """The pass over a row's slabs takes 64 threads for each row, a launch less than 2^32."""
    refused(dict(T=1 << 27, D=8, V=8, ldh=8, ldw=8, dh=None, dw=None, piece=1 << 26, ws_bytes=1 << 62), 'piece is too large')


@pytest.mark.parametrize('a', [(1 << 27, 8, 8, BF16, 0, 0, 1 << 26), ((1 << 21) + 1, 8, 8, BF16, 1, 0, 1 << 30),
                               ((1 << 23) + 1, 1, 1, F32, 1, 0, 1 << 30), (1 << 20, 8, 1 << 26, BF16, 1, 0, 1 << 20)])
def test_no_workspace_for_a_piece_that_is_refused(a):
    assert ws(*a) == -1 and b'piece is too large' in lib().cdll.dpc_last_error()


@pytest.mark.parametrize('dtype', [F32, BF16])
@pytest.mark.parametrize('grads', [0, 1])
@pytest.mark.parametrize('V', [1, 4096, 1 << 20, (1 << 27) - 1, 1 << 27, 1 << 28])
def test_pieces_of_no_given_size_fit(V, grads, dtype):
    """Whatever the rows, where the caller leaves the size of a piece open."""
    for T in (0, 1, 127, 128, 1000, 1 << 22, (1 << 31) - 1):
        assert ws(T, 8, V, dtype, grads, 0, 0) > 0, T
