"""linear_cross_entropy refuses outputs that lie over an operand or each other, wherever they start, and takes those that lie
between another's rows.  Without a GPU: every call here ends at a check."""
import random

import pytest

from test_linear_ce_cpu import test_refused_arguments as refused

# h is 16 rows of 128 bytes at 0x10000, w 100 rows at 0x20000, target 128 bytes at 0x30000, loss 64 at 0x40000, dh and dw as h and w at
# 0x60000 and 0x70000, the workspace at 0x80000


@pytest.mark.parametrize('change', [
    dict(dh=0x10010), dict(dh=0x10000 - 2048 + 16), dict(dh=0x20000 + 99 * 128), dict(dh=0x30000 - 2032), dict(dw=0x10000 - 12800 + 16),
    dict(dw=0x20080), dict(dw=0x60000 + 2032), dict(dh=0x70000 + 12784), dict(loss=0x10000 + 2044), dict(loss=0x20000), dict(loss=0x30040),
    dict(lse=0x40000), dict(lse=0x4003c), dict(total=0x40020), dict(total=0x6000c), dict(lse=0x72000), dict(ws=0x10700), dict(ws=0x22000),
    dict(dh=0x80010), dict(loss=0x80100), dict(total=0x80000), dict(dtype=0, D=64, dh=0x10000 + 4092)])
def test_outputs_over_something_else_are_refused(change):
    refused(change, 'must not lie')


@pytest.mark.parametrize('change', [
    dict(lddh=128, dh=0x20000 - 15 * 256 - 112),                         # only its last row reaches w
    dict(ldh=72, dh=0x10080, lddh=136),                                  # different row lengths: h has 16 spare bytes a row
    dict(ldh=128, lddh=128, dh=0x10080 - 16),                            # 16 bytes of each row
    dict(ldh=128, lddh=128, dh=0x10080 + 256 * 15 - 16)])                # the last row of h, the first of dh
def test_rows_that_meet_are_refused(change):
    refused(change, 'must not lie')


@pytest.mark.parametrize('change', [
    dict(ldh=128, lddh=128, dh=0x10080),                                 # halves of one matrix
    dict(ldw=128, lddw=128, dw=0x20000 - 128),
    dict(ldh=128, lddh=64, dh=0x10000 + 15 * 256 + 128),                 # behind the last row
    dict(ldh=128, lddh=256, dh=0x10080, T=8),
    dict(dh=0x10000 + 2048), dict(dh=0x10000 - 2048), dict(lse=0x40040), dict(total=0x40040)])
def test_rows_between_others_are_not(change):
    """(The workspace is too small here, and that is what is said: the checks of where things lie come first.)"""
    refused(dict(change, ws_bytes=1000), 'smaller')


def test_where_rows_meet_byte_by_byte():
    rng = random.Random(1)
    met = 0
    for _ in range(2000):
        T, D = rng.randint(1, 12), 8 * rng.randint(1, 4)
        ldh, lddh = D + 8 * rng.randint(0, 6), D + 8 * rng.randint(0, 6)
        if rng.random() < 0.5:
            lddh = ldh
        dh = 0x10000 + 16 * rng.randint(-60, 60)
        rows = lambda at, ld: {at + 2 * ld * r + k for r in range(T) for k in range(0, 2 * D, 16)}  # noqa: E731
        meet = bool(rows(0x10000, ldh) & rows(dh, lddh))
        refused(dict(T=T, D=D, ldh=ldh, lddh=lddh, dh=dh, ws_bytes=1000), 'must not lie' if meet else 'smaller')
        met += meet
    assert 300 < met < 1700
