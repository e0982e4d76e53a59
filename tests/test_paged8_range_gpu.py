"""Attention over an 8-bit paged cache at the ends of its ranges: value scales and scores far
apart, query rows with outlying channels, queries near their type's largest number and beyond it,
caches without blocks.  Each case goes through the kernel for few rows and the one for many."""

import math

import pytest
import torch

import paged8_oracle as O8
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P
from test_paged8_attention_gpu import _attend, _check, _problem, _tiles, _wide

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _no_device_error():
    K.check_device_error(torch.device("cuda", 0), "before the test")
    yield
    torch.cuda.synchronize()


def _one(rows, n, dt=BF, hq=8, h=2, seed=5):
    """One sequence with `rows` query rows; 40 of them go to the kernel for many rows."""
    p = _problem([(rows, n)], hq, h, 16, dt, seed, cols_more=_wide(40, 1, hq, h) if rows > 9 else 0)
    assert _tiles(p[2], rows, hq, h, 16) == (rows > 9)
    return p


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("less", [70, 100])
def test_small_values_under_scores_that_rise(rows, less):
    """Two tokens score 73 (as powers of two) above all others, their values are 2^-70 or 2^-100 of
    theirs: the result is the others', from which next to no weight may come."""
    q, cache, table, lens, start = _one(rows, 200)
    q[:] = 1
    cache[:, :, :16] = 0
    cache[:, :, 32] = 127
    for tok in (100, 150):
        block = int(table[0, tok // 16])
        cache[block, :, tok % 16] = 0x49  # 4.5: a score of 50.9
        cache[block, :, 32, 1] = 127 - less
    ref = O8.attend(q, cache, table, lens, start)
    _check(*_attend(q, cache, table, lens, start, rows), ref, BF)
