"""attention_kv4 with query rows at the end of bf16's range and beyond it."""

import math

import pytest
import torch

import paged_oracle as O
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P
from test_paged_gpu import _check, _problem, _tiles, _wide

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    K.check_device_error(torch.device("cuda", 0), "before the test")
    yield
    torch.cuda.synchronize()


def _one(rows, n, dt):
    hq, h = 8, 2
    p = _problem([(rows, n)], hq, h, 16, 64, dt, 41, cols_more=_wide(60, 1, hq, h) if rows > 9 else 0)
    assert _tiles(p[2], rows, hq, h, 16) == (rows > 9)
    return p


@pytest.mark.parametrize("rows", [1, 7, 60])
@pytest.mark.parametrize("up", [101, 112, 125])
def test_queries_near_the_largest_number(rows, up):
    """bf16 queries of 2^101 and more over keys of 2^-100."""
    dt = torch.bfloat16
    q, cache, table, lens, start = _one(rows, 200, dt)
    q = (q.double().clamp(-3, 3) * 2.0 ** up).to(dt)
    codes, step, mid = O.unpack(cache, dt)
    step[0] = (step[0].double() * 2.0 ** -100).to(dt)
    mid[0] = (mid[0].double() * 2.0 ** -100).to(dt)
    cache = O.pack(codes, step, mid)
    scale = 2.0 ** (100 - up - 2) / math.sqrt(128)
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(), rows,
                               scale, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    _check(out, lse, O.attend(q, cache, table, lens, start, scale, tiles=rows > 9), dt)


@pytest.mark.parametrize("rows", [1, 7, 60])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_an_infinite_query_is_not_a_number(dt, rows):
    """Whatever the keys' signs are in its channel: scores of -inf alone are no row without tokens."""
    q, cache, table, lens, start = _one(rows, 100, dt)
    codes, step, mid = O.unpack(cache, dt)
    codes[0, ..., 9] = codes[0, ..., 9] % 8  # below the middle, and that is below zero
    mid[0] = -mid[0].abs() - 0.125
    cache = O.pack(codes, step, mid)
    ref = O.attend(q, cache, table, lens, start, tiles=rows > 9)
    q[0, 1, 9], q[rows - 1, 6, 9] = math.inf, -math.inf
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(), rows,
                               return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    bad = torch.zeros(out.shape[:2], dtype=torch.bool)
    bad[0, 1] = bad[rows - 1, 6] = True
    assert out.cpu()[bad].isnan().all() and lse.cpu()[bad].isnan().all()
    want = ref[0].clone()
    want[bad] = math.nan
    _check(out, None, (want, *ref[1:]), dt)
