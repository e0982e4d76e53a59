"""attention_kv4: tokens that a row does not see, whatever their keys and values are, take nothing
of the row's precision."""

import pytest
import torch

import paged_oracle as O
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P
from test_paged_gpu import _cache4, _gen, _tiles, _wide

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _huge(cache, dt, table, tokens, planes, by):
    """The cache with step and mid of the tokens' keys (plane 0) or values (1) times ``by``."""
    codes, step, mid = O.unpack(cache, dt)
    for t in tokens:
        at = (int(table[t // 16]), slice(None), t % 16)
        for p in planes:
            step[p][at] = (step[p][at].double() * by).to(dt)
            mid[p][at] = (mid[p][at].double() * by).to(dt)
    return O.pack(codes, step, mid)


@pytest.mark.parametrize("planes", [(0,), (1,), (0, 1)])
@pytest.mark.parametrize("rows,length,g_size", [(5, 77, 64), (9, 300, 32), (40, 333, 64),
                                                (90, 90, 128), (90, 700, 64)])
@pytest.mark.parametrize("dt,base,by", [(BF, 1.0, 2.0 ** 20), (BF, 1.0, 2.0 ** 100),
                                        (BF, 2.0 ** -40, 2.0 ** 60), (FP, 2.0 ** -6, 2.0 ** 19)])
def test_a_row_does_not_feel_what_comes_behind_it(dt, base, by, rows, length, g_size, planes):
    """The last third of the rows' own tokens is huge: rows in front of them are as without."""
    g = _gen(rows)
    hq, h, bs = 8, 2, 16
    cols = -(-length // bs)
    tiles = rows >= 40
    table = torch.full((1, cols + (_wide(rows, 1, hq, h) if tiles else 0)), -7, dtype=torch.int32)
    table[0, :cols] = torch.randperm(cols + 2, generator=g)[:cols].int()
    assert _tiles(table, rows, hq, h, bs) == tiles
    cache = _cache4(cols + 2, h, bs, g_size, dt, g)
    codes, step, mid = O.unpack(cache, dt)
    cache = O.pack(codes, *((x.double() * base).to(dt) for x in (step, mid)))
    q = (torch.randn((rows, hq, 128), generator=g) / base ** 0.5).to(dt)
    start, lens = torch.tensor([0, rows]).int(), torch.tensor([length]).int()
    first = length - rows // 3
    hurt = _huge(cache, dt, table[0], range(first, length), planes, by)
    out, lse = P.attention_kv4(q.cuda(), hurt.cuda(), table.cuda(), lens.cuda(), start.cuda(),
                               rows, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    kept = rows - rows // 3
    want, z, tol, ltol = O.attend(q[:kept], cache, table, torch.tensor([first]),
                                  torch.tensor([0, kept]), tiles=tiles)
    bound = tol + O.half_step(dt) * (want.abs() + tol)
    bound = bound + torch.finfo(dt).eps * torch.finfo(dt).tiny
    off = ((out[:kept].double().cpu() - want).abs() / bound).max()
    assert off <= 1, float(off)
    assert ((lse[:kept].double().cpu() - z).abs() <= ltol).all()


@pytest.mark.parametrize("rows", [5, 60])
@pytest.mark.parametrize("planes", [(0,), (1,)])
def test_tokens_of_many_scales(rows, planes):
    """Keys or values of 2^-40 to 2^0 from token to token, all seen, the 64-bit form's result."""
    dt, hq, h, bs, length = BF, 8, 2, 16, 400
    g = _gen(rows + 100)
    cols = -(-length // bs)
    tiles = rows == 60
    table = torch.full((1, cols + (_wide(rows, 1, hq, h) if tiles else 0)), -7, dtype=torch.int32)
    table[0, :cols] = torch.randperm(cols, generator=g).int()
    cache = _cache4(cols, h, bs, 64, dt, g)
    codes, step, mid = O.unpack(cache, dt)
    by = torch.exp2(-torch.randint(0, 41, (cols, 1, bs, 1), generator=g).double())
    for p in planes:
        step[p], mid[p] = (step[p].double() * by).to(dt), (mid[p].double() * by).to(dt)
    cache = O.pack(codes, step, mid)
    q = torch.randn((rows, hq, 128), generator=g).to(dt)
    start, lens = torch.tensor([0, rows]).int(), torch.tensor([length]).int()
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(),
                               rows, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    want, z, tol, ltol = O.attend(q, cache, table, lens, start, tiles=tiles)
    bound = tol + O.half_step(dt) * (want.abs() + tol)
    assert ((out.double().cpu() - want).abs() <= bound).all()
    assert ((lse.double().cpu() - z).abs() <= ltol).all()
