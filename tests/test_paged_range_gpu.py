"""attention_kv4 at the ends of its range: scores far below zero, weights far below the largest."""

import math

import pytest
import torch

import paged_oracle as O
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P
from test_paged_gpu import _cache4, _gen, _tiles, _wide
from test_paged_precision_gpu import one_head

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.mark.parametrize("rows", [1, 5, 60])
@pytest.mark.parametrize("length", [64, 300])
def test_scores_far_below_zero(rows, length):
    """Every score of a row is about -1e33: equal keys weigh alike, as around zero."""
    hq, h, bs, dt = 8, 2, 16, BF
    g = _gen(rows)
    cols = -(-length // bs)
    tiles = rows == 60
    table = torch.full((1, cols + (_wide(rows, 1, hq, h) if tiles else 0)), -7, dtype=torch.int32)
    table[0, :cols] = torch.randperm(cols, generator=g).int()
    assert _tiles(table, rows, hq, h, bs) == tiles
    codes, step, mid = O.unpack(_cache4(cols, h, bs, 64, dt, g), dt)
    step[0], mid[0] = 0, 1e16
    cache = O.pack(codes, step, mid)
    q = (-1e16 * (0.5 + torch.rand((rows, hq, 128), generator=g))).to(dt)
    start, lens = torch.tensor([0, rows]).int(), torch.tensor([length]).int()
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(),
                               rows, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    x = O.values(cache, dt)[0][1][table[0, :cols].long()].transpose(0, 1).flatten(1, 2)
    w = q.double().sum(-1) * float(mid[0].max()) / math.sqrt(128)  # every key is the mid
    assert (w < -1e32).all()
    # fp32's sums of 128 equal signs and one 2^-24 a factor; log of the count is lost beside it
    assert ((lse.double().cpu() - w).abs() <= 2 ** -18 * w.abs()).all()
    for i in range(rows):
        v = x[:, :length - rows + i + 1].repeat_interleave(hq // h, 0)
        want, mag = v.mean(1), v.abs().mean(1)
        # weights and values to fp16, the output's own rounding, fp32's sums
        tol = (2 ** -10 + 2 ** -18) * mag + O.half_step(dt) * (want.abs() + 2 ** -9 * mag)
        assert ((out[i].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("dt,mag", [(BF, 1e5), (BF, 1e9), (FP, 3e4)])
@pytest.mark.parametrize("rows", [1, 7, 60])
def test_scores_of_any_size(dt, mag, rows):
    """Scores of both signs up to 1e10 and 1e18: fp32 holds them to 2^-24 of their size, so a
    row is the value of its largest key, provided that this is ahead of the others by more."""
    hq, h, bs, length = 8, 2, 16, 200
    g = _gen(rows + 3)
    cols = -(-length // bs)
    tiles = rows == 60
    table = torch.full((1, cols + (_wide(rows, 1, hq, h) if tiles else 0)), -7, dtype=torch.int32)
    table[0, :cols] = torch.randperm(cols, generator=g).int()
    codes, step, mid = O.unpack(_cache4(cols, h, bs, 64, dt, g, spread=0.0), dt)
    size = mag / 16
    step[0], mid[0] = (step[0].double() * size).to(dt), (mid[0].double() * size).to(dt)
    cache = O.pack(codes, step, mid)
    q = (torch.randn((rows, hq, 128), generator=g) * size).to(dt)
    start, lens = torch.tensor([0, rows]).int(), torch.tensor([length]).int()
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(),
                               rows, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    x = O.values(cache, dt)[0][:, table[0, :cols].long()].permute(0, 2, 1, 3, 4).flatten(2, 3)
    seen = length - rows + 1 + torch.arange(rows)
    clear = 0
    for head in range(hq):
        k, v = x[0, head // 4, :length], x[1, head // 4, :length]
        _, z, _, werr = one_head(q[:, head], k, v, seen, 1 / math.sqrt(128))
        l = lse[:, head].double().cpu()
        assert ((l - z).abs() <= 2 * werr).all()
        for i in range(rows):
            top = (q[i, head].double() @ k[:seen[i]].T / math.sqrt(128)).topk(2)
            if top.values[0] - top.values[1] < 4 * werr[i] + 50:
                continue
            clear += 1
            want = v[top.indices[0]]
            tol = (2 ** -10 + 2 ** -18) * want.abs() + 2 ** -24 * v.abs().max()
            tol = tol + O.half_step(dt) * (want.abs() + tol)
            assert ((out[i, head].double().cpu() - want).abs() <= tol).all()
    assert clear > rows * hq // 2


@pytest.mark.parametrize("dt", [BF, FP])
def test_many_rows_small_weights_beside_a_large_one(dt):
    """A first token of no value takes nearly all the weight; the others, 2^-16 to 2^-20 of it,
    make up the output and keep their bits: it is off by half a step of fp16 of their p |v|
    (twice in bf16 caches, whose values are rounded too), not of the first one's."""
    hq, h, bs, rows, length = 8, 2, 16, 60, 300
    g = _gen(9)
    cols = -(-length // bs)
    table = torch.full((1, cols + _wide(rows, 1, hq, h)), -7, dtype=torch.int32)
    table[0, :cols] = torch.arange(cols).int()
    assert _tiles(table, rows, hq, h, bs)
    codes, step, mid = O.unpack(_cache4(cols, h, bs, 64, dt, g, spread=0.0), dt)
    step[0], mid[0] = step[0] * 0.125, 0
    step[:, 0, :, 0], mid[1, 0, :, 0], mid[0, 0, :, 0] = 0, 0, 1.0  # token 0: all ones, and zeros
    cache = O.pack(codes, step, mid)
    q = (torch.randn((rows, hq, 128), generator=g) * 0.1 + 1.0).to(dt)
    start, lens = torch.tensor([0, rows]).int(), torch.tensor([length]).int()
    out = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(), rows)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    x = O.values(cache, dt)[0][:, table[0, :cols].long()].permute(0, 2, 1, 3, 4).flatten(2, 3)
    seen = length - rows + 1 + torch.arange(rows)
    for head in range(hq):
        k, v = x[0, head // 4, :length], x[1, head // 4, :length]
        want, _, pv, werr = one_head(q[:, head], k, v, seen, 1 / math.sqrt(128))
        w = q[:, head].double() @ k.T / math.sqrt(128)
        below = (w[:, :1] - w[:, 1:]) / math.log(2)
        assert (below > 13).all() and (below < 21).all()
        tol = (2 ** -11 * (2 if dt == BF else 1) + 2 ** -17 + 2 * werr[:, None]) * pv
        tol = tol + O.half_step(dt) * (want.abs() + tol) + 2 ** -25
        assert ((out[:, head].double().cpu() - want).abs() <= tol).all()
        off = (out[:, head].double().cpu() - want).norm() / want.norm()
        assert off <= 2 * O.half_step(dt)


@pytest.mark.parametrize("mag", [1.0, 1e8, 1e16])
@pytest.mark.parametrize("rows", [1, 60])
def test_equal_scores_of_any_size_over_values_of_many_scales(rows, mag):
    """Equal keys, scores of 10, 1e17 and 1e33; values of 2^0, 2^-6, 2^-30 and 0 by 32 tokens, or
    by token: every token weighs the same, so that a row is the mean of what it sees."""
    hq, h, bs, dt, length = 8, 2, 16, BF, 400
    g = _gen(rows + 50)
    cols = -(-length // bs)
    tiles = rows == 60
    table = torch.full((1, cols + (_wide(rows, 1, hq, h) if tiles else 0)), -7, dtype=torch.int32)
    table[0, :cols] = torch.arange(cols).int()
    start, lens = torch.tensor([0, rows]).int(), torch.tensor([length]).int()
    q = (mag * (0.5 + torch.rand((rows, hq, 128), generator=g))).to(dt)
    codes, step, mid = O.unpack(_cache4(cols, h, bs, 64, dt, g, spread=0.0), dt)
    step[0], mid[0] = 0, mag
    token = torch.arange(cols * bs).view(cols, 1, bs, 1)
    for each in (token // 32, token * 7 // 5):
        by = torch.tensor([1.0, 2.0 ** -6, 2.0 ** -30, 0.0], dtype=torch.float64)[each % 4]
        s, m = step.clone(), mid.clone()
        s[1], m[1] = (step[1].double() * by).to(dt), (mid[1].double() * by).to(dt)
        cache = O.pack(codes, s, m)
        out = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(), rows)
        torch.cuda.synchronize()
        K.check_device_error(out.device)
        x = O.values(cache, dt)[0][1].transpose(0, 1).flatten(1, 2)
        for i in range(rows):
            v = x[:, :length - rows + i + 1].repeat_interleave(hq // h, 0)
            want, size = v.mean(1), v.abs().mean(1)
            # weights and values to fp16 (those 2^-30 below go under: 2^-24 of the largest),
            # the output's own rounding, fp32's sums
            tol = (2 ** -10 + 2 ** -17) * size + 2 ** -24 * v.abs().amax((1, 2))[:, None]
            tol = tol + O.half_step(dt) * (want.abs() + tol)
            assert ((out[i].double().cpu() - want).abs() <= tol).all()
