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


@pytest.mark.parametrize("rows", [1, 40])
def test_large_values_under_small_scores(rows):
    """Values 2^130 times the others' under weights of 2^-122, which fp32 holds: the result is
    theirs.  Tokens 128 to 159 are the second step of the warp that has taken tokens 0 to 31."""
    q, cache, table, lens, start = _one(rows, 160)
    q[:] = 1
    cache[:, :, :16] = 0
    cache[:, :, 32, 0] = 127
    cache[:, :, 32, 1] = 17   # 2^-110
    late = table[0, 8:10].long()
    cache[late, :, :16] = 0xCF  # -7.5: a score of -84.9
    cache[late, :, 32, 1] = 147
    ref = O8.attend(q, cache, table, lens, start, causal=False)
    _check(*_attend(q, cache, table, lens, start, rows, causal=False), ref, BF)


@pytest.mark.parametrize("rows", [1, 9, 40])
@pytest.mark.parametrize("up", [0, 5, 13, 27, 53])
def test_equal_scores_of_any_size_over_values_of_many_scales(rows, up):
    """Equal keys (as codes of 1 and of 2 under half the scale), scores of 2^4 to 2^110: every token
    weighs the same, whatever its values' scale (2^0, 2^-6, 2^-30, and zeros) and its score's size."""
    n, hq, h = 400, 8, 2
    q, cache, table, lens, start = _one(rows, n)
    q = (2.0 ** up * (1 + q.double().abs())).to(BF)
    odd = (torch.arange(25) % 2).to(torch.uint8)
    value = torch.tensor([127, 121, 97, 17], dtype=torch.uint8)[torch.arange(25) * 7 // 5 % 4]
    used = table[0, :25].long()
    cache[used, :, :16] = (0x38 + 8 * odd)[:, None, None, None]
    cache[used, :, 32, 0] = (127 + up - odd)[:, None]
    cache[used, :, 32, 1] = value[:, None]
    cache[used[value == 17], :, 16:32] = 0
    out, _ = _attend(q, cache, table, lens, start, rows)
    t = torch.arange(n)
    x = O8.read(cache, table[0].long()[t // 16] * 16 + t % 16)[1]  # [n, h, 128]
    for i in range(rows):
        v = x[:n - rows + i + 1].repeat_interleave(hq // h, 1)
        want, size = v.mean(0), v.abs().mean(0)
        # weights to fp16 (those 2^-30 below go under: 2^-24 of the largest), fp32's sums, the output
        tol = (2 ** -11 + 2 ** -17) * size + 2 ** -24 * v.abs().amax((0, 2))[:, None]
        tol = tol + O8.half_step(BF) * (want.abs() + tol)
        assert ((out[i].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("rows", [5, 40])
@pytest.mark.parametrize("times", [300, 1000])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_a_query_channel_far_above_the_others(dt, times, rows):
    """A bias makes one channel of the queries large, that channel is small in the keys: the scores
    are the others'.  The kernel for many rows takes a row, scaled to at most 448, in parts that
    are exact but for elements below 2^-6, which are off by 2^-14 (bf16) or 2^-17 (fp16) at most:
    added to the tolerance, element by element."""
    hq, h, scale = 8, 2, 1 / math.sqrt(128)
    q, cache, table, lens, start = _one(rows, 300, dt, hq, h)
    q[:, :, 5] = (q[:, :, 5].double() * times).to(dt)
    cache[:, :, :16, 5] %= 5  # up to 2^-7, where the others are 40 in the mean
    want, wlse, tol, ltol = O8.attend(q, cache, table, lens, start, scale, one_part=rows > 9 or None)
    if rows > 9:
        up = torch.ceil(torch.log2(q.double().abs().amax(-1, keepdim=True) / 448))
        off = 2.0 ** up * (2 ** -14 if dt == BF else 2 ** -17)
        off = off * (q.double().abs() < 2.0 ** (up - 6))            # [T, hq, 128]
        t = torch.arange(300)
        k = O8.read(cache, table[0].long()[t // 16] * 16 + t % 16)[0].abs()  # [300, h, 128]
        move = 2 * scale * torch.einsum("thgd,lhd->thgl", off.view(rows, h, hq // h, 128), k)
        move = move.amax(-1).reshape(rows, hq)                     # of a weight, at most
        size = cache.clone()
        size[:, :, 16:32] &= 0x7F
        of_values = O8.attend(q, size, table, lens, start, scale)[0]  # sum of p |v|
        tol, ltol = tol + move[..., None] * of_values, ltol + move
    _check(*_attend(q, cache, table, lens, start, rows, scale=scale), (want, wlse, tol, ltol), dt)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("up", [101, 112, 125])
def test_queries_near_the_largest_number(rows, up):
    """bf16 queries of 2^101 and more over keys of 2^-100."""
    q, cache, table, lens, start = _one(rows, 200)
    q = (q.double().clamp(-3, 3) * 2.0 ** up).to(BF)
    cache[:, :, 32, 0::2] = (cache[:, :, 32, 0::2].int() - 100).to(torch.uint8)
    scale = 2.0 ** (100 - up - 8) / math.sqrt(128)
    ref = O8.attend(q, cache, table, lens, start, scale)
    _check(*_attend(q, cache, table, lens, start, rows, scale=scale), ref, BF)


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_an_infinite_query_is_not_a_number(dt, rows):
    """Whatever the keys' signs are in its channel: scores of -inf alone are no row without tokens."""
    q, cache, table, lens, start = _one(rows, 100, dt)
    cache[:, :, :16, 9] |= 0x80
    cache[:, :, :16, 9] = cache[:, :, :16, 9].clamp(0x88, 0xF0)  # negative, not zero
    ref = O8.attend(q, cache, table, lens, start, one_part=True)
    q[0, 1, 9], q[rows - 1, 6, 9] = math.inf, -math.inf
    out, lse = _attend(q, cache, table, lens, start, rows)
    bad = torch.zeros(out.shape[:2], dtype=torch.bool)
    bad[0, 1] = bad[rows - 1, 6] = True
    assert out.cpu()[bad].isnan().all() and lse.cpu()[bad].isnan().all()
    want = ref[0].clone()
    want[bad] = math.nan
    _check(out, None, (want, *ref[1:]), dt)


@pytest.mark.parametrize("rows", [1, 40])
def test_a_cache_without_blocks(rows):
    """Sequences of no tokens are zeros; one that names a block records an error."""
    cache = P.kv8_cache(0, 2)
    table = torch.zeros((2, _wide(40, 2, 8, 2)), dtype=torch.int32)
    assert _tiles(table, rows, 8, 2, 16) == (rows == 40)
    q = torch.randn((2 * rows, 8, 128), generator=torch.Generator().manual_seed(1)).to(BF)
    start = torch.tensor([0, rows, 2 * rows]).int()
    for n in (0, 30):
        out, lse = P.attention_kv8(q.cuda(), cache, table.cuda(), torch.tensor([0, n]).int().cuda(),
                                   start.cuda(), rows, return_lse=True)
        if n:
            with pytest.raises(RuntimeError):
                K.check_device_error(out.device)
        else:
            K.check_device_error(out.device)
        assert not out.any() and (lse == -math.inf).all()
