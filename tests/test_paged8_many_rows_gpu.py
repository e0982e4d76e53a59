"""attention_kv8's kernel for many query rows, where its own bounds and addresses are at stake: block
ids out of range, sequences that do not fit, views, results in the queries' place, shared blocks."""

import math

import pytest
import torch

import paged8_oracle as O8
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P
from test_paged8_attention_gpu import _attend, _check, _problem, _tiles, _wide

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_device_error():
    K.check_device_error(torch.device("cuda", 0), "before the test")
    yield
    torch.cuda.synchronize()


def _many(seqs, hq, h, dt, seed, bs=16, spare_rows=0):
    most = max(n for n, _ in seqs)
    p = _problem(seqs, hq, h, bs, dt, seed, spare_rows, _wide(most, len(seqs), hq, h, bs))
    assert _tiles(p[2], most, hq, h, bs)
    return p


def _fails(q, cache, table, lens, start, most, **kw):
    got = P.attention_kv8(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(), most,
                          return_lse=True, **kw)
    with pytest.raises(RuntimeError):
        K.check_device_error(got[0].device)
    return got


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("causal", [True, False])
def test_bad_blocks(dt, causal):
    """Block ids outside the cache hide their tokens: one in the middle of a half of 64 tokens, four
    that are a half, in an item that CTAs share, the last ones, all of a sequence's."""
    seqs, hq, h = [(90, 5003), (90, 333), (40, 200), (33, 90)], 4, 2
    q, cache, table, lens, start = _many(seqs, hq, h, dt, 13)
    nb = cache.shape[0]
    bad = [[1, 100, 200, 201, 202, 203], [3], [9], []]  # in front of every row's limit
    if not causal:
        bad[0].append(312), bad[1].append(20)           # the last blocks, in part
        bad[2] = list(range(13))
    far, packed, left = table.clone(), table.clone(), lens.clone()
    for r, pages in enumerate(bad):
        n = int(lens[r])
        for i, page in enumerate(pages):
            far[r, page] = [nb, -1, 2 ** 31 - 1][i % 3]
            left[r] -= min(16, n - 16 * page)
        keep = [i for i in range((n + 15) // 16) if i not in pages]
        packed[r, :len(keep)] = table[r, keep]
    # the sequences without what is hidden: the blocks kept are whole but for the last
    ref = O8.attend(q, cache, packed, left, start, causal=causal, one_part=True)
    out, lse = _fails(q, cache, far, lens, start, 90, causal=causal)
    _check(out, lse, ref, dt)
    if not causal:
        assert not out[180:220].any() and (lse[180:220] == -math.inf).all()


@pytest.mark.parametrize("given", [False, True])
def test_sequences_that_do_not_fit(given):
    dt, most = BF, 90
    seqs = [(90, 400), (90, 300), (70, 150)]
    q, cache, table, lens, start = _many(seqs, 4, 2, dt, 17, spare_rows=5)
    room = table.shape[1] * 16
    for n, st, fine in (([400, room + 1, 150], [0, 90, 180, 250], [0, 2]),
                        ([400, -1, 150], [0, 90, 180, 250], [0, 2]),
                        ([400, 300, 150], [0, 90, 181, 250], [0, 2]),    # a row too many
                        ([400, 300, 150], [0, 90, 180, 256], [0, 1]),    # behind the rows
                        ([400, 300, 150], [0, 90, 80, 150], [0, 2])):    # backwards
        n, st = torch.tensor(n).int(), torch.tensor(st).int()
        held = torch.full_like(q, 7.0).cuda()
        out, lse = _fails(q, cache, table, n, st, most, out=held if given else None)
        rows = torch.zeros(q.shape[0], dtype=torch.bool)
        for r in fine:
            a, b = int(st[r]), int(st[r + 1])
            one = O8.attend(q[a:b], cache, table[r:r + 1], n[r:r + 1], torch.tensor([0, b - a]))
            if not any(int(st[o]) < b and int(st[o + 1]) > a for o in fine if o != r):
                _check(out[a:b], lse[a:b], one, dt)
            rows[a:b] = True
        assert (out.cpu()[~rows] == (7.0 if given else 0.0)).all()
        assert (lse.cpu()[~rows] == -math.inf).all()


@pytest.mark.parametrize("bs", [16, 48, 128])
def test_views(bs):
    """Queries, caches, tables and results that are slices of larger ones; heads outermost."""
    dt = FP
    q, cache, table, lens, start = _many([(40, 150), (50, 390)], 6, 2, dt, 5, bs)
    ref = O8.attend(q, cache, table, lens, start, one_part=True)
    T = len(q)
    wide = torch.zeros((T, 10, 128), dtype=dt).cuda()
    wide[:, 2:8] = q.cuda()
    big = torch.full((2 * cache.shape[0], 4, 2 * bs + 1, 128), 255, dtype=torch.uint8).cuda()
    big[::2, 1:3] = cache.cuda()
    cols = torch.full((2, 2 * table.shape[1]), -3, dtype=torch.int32).cuda()
    cols[:, ::2] = table.cuda()
    out = torch.zeros((T, 9, 128), dtype=dt).cuda()
    got, lse = P.attention_kv8(wide[:, 2:8], big[::2, 1:3], cols[:, ::2], lens.cuda(), start.cuda(), 50,
                               out=out[:, 3:], return_lse=True)
    K.check_device_error(out.device)
    _check(got, lse, ref, dt)
    assert not out[:, :3].any()
    hm = cache.cuda().transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    again, _ = _attend(q, hm, table, lens, start, 50)
    assert torch.equal(again, got)


def test_in_place():
    """The output may be the query itself, in items that CTAs share too."""
    q, cache, table, lens, start = _many([(90, 90), (40, 6000)], 4, 2, BF, 21)
    want, _ = _attend(q, cache, table, lens, start, 90)
    own = q.cuda()
    assert P.attention_kv8(own, cache.cuda(), table.cuda(), lens.cuda(), start.cuda(), 90,
                           out=own) is own
    assert torch.equal(own, want)
    _check(want, None, O8.attend(q, cache, table, lens, start), BF)


@pytest.mark.parametrize("rows", [1, 40])
def test_sequences_that_share_blocks(rows):
    """A prefix in the same blocks for all, and one block twice in a sequence."""
    seqs, hq, h = [(rows, 200), (rows, 150), (rows, 333)], 8, 2
    q, cache, table, lens, start = (_many(seqs, hq, h, BF, 23) if rows > 9
                                    else _problem(seqs, hq, h, 16, BF, 23))
    table[1:, :5] = table[0, :5]
    table[2, 11] = table[2, 7]
    ref = O8.attend(q, cache, table, lens, start)
    _check(*_attend(q, cache, table, lens, start, rows), ref, BF)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("rows", [1, 9, 40])
def test_a_score_is_an_fp32_sum(dt, rows):
    """Rows that see one token: their logarithm is the score.  The matrix instructions' sums were
    measured off by at most 2^-21.9 of the sum of magnitudes; held to twice that.  The factor, the
    exponential, the logarithm and the way back add some ten roundings, 2^-20 of the score and of 1."""
    hq, h, n = 8, 2, 50
    g = torch.Generator().manual_seed(rows)
    seqs = [(rows, 1)] * n
    q, cache, table, lens, start = (_many(seqs, hq, h, dt, 29) if rows > 9
                                    else _problem(seqs, hq, h, 16, dt, 29))
    sign = torch.randint(0, 2, q.shape, generator=g) * 2 - 1  # 2^-4 to 1, which the parts hold exactly
    q = (sign * torch.exp2(-4 * torch.rand(q.shape, generator=g, dtype=torch.float64))).to(dt)
    out, lse = _attend(q, cache, table, lens, start, rows, causal=False)
    k, v = O8.read(cache, table[:, 0].long() * 16)  # [n, h, 128]
    seq = torch.arange(n).repeat_interleave(rows)
    k = k[seq].repeat_interleave(hq // h, 1)
    want = (q.double() * k).sum(-1) / math.sqrt(128)
    size = (q.double() * k).abs().sum(-1) / math.sqrt(128)
    tol = 2 ** -20.9 * size + 2 ** -20 * (want.abs() + 1)
    off = (lse.double().cpu() - want).abs()
    assert (off <= tol).all()
    v = v[seq].repeat_interleave(hq // h, 1)
    half = O8.half_step(dt) + (2 ** -11 if rows > 9 or dt == BF else 2 ** -21) + 2 ** -20
    assert ((out.double().cpu() - v).abs() <= half * v.abs() + 2 ** -24).all()
