"""attention_kv4: rows of no sequence and of sequences that are left out."""

import math

import pytest
import torch

import paged_oracle as O
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P
from test_paged_gpu import _check, _problem, _tiles, _wide

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def _dirty(q):
    """Leaves NaN in memory that the allocator hands out next."""
    a = torch.full_like(q, math.nan, device="cuda")
    b = torch.full(q.shape[:2], math.nan, device="cuda")
    torch.cuda.synchronize()
    del a, b


def _call(args, most, out=None):
    got, lse = P.attention_kv4(*args, *([most] if len(args) > 4 else []), out=out, return_lse=True)
    torch.cuda.synchronize()
    return got, lse


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("seqs,first,wide", [
    ([(1, 40), (1, 0), (1, 300)], 0, False),             # without query_start
    ([(3, 40), (0, 7), (5, 300)], 2, False),
    ([(40, 140), (0, 7), (33, 300)], 3, True),
])
def test_rows_of_no_sequence(dt, given, seqs, first, wide):
    hq, h, bs = 8, 2, 16
    most = max(n for n, _ in seqs)
    q, cache, table, lens, start = _problem(
        seqs, hq, h, bs, 64, dt, 5, spare_rows=first + 70,
        cols_more=_wide(most, len(seqs), hq, h) if wide else 2)
    start += first
    assert _tiles(table, most, hq, h, bs) == wide
    plain = most == 1
    args = [x.cuda() for x in ((q, cache, table, lens) if plain else (q, cache, table, lens, start))]
    _dirty(q)
    out, lse = _call(args, most, torch.full_like(q, 9.0).cuda() if given else None)
    K.check_device_error(out.device)
    _check(out, lse, O.attend(q, cache, table, lens, None if plain else start, tiles=wide), dt)
    rows = torch.ones(q.shape[0], dtype=torch.bool)
    rows[0 if plain else int(start[0]):len(seqs) if plain else int(start[-1])] = False
    assert rows.sum() == first + 70
    assert (out[rows.cuda()] == (9.0 if given else 0.0)).all()
    assert (lse[rows.cuda()] == -math.inf).all()


@pytest.mark.parametrize("given", [False, True])
@pytest.mark.parametrize("rows", [1, 4, 40])
def test_rows_of_a_sequence_that_is_left_out(rows, given):
    dt, hq, h, bs = BF, 8, 2, 16
    wide = rows == 40
    seqs = [(rows, 90), (rows, 150), (rows, 60)]
    q, cache, table, lens, start = _problem(seqs, hq, h, bs, 64, dt, 6,
                                            cols_more=_wide(rows, 3, hq, h) if wide else 2)
    args = [x.cuda() for x in ((q, cache, table, lens) if rows == 1 else
                               (q, cache, table, lens, start))]
    for bad in (-1, table.shape[1] * bs + 1):  # lengths that do not fit
        args[3][1] = bad
        _dirty(q)
        out, lse = _call(args, rows, torch.full_like(q, 9.0).cuda() if given else None)
        assert K.read_device_error(out.device) == 3
        gone = slice(rows, 2 * rows)
        assert (out[gone] == (9.0 if given else 0.0)).all() and (lse[gone] == -math.inf).all()
        for r in (0, 2):
            at = slice(r * rows, (r + 1) * rows)
            ref = O.attend(q[at], cache, table[r:r + 1], lens[r:r + 1],
                           torch.tensor([0, rows]), tiles=wide)
            _check(out[at], lse[at], ref, dt)
    if rows > 1:  # more rows than max_query_len
        args[3][1] = 150
        args[4][1] += 1
        out, lse = _call(args, rows)
        assert K.read_device_error(out.device) == 3
        assert (out[:rows + 1] == 0).all() and (lse[:rows + 1] == -math.inf).all()
        assert out[rows + 1:].isfinite().all() and lse[rows + 1:].isfinite().all()


def test_no_sequences():
    q = torch.zeros((3, 4, 128), dtype=BF, device="cuda")
    cache = P.kv4_cache(2, 2)
    none = torch.zeros((0,), dtype=torch.int32, device="cuda")
    _dirty(q)
    out, lse = P.attention_kv4(q, cache, none.view(0, 2), none, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()
    kept = torch.full_like(q, 9.0)
    assert P.attention_kv4(q, cache, none.view(0, 2), none, out=kept) is kept
    assert (kept == 9.0).all()


@pytest.mark.parametrize("rows", [3, 40])
def test_starts_out_of_order(rows):
    """A sequence that ends in front of its beginning is left out; the others keep their rows."""
    dt, hq, h, bs = BF, 8, 2, 16
    wide = rows == 40
    q, cache, table, lens, start = _problem([(rows, 90)] * 4, hq, h, bs, 64, dt, 8,
                                            cols_more=_wide(rows, 4, hq, h) if wide else 2)
    start = torch.tensor([rows, 2 * rows, 4 * rows, 3 * rows, 2 * rows]).int()
    for _ in range(3):
        out, lse = _call([x.cuda() for x in (q, cache, table, lens, start)], rows)
        assert K.read_device_error(out.device) == 3  # sequence 1 is too long, 2 and 3 end early
        ref = O.attend(q[rows:2 * rows], cache, table[:1], lens[:1], torch.tensor([0, rows]),
                       tiles=wide)
        _check(out[rows:2 * rows], lse[rows:2 * rows], ref, dt)
        for at in (slice(0, rows), slice(2 * rows, 4 * rows)):
            assert (out[at] == 0).all() and (lse[at] == -math.inf).all()
    # sequence 1 names rows of sequence 0 and of 2, which keep their results
    start = torch.tensor([0, rows, 4 * rows, rows, 2 * rows]).int()
    out, lse = _call([x.cuda() for x in (q, cache, table, lens, start)], rows)
    assert K.read_device_error(out.device) == 3
    for r, at in ((0, slice(0, rows)), (3, slice(rows, 2 * rows))):
        ref = O.attend(q[at], cache, table[r:r + 1], lens[r:r + 1], torch.tensor([0, rows]),
                       tiles=wide)
        _check(out[at], lse[at], ref, dt)
    assert (out[2 * rows:] == 0).all() and (lse[2 * rows:] == -math.inf).all()


@pytest.mark.parametrize("n", [0, 1, 13, 20])
def test_query_rows_behind_the_slots(n):
    q = torch.randn((20, 3, 128), generator=torch.Generator().manual_seed(n)).to(BF).cuda()
    kv = torch.zeros((20, 2, 128), dtype=BF, device="cuda")
    cache = torch.zeros((2, 4, 16, 2, 128), dtype=BF, device="cuda")
    slots = torch.arange(n, device="cuda")
    table = torch.rand((64, 128), device="cuda")
    _dirty(q)
    out = P.append_kv(cache, kv, kv, slots, slots, table, q)
    want, _ = O.rotate(q[:n], table, slots, False)
    assert ((out[:n].double().cpu() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -20).all()
    assert (out[n:] == 0).all()
    kept = torch.full_like(q, 9.0)
    P.append_kv(cache, kv, kv, slots, slots, table, q, query_out=kept)
    assert torch.equal(kept[:n], out[:n]) and (kept[n:] == 9.0).all()


@pytest.mark.parametrize("four", [False, True])
def test_queries_are_rotated_when_there_are_no_kv_heads(four):
    """A rank that holds no kv head of its own still gets its queries."""
    q = torch.randn((5, 3, 128), generator=torch.Generator().manual_seed(3)).to(BF).cuda()
    kv = torch.zeros((5, 0, 128), dtype=BF, device="cuda")
    cache = P.kv4_cache(4, 0) if four else torch.zeros((2, 4, 16, 0, 128), dtype=BF, device="cuda")
    pos = torch.arange(5, device="cuda")
    table = torch.rand((64, 128), device="cuda")
    _dirty(q)
    out = P.append_kv(cache, kv, kv, pos, pos, table, q)
    K.check_device_error(out.device)
    want, _ = O.rotate(q, table, pos, False)
    assert ((out.double().cpu() - want).abs() <= 2 ** -8 * want.abs() + 2 ** -20).all()
    assert P.append_kv(cache, kv, kv, pos) is None


@pytest.mark.parametrize("rows", [1, 40])
def test_lengths_that_ints_cannot_walk(rows):
    """A table wide enough for 2^31 tokens; a length near that is refused as one that does not fit."""
    q = torch.ones((rows, 4, 128), dtype=BF, device="cuda")
    cache = P.kv4_cache(2, 2)
    table = torch.zeros((1, 2 ** 27), dtype=torch.int32, device="cuda")
    start = torch.tensor([0, rows]).int().cuda()
    for n in (2 ** 31 - 1, 2 ** 31 - 2 ** 16 + 1):
        out, lse = _call((q, cache, table, torch.tensor([n]).int().cuda(), start), rows)
        assert K.read_device_error(out.device) == 3
        assert (out == 0).all() and (lse == -math.inf).all()
    out, lse = _call((q, cache, table, torch.tensor([rows + 9]).int().cuda(), start), rows)
    K.check_device_error(out.device)
    seen = torch.arange(10, 10 + rows).double()[:, None].log().expand(rows, 4)
    assert (out == 0).all() and ((lse.double().cpu() - seen).abs() < 2 ** -18).all()
