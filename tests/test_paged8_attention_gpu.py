"""Attention over an 8-bit paged cache against a plain 64-bit form (paged8_oracle.attend derives
the tolerance)."""

import math

import pytest
import torch

import paged8_oracle as O8
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _no_device_error():
    K.check_device_error(torch.device("cuda", 0), "before the test")
    yield
    torch.cuda.synchronize()


def _check(out, lse, ref, dt):
    want, wlse, tol, ltol = ref
    has = ~want.isnan()
    o = out.double().cpu()
    bound = (tol + O8.half_step(dt) * (want.abs() + tol)
             + torch.finfo(dt).eps * torch.finfo(dt).tiny)
    # past the type's largest number a result rounds to infinity
    most = torch.finfo(dt).max * (1 + O8.half_step(dt))
    over = has & (want.abs() - bound > most)
    assert (o[over] == want[over].sign() * math.inf).all()
    near = has & ~over & ~((want.abs() + bound > most) & o.isinf())
    has = near
    worst = ((o - want).abs() / bound)[has].nan_to_num(nan=math.inf).max() if has.any() else 0
    assert worst <= 1, f"{float(worst):.3g} of the tolerance"
    if lse is not None:
        rows = ~wlse.isnan()
        l = lse.double().cpu()[rows]
        assert torch.equal(l == -math.inf, wlse[rows] == -math.inf)
        fin = wlse[rows] > -math.inf
        assert ((l - wlse[rows]).abs()[fin] <= ltol[rows][fin]).all()


def _problem(seqs, hq, h, bs, dt, seed, spare_rows=0, cols_more=2, spread=2):
    """seqs: (query rows, cached tokens) of each sequence."""
    g = torch.Generator().manual_seed(seed)
    need = [(n + bs - 1) // bs for _, n in seqs]
    cols = max(need) + cols_more
    nb = sum(need) + 3
    perm = torch.randperm(nb, generator=g).int()
    table = torch.full((len(seqs), cols), -7, dtype=torch.int32)  # unused entries: not read
    at = 0
    for r, c in enumerate(need):
        table[r, :c] = perm[at:at + c]
        at += c
    cache = O8.random_cache(g, nb, h, bs, spread)
    T = sum(n for n, _ in seqs) + spare_rows
    q = (torch.randn((T, hq, 128), generator=g) * 0.7).to(dt)
    start = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).int()
    lens = torch.tensor([n for _, n in seqs]).int()
    return q, cache, table, lens, start


def _tiles(table, rows, hq, h, bs):
    """Whether a call takes the kernel for many rows, going by what the host knows: rows a kv
    head, and rows times tokens that the table has room for."""
    rows *= hq // h
    return rows > 64 and rows * h * table.numel() * bs > 3 << 20


def _wide(rows, seqs, hq, h, bs=16):
    """Table columns that take a call of few tokens there all the same."""
    return (4 << 20) // (rows * (hq // h) * h * seqs * bs) + 1


def _attend(q, cache, table, lens, start=None, most=1, **kw):
    got = P.attention_kv8(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(),
                          None if start is None else start.cuda(), most, return_lse=True, **kw)
    torch.cuda.synchronize()
    K.check_device_error(torch.device("cuda", 0))
    return got


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hq,h,bs", [(7, 1, 16), (8, 8, 32), (28, 4, 16), (16, 1, 64), (48, 2, 48),
                                     (20, 1, 1024), (40, 1, 16)])
def test_one_token(dt, hq, h, bs):
    lens = [1, 15, 16, 17, 0, 31, 32, 33, 127, 128, 129, 400, 2]
    q, cache, table, lens, _ = _problem([(1, n) for n in lens], hq, h, bs, dt, hq + bs)
    ref = O8.attend(q, cache, table, lens, None)
    _check(*_attend(q, cache, table, lens), ref, dt)


SEVERAL = [
    (5, 1, [(3, 3), (1, 70), (5, 64)]),
    (10, 2, [(2, 1), (4, 0), (0, 50), (7, 200), (1, 1)]),  # rows that see nothing, no rows
    (7, 1, [(130, 130), (33, 160)]),
    (8, 2, [(64, 300), (17, 17)]),
    (3, 3, [(100, 37)]),
    (8, 1, [(16, 500), (0, 30), (33, 0), (40, 129), (1, 128)]),
    (16, 2, [(300, 300), (5, 1000), (64, 64)]),
    (4, 4, [(65, 1111), (1, 1), (257, 256)]),
    (4, 2, [(7, 900), (8, 8)]),
]


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hq,h,seqs", SEVERAL)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("wide", [False, True])
def test_several_rows(dt, hq, h, seqs, causal, wide):
    most = max(n for n, _ in seqs)
    if wide and most * (hq // h) <= 64:
        pytest.skip("too few rows for the other kernel")
    q, cache, table, lens, start = _problem(
        seqs, hq, h, 16, dt, hq * 7, spare_rows=3,
        cols_more=_wide(most, len(seqs), hq, h) if wide else 2)
    tiles = _tiles(table, most, hq, h, 16)
    assert tiles or not wide
    out = torch.full_like(q, 9.0).cuda()
    got, lse = _attend(q, cache, table, lens, start, most, out=out, causal=causal)
    assert got is out
    ref = O8.attend(q, cache, table, lens, start, causal=causal, one_part=tiles or None)
    _check(out, lse, ref, dt)
    assert (out[int(start[-1]):] == 9.0).all()  # rows of no sequence
    got, lse = _attend(q, cache, table, lens, start, most, causal=causal)
    assert not got[int(start[-1]):].any() and (lse[int(start[-1]):] == -math.inf).all()


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("hq,h,rows,n", [(28, 4, 1, 9001), (8, 8, 1, 5003), (28, 4, 4, 7000),
                                         (8, 1, 7, 6007), (4, 4, 3, 8192), (28, 4, 150, 5000)])
def test_long_sequences_are_split(dt, hq, h, rows, n):
    q, cache, table, lens, start = _problem([(rows, n), (1, 40), (rows, 3000)], hq, h, 32, dt, n)
    tiles = _tiles(table, rows, hq, h, 32)
    ref = O8.attend(q, cache, table, lens, start, one_part=tiles or None)
    first = _attend(q, cache, table, lens, start, rows)
    _check(*first, ref, dt)
    again = _attend(q, cache, table, lens, start, rows)  # nothing depends on timing
    assert all(torch.equal(a, b) for a, b in zip(first, again))


@pytest.mark.parametrize("rows", [1, 5, 20, 40])
@pytest.mark.parametrize("dt", DTYPES)
def test_scales_far_apart(dt, rows):
    """Units whose scales are up to 2^40 apart: a row's weight may lie on small ones, beside
    others that it sees with none and others that it does not see at all."""
    g = torch.Generator().manual_seed(rows)
    q, cache, table, lens, start = _problem([(rows, 300), (rows, 200)], 8, 2, 16, dt, 91,
                                            cols_more=_wide(40, 2, 8, 2))
    tiles = _tiles(table, rows, 8, 2, 16)
    assert tiles == (rows == 40)
    up = torch.randint(-20, 20, (cache.shape[0], 2), generator=g)
    cache[:, :, 32, 1] = (cache[:, :, 32, 1] + up).to(torch.uint8)
    big = int(table[0, 18])  # the last tokens of sequence 0: only some rows see them
    cache[big, :, 32, 1] = 160
    huge = int(table[1, 2])  # keys that no row has weight on, with huge values
    cache[huge, :, :16] = torch.where(cache[huge, :, :16] >= 128, cache[huge, :, :16], 0)
    ref = O8.attend(q, cache, table, lens, start, one_part=tiles or None)
    _check(*_attend(q, cache, table, lens, start, rows), ref, dt)


@pytest.mark.parametrize("rows", [1, 30])
def test_weight_on_small_scales(rows):
    """All of a row's weight on a unit of tiny values, beside one of large ones without any."""
    dt = torch.bfloat16
    q, cache, table, lens, start = _problem([(rows, 96)], 4, 1, 16, dt, 92,
                                            cols_more=_wide(30, 1, 4, 1))
    assert _tiles(table, rows, 4, 1, 16) == (rows == 30)
    q[:] = 1
    blocks = table[0][:6].long()
    cache[blocks, :, :16] = 0x28 + 0x80           # keys: a small negative number
    cache[blocks[3], :, 5] = 0x60                 # but for one token
    cache[blocks, :, 32, 0] = 130
    cache[blocks, :, 32, 1] = 127 + 15
    cache[blocks[3], :, 32, 1] = 127 - 15
    ref = O8.attend(q, cache, table, lens, start)
    _check(*_attend(q, cache, table, lens, start, rows), ref, dt)


@pytest.mark.parametrize("rows", [1, 40])
def test_values_of_zero_count_in_the_sum(rows):
    """Units never written or of zeros, next to large ones: their tokens weigh as others do."""
    dt = torch.bfloat16
    q, cache, table, lens, start = _problem([(rows, 150), (rows, rows)], 8, 2, 16, dt, 44,
                                            cols_more=_wide(40, 2, 8, 2))
    assert _tiles(table, rows, 8, 2, 16) == (rows == 40)
    cache[:, :, 32, 1] += 40
    zero = table[0][2:9].long()  # tokens 32 to 143 of sequence 0
    cache[zero, :, 16:32] = 0
    cache[zero, :, 32, 1] = 17
    cache[zero[3]] = 0
    for scale in (0.1, 1e-37):
        ref = O8.attend(q, cache, table, lens, start, scale=scale)
        _check(*_attend(q, cache, table, lens, start, rows, scale=scale), ref, dt)


@pytest.mark.parametrize("rows", [9, 90])
@pytest.mark.parametrize("mag", [1e-30, 1e-6, 1e6, 1e30])
def test_magnitudes_and_scale(mag, rows):
    dt = torch.bfloat16
    q, cache, table, lens, start = _problem([(rows, 300), (2, 20)], 4, 2, 16, dt, 31,
                                            cols_more=_wide(90, 2, 4, 2))
    assert _tiles(table, rows, 4, 2, 16) == (rows == 90)
    byte = round(math.log2(mag))
    cache[:, :, 32, 0::2] = (cache[:, :, 32, 0::2].int() - byte).clamp(17, 247).to(torch.uint8)
    cache[:, :, 32, 1::2] = (cache[:, :, 32, 1::2].int() + byte).clamp(17, 247).to(torch.uint8)
    q = (q.double() * mag).to(dt)
    for scale in (-0.11, 0.3):
        ref = O8.attend(q, cache, table, lens, start, scale=scale)
        _check(*_attend(q, cache, table, lens, start, rows, scale=scale), ref, dt)


@pytest.mark.parametrize("rows", [1, 9, 30, 64])
def test_not_a_number_reaches_those_that_see_it(rows):
    """NaN codes behind the length, in blocks of no sequence and behind a row's own position
    change nothing; one in a value that a row sees is NaN in that channel, one in a key in all."""
    dt, hq, h = torch.bfloat16, 8, 2
    q, cache, table, lens, start = _problem([(rows, 203), (rows, 100), (rows, 64)], hq, h, 16, dt,
                                            rows + 50, cols_more=_wide(30, 3, hq, h))
    assert _tiles(table, rows, hq, h, 16) == (rows >= 30)
    used = torch.zeros(cache.shape[0], dtype=torch.bool)
    for r, n in enumerate(lens.tolist()):
        used[table[r, :(n + 15) // 16].long()] = True
    cache[~used] = 255
    last = int(table[0, 12])  # tokens 192 to 202 of sequence 0, nothing behind
    cache[last, :, 11:16] = 127
    cache[last, :, 27:32] = 255
    clean = cache.clone()
    v_tok = 202                                  # the last token: only the last row sees it
    cache[last, 1, 16 + v_tok % 16, 77] = 0x7F
    cache[int(table[1, 0]), 0, 16 + 3, 5] = 0xFF  # token 3 of sequence 1, which all rows see
    cache[int(table[2, 3]), 0, 15, 9] = 0x7F      # the last token's key of sequence 2
    ref = O8.attend(q, clean, table, lens, start)
    out, lse = _attend(q, cache, table, lens, start, rows)
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[rows - 1, 4:, 77] = True
    bad[rows:2 * rows, :4, 5] = True
    bad[3 * rows - 1, :4] = True
    assert torch.equal(out.cpu().isnan(), bad)
    want = ref[0].clone()
    want[bad] = math.nan
    _check(out, None, (want, *ref[1:]), dt)
    fine = torch.ones(lse.shape, dtype=torch.bool)
    fine[3 * rows - 1, :4] = False
    assert ((lse.double().cpu() - ref[1]).abs() <= ref[3])[fine].all()


def test_bad_blocks_and_extents():
    """A block id outside the cache hides its tokens; a sequence that does not fit is left out."""
    dt = torch.bfloat16
    q, cache, table, lens, start = _problem([(3, 90), (3, 40), (3, 70)], 4, 2, 16, dt, 77)
    ref = O8.attend(q, cache, table, lens, start)

    def call(t, n, st):
        got = P.attention_kv8(q.cuda(), cache.cuda(), t.cuda(), n.cuda(), st.cuda(), 3,
                              return_lse=True)
        with pytest.raises(RuntimeError):
            K.check_device_error(torch.device("cuda", 0))
        return got

    far = table.clone()
    far[0, 1] = cache.shape[0]  # tokens 16 to 31
    far[2, 4] = -1              # tokens 64 to 69: the last rows'
    out, lse = call(far, lens, start)
    keep = torch.tensor([i for i in range(90) if not 16 <= i < 32])
    k64 = O8.read(cache, table[0].long()[torch.arange(90) // 16] * 16 + torch.arange(90) % 16)
    for i in range(3):
        mine = keep[keep < 88 + i]
        for hq in range(4):
            w = k64[0, mine, hq // 2] @ q[i, hq].double() / math.sqrt(128)
            want = torch.softmax(w, 0) @ k64[1, mine, hq // 2]
            assert (out[i, hq].double().cpu() - want).abs().max() <= 2 ** -7 * want.abs().max()
    _check(out[3:6], lse[3:6], [x[3:6] for x in ref], dt)
    for n, st in ((torch.tensor([90, 10 ** 6, 70]), start), (torch.tensor([90, -1, 70]), start),
                  (lens, torch.tensor([0, 3, 7, 10])), (lens, torch.tensor([0, 3, 2, 9]))):
        out, lse = call(table, n.int(), st.int())
        _check(out[:3], lse[:3], [x[:3] for x in ref], dt)


def test_more_sequences_than_threads():
    g = torch.Generator().manual_seed(3)
    for first in (1, 6, 30):
        seqs = [(int(n > 0), n) for n in torch.randint(0, 60, (700,), generator=g).tolist()]
        seqs[3], seqs[650] = (0, 25), (first, 77)
        q, cache, table, lens, start = _problem(seqs, 4, 1, 16, torch.bfloat16, first)
        assert _tiles(table, first, 4, 1, 16) == (first == 30)
        ref = O8.attend(q, cache, table, lens, start)
        _check(*_attend(q, cache, table, lens, start, first), ref, torch.bfloat16)


def test_strides_and_empty_calls():
    dt = torch.float16
    q, cache, table, lens, start = _problem([(2, 50), (3, 90)], 6, 2, 16, dt, 5)
    ref = O8.attend(q, cache, table, lens, start)
    wide = torch.zeros((5, 10, 128), dtype=dt).cuda()
    wide[:, 2:8] = q.cuda()
    big = torch.full((2 * cache.shape[0], 4, 33, 128), 255, dtype=torch.uint8).cuda()
    big[::2, 1:3] = cache.cuda()
    cols = torch.full((2, 2 * table.shape[1]), -3, dtype=torch.int32).cuda()
    cols[:, ::2] = table.cuda()
    out = torch.zeros((5, 9, 128), dtype=dt).cuda()
    got, lse = P.attention_kv8(wide[:, 2:8], big[::2, 1:3], cols[:, ::2], lens.cuda(),
                               start.cuda(), 3, out=out[:, 3:], return_lse=True)
    _check(got, lse, ref, dt)
    assert not out[:, :3].any()
    hm = cache.cuda().transpose(0, 1).contiguous().transpose(0, 1)  # heads outermost
    _check(P.attention_kv8(q.cuda(), hm, table.cuda(), lens.cuda(), start.cuda(), 3), None, ref, dt)
    one = cache[:1].cuda()
    few = P.attention_kv8(q[:1].cuda(), one, torch.zeros((1, 1), dtype=torch.int32).cuda(),
                          torch.tensor([7]).int().cuda())
    t0 = torch.zeros((1, 1), dtype=torch.int32)
    _check(few, None, O8.attend(q[:1], cache[:1], t0, torch.tensor([7]), None), dt)
    none = P.attention_kv8(q.cuda(), cache.cuda(), table[:0].cuda(), lens[:0].cuda(),
                           torch.zeros(1, dtype=torch.int32).cuda())
    assert not none.any()
    K.check_device_error(out.device)


@pytest.mark.parametrize("dt", DTYPES)
def test_a_step_as_it_is_used(dt):
    """Append (rotated), attend, read: prompts in chunks, then single tokens; the cache attended
    over is the one read back."""
    g = torch.Generator().manual_seed(12)
    hq, h, bs, maxpos = 8, 2, 16, 400
    cache = P.kv8_cache(40, h, bs)
    table = torch.randperm(40, generator=g)[:36].view(2, 18).int()
    ang = torch.arange(maxpos).double()[:, None] / 1e4 ** (torch.arange(0, 128, 2).double() / 128)
    cs = torch.cat([ang.cos(), ang.sin()], 1).float().cuda()
    lens = torch.zeros(2, dtype=torch.int64)
    for rows in ([37, 64], [50, 5], [1, 1], [1, 1], [1, 0], [0, 1], [1, 1]):
        pos = torch.cat([lens[r] + torch.arange(n) for r, n in enumerate(rows)])
        seq = torch.cat([torch.full((n,), r) for r, n in enumerate(rows)])
        slots = table[seq, pos // bs].long() * bs + pos % bs
        T = len(pos)
        q, k, v = (torch.randn((T, x, 128), generator=g).to(dt).cuda() for x in (hq, h, h))
        lens += torch.tensor(rows)
        start = torch.tensor([0] + rows).cumsum(0).int()
        q = P.append_kv(cache, k, v, slots.cuda(), pos.cuda(), cs, q)
        back = P.read_kv8(cache, slots.cuda(), dt)
        assert ((back[1] - v).abs().float() <= 2 ** -4 * v.abs().float() + 2 ** -6).all()
        out, lse = _attend(q, cache, table, lens.int(), start, max(rows))
        ref = O8.attend(q.cpu(), cache.cpu(), table, lens, start)
        _check(out, lse, ref, dt)
