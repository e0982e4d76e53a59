"""Paged-cache operators (rotated appends, 4-bit rows, attention over a 4-bit
cache) against plain 64-bit forms.

Tolerances are the roundings: half a step of the 16-bit type for a stored
value, fp32's for what is added up before it (paged_oracle.attend derives the
attention's).
"""

import math

import pytest
import torch

import paged_oracle as O
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16]


@pytest.fixture(autouse=True)
def _no_device_error():
    K.check_device_error(torch.device("cuda", 0), "before the test")
    yield
    torch.cuda.synchronize()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _table(maxpos, rd, dtype=torch.float32):
    ang = torch.arange(maxpos, dtype=torch.float64)[:, None] / 1e4 ** (
        torch.arange(0, rd, 2, dtype=torch.float64) / rd)
    return torch.cat([ang.cos(), ang.sin()], 1).to(dtype).cuda()


def _slots(n, nb, bs, g, holes=True):
    s = torch.randperm(nb * bs, generator=g)[:n]
    if holes and n > 3:
        s[1::5] = -1
    return s


def _layer(nb, bs, h, dt, form, g):
    """A paged layer of random bits: planes first or blocks first, token- or head-major."""
    x = torch.randn((2, nb, bs, h, 128), generator=g).to(dt)
    if form == "nhd":
        return x.cuda()
    if form == "hnd":
        return x.transpose(2, 3).contiguous().cuda().transpose(2, 3)
    return x.transpose(0, 1).contiguous().cuda()  # blocks first


# -------------------------------------------------------------------- append
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("form", ["nhd", "hnd", "blocks"])
@pytest.mark.parametrize("tokens,hq,h,rd,inter", [
    (1, 7, 1, 128, False), (5, 28, 4, 128, True), (33, 8, 8, 64, False), (300, 6, 2, 96, True),
    (40, 5, 5, 16, False), (64, 16, 2, 112, False)])
def test_append_16bit(dt, form, tokens, hq, h, rd, inter):
    g = _gen(tokens * 31 + rd)
    bs, nb, maxpos = 16, 23, 500
    cache = _layer(nb, bs, h, dt, form, g)
    before = cache.clone()
    qkv = torch.randn((tokens, hq + 2 * h, 128), generator=g).to(dt).cuda()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + h], qkv[:, hq + h:]
    slots = _slots(tokens, nb, bs, g)
    pos = torch.randint(0, maxpos, (tokens,), generator=g)
    table = _table(maxpos, rd, dt if tokens == 33 else torch.float32)
    idx = torch.int32 if tokens % 2 else torch.int64
    got = P.append_kv(cache, k, v, slots.to(idx).cuda(), pos.to(idx).cuda(), table, q,
                      interleaved=inter)
    torch.cuda.synchronize()
    K.check_device_error(cache.device)
    planes, old = ((c if form != "blocks" else c.transpose(0, 1)).cpu() for c in (cache, before))
    half = O.half_step(dt)

    def near(a, ref, mag):
        smallest = torch.finfo(dt).eps * torch.finfo(dt).tiny
        bound = half * ref.abs() * (1 + 2 ** -20) + 2 ** -23 * mag + smallest
        assert ((a.double().cpu() - ref).abs() <= bound).all()

    near(got, *O.rotate(q, table, pos, inter))
    keep = slots >= 0
    b, o = slots[keep] // bs, slots[keep] % bs
    ref, mag = O.rotate(k, table, pos, inter)
    near(planes[0][b, o], ref[keep], mag[keep])
    assert torch.equal(planes[1][b, o], v.cpu()[keep])
    for p in range(2):  # all other rows keep their bits
        old[p][b, o] = planes[p][b, o]
    assert torch.equal(planes, old)


def test_append_any_block_size_and_many_slots():
    """16-bit caches have no rule for the block size; enough tokens for four rows a group."""
    g = _gen(8)
    for bs, h, hq in ((7, 3, 5), (1, 2, 2), (24, 8, 32)):
        T = 3000
        nb = T // bs + 3
        cache = _layer(nb, bs, h, torch.float16, "nhd", g)
        k, v = (torch.randn((T, h, 128), generator=g).half().cuda() for _ in range(2))
        q = torch.randn((T, hq, 128), generator=g).half().cuda()
        slots = torch.randperm(nb * bs, generator=g)[:T]
        pos = torch.randint(0, 99, (T,), generator=g)
        for rd, inter in ((128, False), (48, False), (128, True)):
            table = _table(99, rd)
            out = P.append_kv(cache, k, v, slots.cuda(), pos.cuda(), table, q, interleaved=inter)
            for got, x in ((out, q), (cache[0].flatten(0, 1)[slots.cuda()], k)):
                ref, mag = O.rotate(x, table, pos, inter)
                bound = O.half_step(torch.float16) * ref.abs() * (1 + 2 ** -20) + \
                    2 ** -23 * mag + 2 ** -24
                assert ((got.double().cpu() - ref).abs() <= bound).all()
            assert torch.equal(cache[1].flatten(0, 1)[slots.cuda()], v)
    K.check_device_error(cache.device)


def test_append_plain_padded_and_in_place():
    g = _gen(3)
    cache = _layer(9, 16, 2, torch.bfloat16, "nhd", g)
    k = torch.randn((20, 2, 128), generator=g).bfloat16().cuda()
    v = torch.randn((20, 2, 128), generator=g).bfloat16().cuda()
    slots = torch.arange(30, 42).cuda()
    assert P.append_kv(cache, k, v, slots) is None  # no rotation, 12 of 20 rows
    assert torch.equal(cache[0].flatten(0, 1)[30:42], k[:12])
    assert torch.equal(cache[1].flatten(0, 1)[30:42], v[:12])
    # in place, halves whose partners lie in other lanes' chunks; rows behind the slots stay
    q = torch.randn((20, 3, 128), generator=g).bfloat16().cuda()
    want = P.append_kv(cache, k, v, slots, slots.int(), _table(64, 96), q.clone())
    inplace = q.clone()
    out = P.append_kv(cache, k, v, slots, slots.int(), _table(64, 96), inplace, query_out=inplace)
    assert out is inplace
    assert torch.equal(inplace[:12], want[:12]) and torch.equal(inplace[12:], q[12:])
    # unaligned and broadcast inputs
    odd = torch.randn(20 * 256 + 1, generator=g).bfloat16().cuda()[1:].view(20, 2, 128)
    one = torch.randn((1, 2, 128), generator=g).bfloat16().cuda().expand(20, 2, 128)
    P.append_kv(cache, odd, one, slots)
    assert torch.equal(cache[0].flatten(0, 1)[30:42], odd[:12])
    assert torch.equal(cache[1].flatten(0, 1)[30:42], one[:12])
    P.append_kv(cache, k[:0], v[:0], slots[:0])
    K.check_device_error(cache.device)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("g_size", [32, 64, 128])
@pytest.mark.parametrize("tokens,h,bs,rd", [(1, 1, 16, 128), (77, 4, 16, 128), (130, 3, 48, 64),
                                            (9, 2, 32, 0)])
def test_append_4bit(dt, g_size, tokens, h, bs, rd):
    g = _gen(tokens + g_size)
    nb = tokens // bs + 5
    cache = P.kv4_cache(nb, h, bs, g_size)
    cache.random_(0, 256)
    before = cache.cpu()
    k = torch.randn((tokens, h, 128), generator=g)
    k[..., :3] *= 12
    k[0, 0, :g_size] = 0.75           # a flat group
    if tokens > 8:
        k[2] *= 1e-30 if dt == torch.bfloat16 else 1e-4
        k[3] += 100.0
    k, v = k.to(dt).cuda(), torch.randn((tokens, h, 128), generator=g).to(dt).cuda()
    slots = _slots(tokens, nb, bs, g)
    pos = torch.randint(0, 400, (tokens,), generator=g)
    if rd:
        table = _table(400, rd)
        P.append_kv(cache, k, v, slots.cuda(), pos.cuda(), table)
        kref, kmag = O.rotate(k, table, pos, False)
    else:
        P.append_kv(cache, k, v, slots.cuda())
        kref = k.double().cpu()
        kmag = kref.abs()
    torch.cuda.synchronize()
    K.check_device_error(cache.device)
    keep = slots >= 0
    b, o = slots[keep] // bs, slots[keep] % bs
    codes, step, mid = O.unpack(cache.cpu(), dt)
    half, tiny = O.half_step(dt), torch.finfo(dt).smallest_normal
    sub = torch.finfo(dt).eps * tiny  # the type's smallest step
    for plane, (x, mag) in enumerate(((kref, kmag), (v.double().cpu(), v.double().cpu().abs()))):
        x, mag = (y[keep].unflatten(-1, (128 // g_size, g_size)) for y in (x, mag))
        c = codes[plane][b, :, o].unflatten(-1, (128 // g_size, g_size))
        s, m = step[plane][b, :, o].double(), mid[plane][b, :, o].double()
        lo, hi = x.amin(-1), x.amax(-1)
        err = 2 ** -22 * mag.amax(-1)  # fp32 of the rotation and of the formulas
        assert ((s - (hi - lo) / 15).abs() <= half * s.abs() * 1.01 + err / 7 + sub).all()
        assert ((m - lo - 8 * s).abs() <= half * m.abs() * 1.01 + 2 * err + sub).all()
        t = torch.where(s[..., None] > 0, (x - m[..., None]) / s[..., None] + 8, 8.0).clamp(0, 15)
        slack = torch.where(s > 0, 4 * err / s, 0.0)
        assert ((c - t).abs() <= 0.5 + slack[..., None] + 2 ** -18).all()
    # what was not appended keeps its bytes
    now = O.unpack(cache.cpu(), torch.int16)
    for a, z in zip(now, O.unpack(before, torch.int16)):
        z[:, b, :, o] = a[:, b, :, o]
        assert torch.equal(a, z)


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("g_size", [32, 64, 128])
def test_append_4bit_is_the_fp32_formula(dt, g_size):
    """The stored bytes are those of the formula in fp32, one rounding an operation."""
    g = _gen(g_size)
    T, h, bs, rd = 600, 3, 16, 128
    k, v = (torch.randn((T, h, 128), generator=g) for _ in range(2))
    k[..., ::17] *= 12
    k, v = k.to(dt), v.to(dt)
    pos = torch.randint(0, 300, (T,), generator=g)
    table = _table(300, rd).cpu()
    cache = P.kv4_cache(T // bs + 1, h, bs, g_size)
    P.append_kv(cache, k.cuda(), v.cuda(), torch.arange(T).cuda(), pos.cuda(), table.cuda())
    c, s = table[pos][:, None, :64], table[pos][:, None, 64:]
    a, b = k.float()[..., :64], k.float()[..., 64:]
    x = torch.stack([torch.cat([a * c - b * s, b * c + a * s], -1), v.float()])
    x = x.unflatten(-1, (128 // g_size, g_size))
    lo, hi = x.amin(-1), x.amax(-1)
    step = ((hi - lo) * torch.tensor(1 / 15)).to(dt)
    mid = (lo + 8 * step.float()).to(dt)
    code = ((x - mid.float()[..., None]) * (1 / step.float())[..., None] + 8.5).floor()
    code = code.clamp(0, 15).flatten(-2).long()
    got = O.unpack(cache.cpu(), dt)
    for have, want in zip(got, (code, step, mid)):
        have = have.transpose(2, 3).flatten(1, 2)[:, :T]  # [2, tokens, heads, ...]
        assert torch.equal(have, want)


def test_append_4bit_infinities_and_nans_stay_in_their_group():
    k = torch.zeros((4, 1, 128), dtype=torch.bfloat16)
    k[:] = torch.arange(128) / 8
    k[0, 0, 5], k[1, 0, 40], k[2, 0, 70], k[2, 0, 71] = math.inf, math.nan, math.inf, -math.inf
    cache = P.kv4_cache(1, 1, 16, 32)
    P.append_kv(cache, k.cuda(), k.cuda(), torch.arange(4).cuda())
    got = P.read_kv4(cache, torch.arange(4).cuda(), torch.bfloat16).cpu()[:, :, 0]
    bad = torch.zeros((4, 128), dtype=torch.bool)
    bad[0, :32] = bad[1, 32:64] = bad[2, 64:96] = True
    for plane in got:
        assert torch.equal(plane.isnan(), bad)
        d = (plane.double() - k[:, 0].double()).abs()[~bad]
        assert (d <= 0.5 * 31 / 8 / 15 + 0.1).all()


# ---------------------------------------------------------------------- read
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("g_size", [32, 64, 128])
@pytest.mark.parametrize("n,h,bs", [(1, 1, 16), (37, 5, 16), (200, 2, 64)])
def test_read_is_the_formula(dt, g_size, n, h, bs):
    g = _gen(n * g_size)
    nb, ng = 7, 128 // g_size
    codes = torch.randint(0, 16, (2, nb, h, bs, 128), generator=g)
    step = torch.rand((2, nb, h, bs, ng), generator=g).to(dt)
    mid = torch.randn((2, nb, h, bs, ng), generator=g).to(dt)
    cache = O.pack(codes, step, mid)
    again = O.unpack(cache, dt)
    assert all(torch.equal(a, z) for a, z in zip(again, (codes, step, mid)))
    slots = torch.randint(0, nb * bs, (n,), generator=g)  # repeats are fine to read
    if n > 2:
        slots[1] = -1
    got = P.read_kv4(cache.cuda(), slots.cuda(), dt).cpu()
    # code * step is exact in fp32, the sum rounds once, the type once: the same bits
    s, m = (x.float().repeat_interleave(g_size, -1) for x in (step, mid))
    want = (m + (codes - 8) * s).to(dt)
    blk, off = slots.clamp(min=0) // bs, slots.clamp(min=0) % bs
    want = want[:, blk, :, off].transpose(0, 1).clone()
    want[:, slots < 0] = 0
    assert torch.equal(got, want)
    out = torch.empty_like(got).cuda()
    assert P.read_kv4(cache.cuda(), slots.int().cuda(), dt, out=out) is out
    assert torch.equal(out.cpu(), want)
    K.check_device_error(out.device)


# ----------------------------------------------------------------- attention
def _cache4(nb, h, bs, g_size, dt, g, spread=1.0):
    """A 4-bit cache of N(0, 1)-like rows with outlier key channels (CPU)."""
    ng = 128 // g_size
    codes = torch.randint(0, 16, (2, nb, h, bs, 128), generator=g)
    step = 0.1 + 0.3 * torch.rand((2, nb, h, bs, ng), generator=g)
    step[0, ..., 0] *= 4
    step *= torch.exp2(torch.randint(-2, 3, step.shape, generator=g) * spread)
    mid = 0.3 * torch.randn((2, nb, h, bs, ng), generator=g)
    return O.pack(codes, step.to(dt), mid.to(dt))


def _check(out, lse, ref, dt):
    want, wlse, tol, ltol = ref
    has = ~want.isnan()
    o = out.double().cpu()
    bound = tol + O.half_step(dt) * (want.abs() + tol) + torch.finfo(dt).eps * torch.finfo(dt).tiny
    worst = ((o - want).abs() / bound)[has].max() if has.any() else 0
    assert worst <= 1, f"{float(worst):.3g} of the tolerance"
    if lse is not None:
        rows = ~wlse.isnan()
        l = lse.double().cpu()[rows]
        assert torch.equal(l == -math.inf, wlse[rows] == -math.inf)
        fin = wlse[rows] > -math.inf
        assert ((l - wlse[rows]).abs()[fin] <= ltol[rows][fin]).all()


def _problem(seqs, hq, h, bs, g_size, dt, seed, spare_rows=0, cols_more=2, spread=1.0):
    """seqs: (query rows, cached tokens) of each sequence."""
    g = _gen(seed)
    cols = max((n + bs - 1) // bs for _, n in seqs) + cols_more
    need = [(n + bs - 1) // bs for _, n in seqs]
    nb = sum(need) + 3
    perm = torch.randperm(nb, generator=g).int()
    table = torch.full((len(seqs), cols), -7, dtype=torch.int32)  # unused entries: not read
    at = 0
    for r, c in enumerate(need):
        table[r, :c] = perm[at:at + c]
        at += c
    cache = _cache4(nb, h, bs, g_size, dt, g, spread)
    T = sum(n for n, _ in seqs) + spare_rows
    q = (torch.randn((T, hq, 128), generator=g) * 0.7).to(dt)
    start = torch.tensor([0] + [n for n, _ in seqs]).cumsum(0).int()
    lens = torch.tensor([n for _, n in seqs]).int()
    return q, cache, table, lens, start


def _tiles(table, rows, hq, h, bs):
    """Whether a call takes the kernel for many rows, going by what the host knows: rows a kv
    head, and rows times tokens that the table has room for."""
    rows *= hq // h
    return rows > 48 and rows * h * table.numel() * bs > 5 << 20


def _wide(rows, seqs, hq, h, bs=16):
    """Table columns that take a call of few tokens there all the same."""
    return (6 << 20) // (rows * (hq // h) * h * seqs * bs) + 1


@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("g_size", [32, 64, 128])
@pytest.mark.parametrize("hq,h,bs", [(7, 1, 16), (8, 8, 32), (28, 4, 16), (16, 1, 16), (48, 2, 48)])
def test_attention_one_token(dt, g_size, hq, h, bs):
    lens = [1, 15, 16, 17, 0, 31, 32, 33, 127, 128, 129, 400, 2]
    q, cache, table, lens, _ = _problem([(1, n) for n in lens], hq, h, bs, g_size, dt, hq + bs)
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    _check(out, lse, O.attend(q, cache, table, lens, None), dt)


@pytest.mark.parametrize("dt,g_size", [(torch.bfloat16, 64), (torch.float16, 32),
                                       (torch.bfloat16, 128)])
@pytest.mark.parametrize("hq,h,seqs", [
    (5, 1, [(3, 3), (1, 70), (5, 64)]),
    (10, 2, [(2, 1), (4, 0), (0, 50), (7, 200), (1, 1)]),  # rows that see nothing, no rows
    (7, 1, [(130, 130), (33, 160)]),
    (8, 2, [(64, 300), (17, 17)]),
    (3, 3, [(100, 37)]),
    (8, 1, [(16, 500), (0, 30), (33, 0), (40, 129), (1, 128)]),   # one tile and two, no keys
    (16, 2, [(300, 300), (5, 1000), (64, 64)]),
    (4, 4, [(65, 1111), (1, 1), (257, 256)]),
])
@pytest.mark.parametrize("wide", [False, True])
def test_attention_several_rows(dt, g_size, hq, h, seqs, wide):
    most = max(n for n, _ in seqs)
    if wide and most * (hq // h) <= 48:
        pytest.skip("too few rows for the other kernel")
    q, cache, table, lens, start = _problem(
        seqs, hq, h, 16, g_size, dt, hq * 7, spare_rows=3,
        cols_more=_wide(most, len(seqs), hq, h) if wide else 2)
    tiles = _tiles(table, most, hq, h, 16)
    assert tiles or not wide
    out = torch.full_like(q, 9.0).cuda()
    got, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(),
                               max(n for n, _ in seqs), out=out, return_lse=True)
    torch.cuda.synchronize()
    assert got is out
    K.check_device_error(out.device)
    ref = O.attend(q, cache, table, lens, start, tiles=tiles)
    _check(out, lse, ref, dt)
    assert (out[int(start[-1]):] == 9.0).all()  # rows of no sequence


@pytest.mark.parametrize("first", [1, 30])
def test_attention_more_sequences_than_threads(first):
    """Both kernels find a share's beginning in several rounds over the lengths."""
    g = torch.Generator().manual_seed(first)
    dt, hq, h = torch.bfloat16, 4, 1
    seqs = [(int(n > 0), n) for n in torch.randint(0, 60, (700,), generator=g).tolist()]
    seqs[3] = (0, 25)
    seqs[650] = (first, 77)
    q, cache, table, lens, start = _problem(seqs, hq, h, 16, 64, dt, first, cols_more=2)
    assert _tiles(table, first, hq, h, 16) == (first == 30)
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), start.cuda(),
                               first, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    _check(out, lse, O.attend(q, cache, table, lens, start, tiles=first == 30), dt)


def test_attention_many_rows_magnitudes_and_growth():
    """Values far from 1, steps and scores that rise along the sequence, a negative scale."""
    for dt, mag in ((torch.bfloat16, 1e-18), (torch.bfloat16, 1e6), (torch.float16, 1.0)):
        q, cache, table, lens, start = _problem([(90, 700), (20, 20)], 4, 2, 16, 64, dt, 31,
                                                cols_more=_wide(90, 2, 4, 2))
        assert _tiles(table, 90, 4, 2, 16)
        codes, step, mid = O.unpack(cache, dt)
        grow = torch.zeros(cache.shape[0])
        used = table[0][:44].long()
        grow[used] = torch.linspace(-6, 3, 44)
        grow = torch.exp2(grow)[:, None, None, None].double()
        up = torch.tensor([1 / mag, mag]).double()[:, None, None, None, None]
        up = up * torch.stack([grow.sqrt(), grow])
        step, mid = (step.double() * up).to(dt), (mid.double() * up).to(dt)
        cache = O.pack(codes, step, mid)
        q = (q.double() * mag).to(dt)
        out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(),
                                   start.cuda(), 90, scale=-0.11, return_lse=True)
        torch.cuda.synchronize()
        K.check_device_error(out.device)
        want, wlse, tol, ltol = O.attend(q, cache, table, lens, start, scale=-0.11, tiles=True)
        bound = tol + O.half_step(dt) * (want.abs() + tol)
        assert ((out.double().cpu() - want).abs() <= bound).all()
        assert ((lse.double().cpu() - wlse).abs() <= ltol).all()


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_infinite_values_stay_in_their_channels(rows):
    dt = torch.bfloat16
    q, cache, table, lens, start = _problem([(rows, 300), (rows, 200)], 8, 2, 16, 64, dt, 45,
                                            cols_more=_wide(40, 2, 8, 2))
    ref = O.attend(q, cache, table, lens, start, tiles=rows > 16)
    codes, step, mid = O.unpack(cache, dt)
    step[1, int(table[0, 3]), 1, 5, 0] = math.inf  # token 53 of sequence 0: every row sees it
    mid[1, int(table[1, 8]), 0, 2, 1] = -math.inf  # token 130 of sequence 1
    out = P.attention_kv4(q.cuda(), O.pack(codes, step, mid).cuda(), table.cuda(), lens.cuda(),
                          start.cuda(), rows).cpu().double()
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[:rows, 4:, :64] = bad[rows:, :4, 64:] = True
    assert not out[bad].isfinite().any()
    want, _, tol, _ = ref
    assert ((out - want).abs() <= tol + O.half_step(dt) * (want.abs() + tol) + 1e-30)[~bad].all()


@pytest.mark.parametrize("rows", [1, 40])
def test_attention_values_of_zero_and_tiny_scales(rows):
    """Tokens whose values are all zero still count in the sum, next to large ones; scales
    and keys so small that every score is the same."""
    dt = torch.bfloat16
    q, cache, table, lens, start = _problem([(rows, 150), (rows, rows)], 8, 2, 16, 64, dt, 44,
                                            cols_more=_wide(40, 2, 8, 2))
    assert _tiles(table, rows, 8, 2, 16) == (rows == 40)
    codes, step, mid = O.unpack(cache, dt)
    big = step[1].double() * 2.0 ** 40
    big[table[0][2:9].long()] = 0  # tokens 32 to 143 of sequence 0
    step[1], mid[1] = big.to(dt), 0
    cache = O.pack(codes, step, mid)
    for scale in (0.1, 1e-37):
        out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(),
                                   start.cuda(), rows, scale=scale, return_lse=True)
        torch.cuda.synchronize()
        K.check_device_error(out.device)
        _check(out, lse, O.attend(q, cache, table, lens, start, scale=scale, tiles=rows > 16), dt)


def test_attention_many_rows_bad_blocks_and_numbers():
    """A block id outside the cache hides its tokens; NaN and infinities behind the length or
    behind a row's own position do not reach it, and those that it sees stay in their group."""
    dt, h, hq = torch.bfloat16, 2, 8
    q, cache, table, lens, start = _problem([(40, 100), (30, 77)], hq, h, 16, 64, dt, 12,
                                            cols_more=_wide(40, 2, hq, h))
    assert _tiles(table, 40, hq, h, 16)
    ref = O.attend(q, cache, table, lens, start, tiles=True)
    codes, step, mid = O.unpack(cache, dt)
    for r, n in enumerate(lens.tolist()):
        last = int(table[r, (n - 1) // 16])
        step[:, last, :, n % 16:] = math.nan
        mid[:, last, :, n % 16:] = -math.inf
    hurt = O.pack(codes, step, mid)
    args = [x.cuda() for x in (table, lens, start)]
    out = P.attention_kv4(q.cuda(), hurt.cuda(), *args, 40)
    _check(out, None, ref, dt)
    # token 90 of sequence 0 holds a NaN value in the second group of head 1: rows 30 and on see it
    mid[1, int(table[0, 5]), 1, 10, 1] = math.nan
    out = P.attention_kv4(q.cuda(), O.pack(codes, step, mid).cuda(), *args, 40).cpu()
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[30:40, 4:, 64:] = True
    assert torch.equal(out.isnan(), bad)
    want, _, tol, _ = ref
    d = (out.double() - want).abs() / (tol + O.half_step(dt) * (want.abs() + tol) + 1e-30)
    assert (d[~bad & ~want.isnan()] <= 1).all()
    # the last two blocks of sequence 0 are full of hidden tokens
    gone = table.clone()
    gone[0, 5], gone[0, 6] = cache.shape[0] + 7, -2
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), gone.cuda(), *args[1:], 40,
                               return_lse=True)
    assert _error() == 3
    for i in (0, 19, 39):  # row i sees tokens up to 60 + i, of them those below 80
        n = min(61 + i, 80)
        one = O.attend(q[i:i + 1], cache, table[:1], torch.tensor([n]).int(), None, tiles=True)
        _check(out[i:i + 1], lse[i:i + 1], one, dt)


@pytest.mark.parametrize("n", [5000, 20011])
def test_attention_long(n):
    q, cache, table, lens, _ = _problem([(1, n), (1, 3)], 7, 1, 16, 64, torch.bfloat16, n)
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    _check(out, lse, O.attend(q, cache, table, lens, None), q.dtype)


def test_attention_scores_that_grow_and_steps_that_vary():
    """The running maximum and the largest step both rise along the sequence."""
    g = _gen(11)
    n, h, bs = 700, 2, 16
    codes = torch.randint(0, 16, (2, 50, h, bs, 128), generator=g)
    step = 0.2 * torch.rand((2, 50, h, bs, 2), generator=g) + 0.05
    table = torch.arange(50).int()[None]
    grow = torch.linspace(-9, 4, 50)[:, None, None, None]
    step[1] *= torch.exp2(grow)
    step[0] *= torch.exp2(torch.linspace(-3, 3, 50))[:, None, None, None]
    mid = torch.zeros_like(step)
    for dt in DTYPES:
        cache = O.pack(codes, step.to(dt), mid.to(dt))
        q = (torch.randn((1, 8, 128), generator=g) * 2).to(dt)
        lens = torch.tensor([n]).int()
        out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(),
                                   return_lse=True)
        _check(out, lse, O.attend(q, cache, table, lens, None), dt)


@pytest.mark.parametrize("mag", [1e-20, 1e-3, 1e4])
def test_attention_magnitudes(mag):
    """Queries and values far from 1 (bf16): tiny values keep their relative precision."""
    dt = torch.bfloat16
    q, cache, table, lens, _ = _problem([(1, 100), (1, 40)], 4, 2, 16, 64, dt, 5)
    codes, step, mid = O.unpack(cache, dt)
    step[1] = (step[1].double() * mag).to(dt)
    mid[1] = (mid[1].double() * mag).to(dt)
    step[0] = (step[0].double() / mag).to(dt)
    mid[0] = (mid[0].double() / mag).to(dt)
    cache = O.pack(codes, step, mid)
    q = (q.double() * mag).to(dt)
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(), lens.cuda(), return_lse=True)
    want, wlse, tol, ltol = O.attend(q, cache, table, lens, None)
    bound = tol + O.half_step(dt) * (want.abs() + tol)
    assert ((out.double().cpu() - want).abs() <= bound).all()
    assert ((lse.double().cpu() - wlse).abs() <= ltol).all()


def test_attention_scale_strides_and_views():
    dt = torch.float16
    q, cache, table, lens, _ = _problem([(1, 90), (1, 33)], 6, 2, 16, 32, dt, 21)
    ref = O.attend(q, cache, table, lens, None, scale=0.25)
    wide = torch.zeros((2, 14, 128), dtype=dt).cuda()
    wide[:, 3:9] = q.cuda()
    big = torch.zeros((cache.shape[0], 3, *cache.shape[1:]), dtype=torch.uint8).cuda()
    big[:, 1] = cache.cuda()  # one layer of a cache that holds several, block by block
    tab = torch.full((2, 2 * table.shape[1]), -3, dtype=torch.int32).cuda()
    tab[:, :table.shape[1]] = table.cuda()
    outw = torch.zeros((2, 10, 128), dtype=dt).cuda()
    out = P.attention_kv4(wide[:, 3:9], big[:, 1], tab, lens.cuda(), scale=0.25,
                          out=outw[:, 2:8])
    _check(out, None, ref, dt)
    assert (outw[:, :2] == 0).all() and (outw[:, 8:] == 0).all()


def test_attention_ignores_what_lies_behind_the_length():
    """NaN and infinite metadata in unused slots of used blocks, any dtype."""
    for dt in DTYPES:
        for lens in ([5, 17, 40], [64, 1, 33]):
            q, cache, table, lens, _ = _problem([(1, n) for n in lens], 4, 2, 16, 64, dt, 8)
            ref = O.attend(q, cache, table, lens, None)
            codes, step, mid = O.unpack(cache, dt)
            for r, n in enumerate(lens.tolist()):
                last = int(table[r, (n - 1) // 16])
                step[:, last, :, n % 16 if n % 16 else 16:] = math.nan
                mid[:, last, :, n % 16 if n % 16 else 16:] = -math.inf
            out, lse = P.attention_kv4(q.cuda(), O.pack(codes, step, mid).cuda(), table.cuda(),
                                       lens.cuda(), return_lse=True)
            _check(out, lse, ref, dt)


def test_attention_nan_in_a_seen_key_reaches_only_its_rows():
    dt = torch.bfloat16
    q, cache, table, lens, _ = _problem([(1, 40), (1, 40)], 4, 2, 16, 64, dt, 9)
    codes, step, mid = O.unpack(cache, dt)
    mid[0, int(table[0, 1]), 1, 3] = math.nan  # sequence 0, head 1
    out = P.attention_kv4(q.cuda(), O.pack(codes, step, mid).cuda(), table.cuda(), lens.cuda())
    bad = out.isnan().all(-1).cpu()
    assert bad.tolist() == [[False, False, True, True], [False] * 4]
    assert not out[~bad.cuda()].isnan().any()


def test_offsets_beyond_32_bits():
    """Blocks whose records lie more than 4 GB into the cache."""
    dt, h, bs = torch.bfloat16, 1, 16
    rec = bs * P.kv4_row_bytes(64)
    nb = (5 << 30) // rec
    cache = P.kv4_cache(nb, h, bs, 64)
    g = _gen(4)
    k, v = (torch.randn((40, h, 128), generator=g).to(dt).cuda() for _ in range(2))
    blocks = torch.tensor([nb - 1, 3, nb - 5])
    slots = torch.cat([b * bs + torch.arange(bs) for b in blocks])[:40]
    P.append_kv(cache, k, v, slots.cuda())
    got = P.read_kv4(cache, slots.cuda(), dt).cpu().double()
    for plane, x in zip(got, (k, v)):
        d = (plane - x.cpu().double()).abs()
        span = x.cpu().double().unflatten(-1, (2, 64))
        span = (span.amax(-1) - span.amin(-1)).amax()
        assert d.max() <= span / 15 * (0.5 + 15 * 2 ** -8) + 2 ** -7
    q = torch.randn((1, 4, 128), generator=g).to(dt)
    out = P.attention_kv4(q.cuda(), cache, blocks.int()[None].cuda(),
                          torch.tensor([40]).int().cuda())
    small = cache[blocks.cuda()].cpu()
    ref = O.attend(q, small, torch.arange(3).int()[None], torch.tensor([40]).int(), None)
    _check(out, None, ref, dt)
    K.check_device_error(out.device)


def _error():
    torch.cuda.synchronize()
    return K.read_device_error(torch.device("cuda", 0))


def test_indices_out_of_range_are_recorded_and_left_out():
    """Every access of these calls is checked in the kernels before it is made."""
    dt = torch.bfloat16
    cache = P.kv4_cache(4, 2, 16, 64)
    k = torch.randn((4, 2, 128), generator=_gen(1)).to(dt).cuda()
    table = _table(32, 128)
    P.append_kv(cache, k, k, torch.tensor([0, 64, 1 << 40, 3]).cuda())
    assert _error() == 3
    rows = P.read_kv4(cache, torch.arange(64).cuda(), dt)
    assert (rows[:, [0, 3]] != 0).any(-1).all() and (rows[:, 4:] == 0).all()
    assert (rows[:, 1:3] == 0).all()
    q = torch.randn((4, 2, 128), generator=_gen(2)).to(dt).cuda()
    turned = P.append_kv(cache, k, k, torch.arange(8, 12).cuda(),
                         torch.tensor([0, 32, -1, 31]).cuda(), table, q)
    assert _error() == 3
    rows = P.read_kv4(cache, torch.arange(64).cuda(), dt)
    assert (rows[:, [9, 10]] == 0).all() and (rows[:, [8, 11]] != 0).any(-1).all()
    assert torch.equal(turned[[1, 2]], q[[1, 2]])
    assert (P.read_kv4(cache, torch.tensor([64, 8]).cuda(), dt)[:, 0] == 0).all()
    assert _error() == 3
    # a block id outside the cache: its tokens are not seen
    q, c4, tab, lens, _ = _problem([(1, 48), (1, 20)], 4, 2, 16, 64, dt, 3)
    bad = tab.clone()
    bad[0, 1] = c4.shape[0]
    out = P.attention_kv4(q.cuda(), c4.cuda(), bad.cuda(), lens.cuda())
    assert _error() == 3
    gone = tab.clone()
    gone[0, 1] = tab[0, 2]
    gone[0, 2] = -1
    ref = O.attend(q, c4, gone, torch.tensor([32, 20]).int(), None)
    _check(out, None, ref, dt)
    # lengths and rows that do not fit: the sequence is left out
    out = torch.full_like(q, 5.0).cuda()
    P.attention_kv4(q.cuda(), c4.cuda(), tab.cuda(), torch.tensor([10 ** 6, 20]).int().cuda(),
                    out=out)
    assert _error() == 3
    assert (out[0] == 5.0).all() and (out[1] != 5.0).any()
    P.attention_kv4(q.cuda(), c4.cuda(), tab.cuda(), lens.cuda(),
                    torch.tensor([0, 9, 2]).int().cuda(), 2, out=out)
    assert _error() == 3


# ------------------------------------------------------------------ together
def _decode(cache, table, state, steps, q, k, v, cos_sin):
    """Append and attend, step by step, with everything on the device."""
    outs = []
    for i in range(steps):
        state["lens"] += 1
        pos = state["lens"] - 1
        blk = table.gather(1, (pos // cache.shape[2]).long()[:, None])[:, 0]
        slots = blk * cache.shape[2] + pos % cache.shape[2]
        turned = P.append_kv(cache, k[i], v[i], slots, pos, cos_sin, q[i])
        outs.append(P.attention_kv4(turned, cache, table, state["lens"]))
    return outs


@pytest.mark.parametrize("dt,g_size", [(torch.bfloat16, 64), (torch.float16, 32)])
def test_decode_steps_eager_and_captured(dt, g_size):
    """Prefill, then decode steps through append and attention; the same steps in a
    captured graph give the same bits."""
    g = _gen(77)
    R, hq, h, bs, steps = 3, 8, 2, 16, 5
    prompt = [30, 47, 1]
    cos_sin = _table(128, 128)
    table = torch.randperm(20, generator=g)[:R * 6].view(R, 6).int().cuda()

    def rows(*shape):
        return torch.randn(shape, generator=g).to(dt).cuda()

    T = sum(prompt)
    pq, pk, pv = rows(T, hq, 128), rows(T, h, 128), rows(T, h, 128)
    q, k, v = rows(steps, R, hq, 128), rows(steps, R, h, 128), rows(steps, R, h, 128)
    pos = torch.cat([torch.arange(n) for n in prompt])
    seq = torch.repeat_interleave(torch.arange(R), torch.tensor(prompt))
    slots = table.cpu()[seq, pos // bs] * bs + pos % bs
    start = torch.tensor([0] + prompt).cumsum(0).int().cuda()
    runs = []
    for captured in (False, True):
        cache = P.kv4_cache(20, h, bs, g_size)
        lens = torch.tensor(prompt).int().cuda()
        turned = P.append_kv(cache, pk, pv, slots.cuda(), pos.cuda(), cos_sin, pq)
        first = P.attention_kv4(turned, cache, table, lens, start, max(prompt))
        ref = O.attend(turned.cpu(), cache, table, lens, start)
        _check(first, None, ref, dt)
        state = {"lens": lens}
        if captured:
            one = {"q": torch.empty_like(q[:1]), "k": torch.empty_like(k[:1]),
                   "v": torch.empty_like(v[:1])}
            graph = torch.cuda.CUDAGraph()
            saved, kept = lens.clone(), cache.clone()
            for x, y in (("q", q), ("k", k), ("v", v)):
                one[x].copy_(y[:1])
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                _decode(cache, table, state, 1, one["q"], one["k"], one["v"], cos_sin)
            torch.cuda.current_stream().wait_stream(side)
            lens.copy_(saved)
            cache.copy_(kept)
            with torch.cuda.graph(graph):
                res = _decode(cache, table, state, 1, one["q"], one["k"], one["v"], cos_sin)
            outs = []
            for i in range(steps):
                for x, y in (("q", q), ("k", k), ("v", v)):
                    one[x].copy_(y[i:i + 1])
                graph.replay()
                outs.append(res[0].clone())
        else:
            outs = _decode(cache, table, state, steps, q, k, v, cos_sin)
            end = lens.clone()
            turned = P.append_kv(P.kv4_cache(20, h, bs, g_size), k[-1], v[-1],
                                 torch.arange(R).cuda(), end - 1, cos_sin, q[-1])
            _check(outs[-1], None, O.attend(turned.cpu(), cache, table, end, None), dt)
        torch.cuda.synchronize()
        K.check_device_error(cache.device)
        runs.append((outs, cache))
    for a, z in zip(*(r[0] for r in runs)):
        assert torch.equal(a, z)
    assert torch.equal(runs[0][1], runs[1][1])


def test_two_graphs_at_once():
    """Two graphs captured one after the other, replayed on two streams at the same time."""
    dt = torch.bfloat16
    probs = [_problem([(1, n), (1, 37)], 8, 2, 16, 64, dt, n) for n in (3000, 2500)]
    args = [[x.cuda() for x in p[:4]] for p in probs]
    want = [P.attention_kv4(*a) for a in args]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(P.attention_kv4(*a))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    torch.cuda.synchronize()
    for _ in range(20):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert torch.equal(o, w)


def test_component_speed_times_the_serving_operators():
    from kvserve_hpdps_b200.offline import component_speed as CS
    rows = CS.run_serving(tokens=300, heads=2, q_heads=8, requests=3, chunk=40, iters=2, warmup=1)
    assert [r["stage"] for r in rows] == [*CS.SERVING, "summary"]
    assert all(r["ms"] > 0 for r in rows[:-1])
    assert rows[-1]["device_error"] == 0 and rows[-1]["cosine"] > 0.98


def test_results_do_not_change_from_call_to_call():
    q, cache, table, lens, start = _problem([(9, 1500), (2, 800), (1, 5)], 12, 3, 16, 32,
                                            torch.float16, 2)
    a = [x.cuda() for x in (q, cache, table, lens, start)]
    _same_again(a, 9)
    q, cache, table, lens, start = _problem([(200, 900), (77, 300)], 8, 2, 16, 64,
                                            torch.bfloat16, 6, cols_more=_wide(200, 2, 8, 2))
    assert _tiles(table, 200, 8, 2, 16)
    _same_again([x.cuda() for x in (q, cache, table, lens, start)], 200)


def _same_again(a, most):
    first = P.attention_kv4(*a, most)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for i in range(5):
        with torch.cuda.stream(side if i % 2 else torch.cuda.current_stream()):
            again = P.attention_kv4(*a, most)
        torch.cuda.synchronize()
        assert torch.equal(first, again)
