"""8-bit paged cache: appended and re-scaled units byte for byte against the definition,
rows read back, and the order and number of a call's tokens."""

import math

import pytest
import torch

import paged8_oracle as O8
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
    return torch.cat([ang.cos(), ang.sin()], 1).to(dtype)


def _rows(g, n, h, dt, wild=True):
    x = torch.randn((n, h, 128), generator=g)
    if wild:
        x = x * 2.0 ** (20 * torch.rand((n, 1, 1), generator=g) - 10)
    return x.to(dt)


def _random_cache(g, nb, h, bs):
    """Random codes (not a number among them) under scales near 1."""
    c = torch.randint(0, 256, (nb, h, 2 * bs + 1, 128), generator=g, dtype=torch.uint8)
    c[:, :, 2 * bs] = torch.randint(115, 130, (nb, h, 128), generator=g, dtype=torch.uint8)
    return c


def _same(got, want):
    """Bytes equal; of what is not a number the sign is free."""
    a, b = got.cpu(), want
    rows = a.shape[2] - 1
    nan = (a[:, :, :rows] & 127 == 127) & (b[:, :, :rows] & 127 == 127)
    assert ((a[:, :, :rows] == b[:, :, :rows]) | nan).all()
    assert torch.equal(a[:, :, rows], b[:, :, rows])


def _check_append(cache, k, v, slots, pos=None, table=None, inter=False, q=None):
    want = cache.clone()
    O8.append(want, k, v, slots, pos, table, inter)
    dev = cache.cuda()
    on = lambda x: None if x is None else x.cuda()  # noqa: E731
    out = P.append_kv(dev, k.cuda(), v.cuda(), slots.cuda(), on(pos), on(table), on(q),
                      interleaved=inter)
    K.check_device_error(dev.device)
    _same(dev, want)
    return dev, out


# -------------------------------------------------------------------- append
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("tokens,hq,h,bs,rd,inter", [
    (1, 7, 1, 16, 128, False), (5, 28, 4, 32, 128, True), (33, 8, 8, 16, 64, False),
    (300, 6, 2, 48, 96, True), (40, 5, 5, 16, 16, False), (64, 16, 3, 1024, 112, False),
    (17, 40, 16, 64, 128, False)])
def test_append_scattered(dt, tokens, hq, h, bs, rd, inter):
    """Tokens at random slots of units that hold others: scales grow, some units begin anew."""
    g = _gen(tokens * 37 + rd)
    nb = max(3, tokens * 3 // bs + 2)
    cache = _random_cache(g, nb, h, bs)
    slots = torch.randperm(nb * bs, generator=g)[:tokens]
    if tokens > 3:
        slots[1::5] = -1
    pos = torch.randint(0, 500, (tokens,), generator=g)
    table = _table(500, rd, dt if tokens == 33 else torch.float32)
    k, v, q = _rows(g, tokens, h, dt), _rows(g, tokens, h, dt), _rows(g, tokens, hq, dt, False)
    idx = torch.int32 if tokens % 2 else torch.int64
    _, out = _check_append(cache, k, v, slots.to(idx), pos.to(idx), table, inter, q)
    ref, mag = O.rotate(q, table, pos, inter)
    half = O.half_step(dt)
    smallest = torch.finfo(dt).eps * torch.finfo(dt).tiny
    bound = half * ref.abs() * (1 + 2 ** -20) + 2 ** -23 * mag + smallest
    assert ((out.double().cpu() - ref).abs() <= bound).all()


@pytest.mark.parametrize("order", ["rising", "falling", "shuffled"])
@pytest.mark.parametrize("tokens,first", [(16, 0), (16, 5), (47, 0), (200, 3), (700, 9),
                                          (4097, 0), (4200, 11)])
def test_append_prompts(tokens, first, order):
    """A prompt's tokens into consecutive slots, from inside a unit on and in any order: a unit's
    tokens need not stand next to each other.  From 4097 tokens on a CTA takes 16."""
    g = _gen(tokens + first)
    bs, h, nb = 32, 1 if tokens > 1000 else 2, (tokens + first) // 32 + 3
    perm = torch.randperm(nb, generator=g)
    t = torch.arange(tokens) + first
    slots = perm[t // bs] * bs + t % bs
    at = {"rising": torch.arange(tokens), "falling": torch.arange(tokens).flip(0),
          "shuffled": torch.randperm(tokens, generator=g)}[order]
    k, v = _rows(g, tokens, h, torch.bfloat16), _rows(g, tokens, h, torch.bfloat16)
    _check_append(_random_cache(g, nb, h, bs), k[at], v[at], slots[at], t[at], _table(5000, 128))


def test_append_token_by_token_keeps_what_was_there():
    """16 tokens one by one, each up to twice the last: every step's bytes are the definition's, and
    a row is off by a rounding to e4m3 and, of the unit's largest, 2^-18 a move at most."""
    g = _gen(5)
    cache = P.kv8_cache(2, 2, 16, device="cpu")
    k = torch.randn((16, 2, 128), generator=g) * 1.7 ** torch.arange(16)[:, None, None]
    k, v = k.half(), torch.randn((16, 2, 128), generator=g).half()
    dev = cache.cuda()
    for t in range(16):
        O8.append(cache, k[t:t + 1], v[t:t + 1], torch.tensor([16 + t]))
        P.append_kv(dev, k[t:t + 1].cuda(), v[t:t + 1].cuda(), torch.tensor([16 + t]).cuda())
        _same(dev, cache)
    back = P.read_kv8(dev, torch.arange(16, 32).cuda(), torch.bfloat16).double().cpu()
    for x, y in zip(back, (k, v)):
        y = y.double()
        top = y.abs().amax((0, 2), keepdim=True)
        assert ((x - y).abs() <= 2 ** -4 * y.abs() + 10 * 2 ** -18 * top).all()


def test_append_begins_anew_at_offset_0():
    """A unit of a former sequence, with a large scale, takes a small one with offset 0."""
    cache = P.kv8_cache(1, 1, 16, device="cuda")
    big = torch.full((16, 1, 128), 3e4, dtype=torch.float16).cuda()
    P.append_kv(cache, big, big, torch.arange(16).cuda())
    small = (torch.randn((3, 1, 128), generator=_gen(1)) * 1e-3).half().cuda()
    P.append_kv(cache, small, small, torch.arange(3).cuda())
    got = P.read_kv8(cache, torch.arange(3).cuda(), torch.float16)[0]
    assert ((got - small).abs().float() <= 2 ** -4 * small.abs().float() + 2 ** -22).all()


def test_append_not_finite_and_extreme():
    """Infinities and NaN are NaN and have no say in the scale; the type's largest and smallest
    numbers are held; zeros are zeros."""
    g = _gen(6)
    k = torch.randn((48, 1, 128), generator=g).bfloat16()
    k[0, 0, 3], k[1, 0, 4], k[2, 0, 5] = math.inf, -math.inf, math.nan
    k[16:32] = 0
    k[32] = torch.finfo(torch.bfloat16).max
    k[33] *= 1e-38
    v = torch.randn((48, 1, 128), generator=g).bfloat16() * 1e-36
    v[5] = math.nan  # a whole row
    v[16:32] = math.inf
    dev, _ = _check_append(P.kv8_cache(4, 1, 16, device="cpu"), k, v, torch.arange(16, 64))
    back = P.read_kv8(dev, torch.arange(16, 64).cuda(), torch.bfloat16).cpu()
    assert torch.equal(torch.isfinite(back[0]), torch.isfinite(k))
    assert torch.isnan(back[1, 16:32]).all() and not back[0, 16:32].any()
    big = torch.finfo(torch.bfloat16).max
    assert ((back[0, 32].double() - big).abs() <= 2 ** -4 * big).all()


def test_append_into_a_cache_never_cleared():
    """Bytes that no append writes have no say in a scale."""
    g = _gen(7)
    cache = torch.full((2, 2, 33, 128), 255, dtype=torch.uint8)
    k, v = _rows(g, 7, 2, torch.float16), _rows(g, 7, 2, torch.float16)
    _check_append(cache, k, v, torch.arange(4, 11))


def test_append_repeats_and_misses():
    """A slot named twice stays inside its unit; slots and positions out of range are left out
    with an error."""
    g = _gen(8)
    cache = _random_cache(g, 4, 2, 16)
    dev = cache.cuda()
    k, v = _rows(g, 6, 2, torch.bfloat16).cuda(), _rows(g, 6, 2, torch.bfloat16).cuda()
    slots = torch.tensor([17, 18, 17, 19, 17, 17])
    want = cache.clone()
    O8.append(want, k.cpu(), v.cpu(), slots)  # of a slot's tokens the last
    P.append_kv(dev, k, v, slots.cuda())
    K.check_device_error(dev.device)
    _same(dev, want)
    for slots, pos in (([64, 3], [0, 1]), ([2, 3], [64, 1]), ([2, 3], [-1, 1])):
        want, dev = cache.clone(), cache.cuda()
        O8.append(want, k[1:2].cpu(), v[1:2].cpu(), torch.tensor([3]), torch.tensor([1]),
                  _table(64, 128))
        q = torch.randn((2, 3, 128), generator=g).bfloat16()
        out = P.append_kv(dev, k[:2], v[:2], torch.tensor(slots).cuda(), torch.tensor(pos).cuda(),
                          _table(64, 128).cuda(), q.cuda())
        with pytest.raises(RuntimeError):
            K.check_device_error(dev.device)
        _same(dev, want)
        if not 0 <= pos[0] < 64:
            assert torch.equal(out[0].cpu(), q[0])


def test_append_strides_and_padding():
    """Slices of one projection, a view of a larger cache, rows behind the slots, no queries, no
    heads, no tokens."""
    g = _gen(9)
    T, hq, h = 21, 6, 2
    qkv = torch.randn((T, hq + 2 * h, 128), generator=g).half()
    q, k, v = qkv[:, :hq], qkv[:, hq:hq + h], qkv[:, hq + h:]
    big = _random_cache(g, 10, 5, 32)
    view = big[::2, 1:3]
    want = view.clone()
    slots = torch.arange(37, 37 + 18)
    O8.append(want, k[:18], v[:18], slots, slots, _table(99, 96))
    dev = big.cuda()
    inplace = qkv.cuda()
    qq, kk, vv = inplace[:, :hq], inplace[:, hq:hq + h], inplace[:, hq + h:]
    out = P.append_kv(dev[::2, 1:3], kk, vv, slots.cuda(), slots.cuda(), _table(99, 96).cuda(), qq,
                      query_out=qq)
    assert out is qq and torch.equal(qq[18:].cpu(), q[18:])
    _same(dev[::2, 1:3], want)
    untouched = dev.cpu()
    untouched[::2, 1:3] = view
    assert torch.equal(untouched, big)
    full = P.append_kv(dev[::2, 1:3], kk, vv, slots.cuda(), slots.cuda(), _table(99, 96).cuda(),
                       q.cuda())
    assert torch.equal(full[:18], qq[:18]) and not full[18:].any()
    none = P.kv8_cache(2, 0)
    only = P.append_kv(none, kk[:, :0], vv[:, :0], slots.cuda(), slots.cuda(),
                       _table(99, 96).cuda(), q.cuda())
    assert torch.equal(only, full)
    assert P.append_kv(dev[::2, 1:3], kk, vv, slots[:0].cuda()) is None


# ---------------------------------------------------------------------- read
@pytest.mark.parametrize("dt", DTYPES)
@pytest.mark.parametrize("n,h,bs", [(1, 1, 16), (77, 3, 48), (3000, 8, 32), (5, 2, 1024)])
def test_read_rows(dt, n, h, bs):
    g = _gen(n + bs)
    nb = n // bs + 3
    cache = _random_cache(g, nb, h, bs)
    cache[0, 0, bs // 2] = torch.arange(128, dtype=torch.uint8)       # every number there is
    cache[0, 0, bs // 2 + 1] = torch.arange(128, 256, dtype=torch.uint8)
    cache[1, 0, 2 * bs, :4] = torch.tensor([0, 17, 100, 247], dtype=torch.uint8)
    slots = torch.randint(-1, nb * bs, (n,), generator=g)
    slots[:2] = torch.tensor([bs // 2, bs // 2 + 1])[:n]
    got = P.read_kv8(cache.cuda(), slots.cuda(), dt).cpu()
    want = O8.read(cache, slots)
    nan = torch.isnan(want)
    assert torch.equal(nan, torch.isnan(got))
    most = torch.finfo(dt).max
    assert torch.equal(got[~nan], want[~nan].clamp(-most, most).to(dt))  # one rounding
    out = torch.empty((2, n, h, 128), dtype=dt, device="cuda")
    assert P.read_kv8(cache.cuda(), slots.int().cuda(), dt, out) is out
    assert torch.equal(out.cpu()[~nan], got[~nan])


def test_read_out_of_range():
    cache = P.kv8_cache(2, 2)
    got = P.read_kv8(cache + 130, torch.tensor([32, 1]).cuda(), torch.float16)
    with pytest.raises(RuntimeError):
        K.check_device_error(cache.device)
    assert not got[:, 0].any() and got[:, 1].all()


@pytest.mark.parametrize("rd,inter", [(128, False), (64, False), (96, True)])
@pytest.mark.parametrize("tokens", [148, 149, 512, 513, 2368, 2385, 6400, 6417])
def test_append_where_the_work_is_dealt_otherwise(tokens, rd, inter):
    """Both sides of the sizes at which windows, heads a CTA and registers change: three sequences,
    their ends and starts inside units, in an order that goes on in the middle."""
    g = _gen(tokens + rd)
    bs, h, first = 32, 3, 5
    nb = (tokens + 120) // bs + 2
    blocks = torch.randperm(nb, generator=g)
    i = torch.arange(tokens) + first + 37 * (torch.arange(tokens) // (tokens // 3 + 1))
    slots = (blocks[i // bs] * bs + i % bs).roll(tokens // 2)
    k, v = _rows(g, tokens, h, torch.bfloat16), _rows(g, tokens, h, torch.bfloat16)
    q = _rows(g, tokens, 2, torch.bfloat16)
    pos = torch.randint(0, 99, (tokens,), generator=g)
    _check_append(_random_cache(g, nb, h, bs), k, v, slots, pos, _table(99, rd), inter, q)
