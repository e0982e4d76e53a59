"""The 8-bit paged cache's operators as a serving step uses them: captured and replayed, two graphs
at once, on other streams, caches past 2^32 bytes, long sequences, rows that are not finite."""

import math

import pytest
import torch

import paged8_oracle as O8
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P
from test_paged8_attention_gpu import _attend, _check, _problem, _tiles, _wide

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _no_device_error():
    K.check_device_error(torch.device("cuda", 0), "before the test")
    yield
    torch.cuda.synchronize()


def _angles(maxpos):
    ang = torch.arange(maxpos).double()[:, None] / 1e4 ** (torch.arange(0, 128, 2).double() / 128)
    return torch.cat([ang.cos(), ang.sin()], 1).float().cuda()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_decode_steps_eager_and_captured(dt):
    """Steps of a graph (append, attend, read, count up) leave what eager steps leave, bit for bit."""
    g = torch.Generator().manual_seed(4)
    R, hq, h, bs, steps = 5, 12, 2, 16, 20
    table = torch.randperm(R * 8, generator=g).view(R, 8).int().cuda()
    begin = torch.tensor([0, 3, 15, 60, 100])
    cs = _angles(200)
    q, k, v = (torch.randn((steps, R, x, 128), generator=g).to(dt).cuda() for x in (hq, h, h))
    cache0 = P.kv8_cache(R * 8, h, bs)
    for r, n in enumerate(begin.tolist()):
        if n:
            t = torch.arange(n)
            slots = table[r].cpu().long()[t // bs] * bs + t % bs
            rows = torch.randn((2, n, h, 128), generator=g).to(dt).cuda()
            P.append_kv(cache0, rows[0], rows[1], slots.cuda(), t.cuda(), cs)

    def step(cache, lens, q, k, v):
        slots = table.gather(1, (lens // bs).long()[:, None])[:, 0].long() * bs + lens % bs
        qr = P.append_kv(cache, k, v, slots, lens, cs, q)
        lens += 1
        out, lse = P.attention_kv8(qr, cache, table, lens, return_lse=True)
        return out, lse, P.read_kv8(cache, slots, dt)

    cache, lens = cache0.clone(), begin.int().cuda()
    eager = [step(cache, lens, q[i], k[i], v[i]) for i in range(steps)]
    cache2, lens2 = cache0.clone(), begin.int().cuda()
    one = [x[0].clone() for x in (q, k, v)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache2, lens2, *one)
    torch.cuda.current_stream().wait_stream(side)
    cache2.copy_(cache0)
    lens2.copy_(begin.int())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = step(cache2, lens2, *one)
    for i in range(steps):
        for x, y in zip(one, (q, k, v)):
            x.copy_(y[i])
        graph.replay()
        for a, b in zip(res, eager[i]):
            assert torch.equal(a, b)
    assert torch.equal(cache, cache2) and torch.equal(lens, lens2)
    K.check_device_error(cache.device)


@pytest.mark.parametrize("rows", [1, 40])
def test_two_graphs_at_once(rows):
    probs = [_problem([(rows, 3000 + 100 * i), (1, 9), (rows, 1200)], 8, 2, 16, torch.bfloat16,
                      60 + i, cols_more=_wide(40, 3, 8, 2)) for i in range(2)]
    assert _tiles(probs[0][2], rows, 8, 2, 16) == (rows == 40)
    args = [[x.cuda() for x in p] for p in probs]
    want = [P.attention_kv8(*a, rows) for a in args]
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(P.attention_kv8(*a, rows))
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
    K.check_device_error(outs[0].device)


def test_calls_on_other_streams():
    """Four streams, each appending to and attending over its own cache, beside one another."""
    g = torch.Generator().manual_seed(9)
    cs = _angles(600)
    data = [[torch.randn((500, x, 128), generator=g).bfloat16().cuda() for x in (8, 2, 2)]
            for _ in range(4)]
    table = torch.arange(32).int().cuda()[None]
    start, pos = torch.tensor([0, 500]).int().cuda(), torch.arange(500).cuda()
    lens = torch.tensor([500]).int().cuda()

    def work(q, k, v):
        cache = P.kv8_cache(32, 2)
        q = P.append_kv(cache, k, v, pos, pos, cs, q)
        return P.attention_kv8(q, cache, table, lens, start, 500)

    want = [work(*d) for d in data]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in data]
    got = []
    for _ in range(3):
        for s, d in zip(streams, data):
            with torch.cuda.stream(s):
                got.append(work(*d))
    torch.cuda.synchronize()
    for i, o in enumerate(got):
        assert torch.equal(o, want[i % 4])


@pytest.mark.parametrize("rows", [1, 30])
def test_offsets_beyond_32_bits(rows):
    """Blocks at both ends of a cache of 5.4 GB."""
    g = torch.Generator().manual_seed(rows)
    nb, h, hq, n = 1_280_000, 1, 4, 700
    big = torch.empty((nb, h, 33, 128), dtype=torch.uint8, device="cuda")
    ids = torch.cat([torch.arange(22), torch.arange(nb - 22, nb)])
    big[ids.cuda()] = 0
    small = P.kv8_cache(44, h)
    order = torch.randperm(44, generator=g)
    t = torch.arange(n)
    k, v = (torch.randn((n, h, 128), generator=g).bfloat16().cuda() for _ in range(2))
    q = torch.randn((rows, hq, 128), generator=g).bfloat16().cuda()
    far, near = ids[order[t // 16]] * 16 + t % 16, order[t // 16] * 16 + t % 16
    P.append_kv(big, k, v, far.cuda())
    P.append_kv(small, k, v, near.cuda())
    assert torch.equal(big[ids.cuda()], small)
    assert torch.equal(P.read_kv8(big, far.cuda(), torch.bfloat16),
                       P.read_kv8(small, near.cuda(), torch.bfloat16))
    cols = _wide(30, 1, hq, h)
    table = torch.zeros((2, 1, max(44, cols)), dtype=torch.int32)
    table[0, 0, :44], table[1, 0, :44] = ids[order].int(), order.int()
    start, lens = torch.tensor([0, rows]).int().cuda(), torch.tensor([n]).int().cuda()
    a, b = (P.attention_kv8(q, c, tb.cuda(), lens, start, rows) for c, tb in zip((big, small), table))
    assert torch.equal(a, b)
    K.check_device_error(big.device)


@pytest.mark.parametrize("hq,h,n", [(4, 1, 200_003), (28, 4, 40_000)])
def test_long_sequences(hq, h, n):
    dt = torch.bfloat16
    q, cache, table, lens, _ = _problem([(1, n)], hq, h, 64, dt, n)
    _check(*_attend(q, cache, table, lens), O8.attend(q, cache, table, lens, None), dt)


@pytest.mark.parametrize("rows", [2, 40])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_query_rows_that_are_not_finite(dt, rows):
    """They are NaN themselves and change nothing in the others."""
    q, cache, table, lens, start = _problem([(rows, 200), (rows, 90)], 8, 2, 16, dt, 33,
                                            cols_more=_wide(40, 2, 8, 2))
    assert _tiles(table, rows, 8, 2, 16) == (rows == 40)
    ref = O8.attend(q, cache, table, lens, start, one_part=True)
    q[1, 3, 5], q[rows, 0, 100] = math.nan, math.inf
    out, lse = _attend(q, cache, table, lens, start, rows)
    bad = torch.zeros(out.shape[:2], dtype=torch.bool)
    bad[1, 3] = bad[rows, 0] = True
    assert out.cpu()[bad].isnan().all() and lse.cpu()[bad].isnan().all()
    want = ref[0].clone()
    want[bad] = math.nan
    _check(out, None, (want, *ref[1:]), dt)


def test_a_bound_above_the_rows_and_a_padded_batch():
    """max_query_len and the rows behind the last sequence change nothing but the time."""
    dt = torch.float16
    q, cache, table, lens, start = _problem([(3, 100), (0, 40), (2, 64)], 6, 2, 16, dt, 8,
                                            spare_rows=500)
    ref = O8.attend(q, cache, table, lens, start, one_part=True)
    for most in (3, 17, 400, 10 ** 6):
        out, lse = _attend(q, cache, table, lens, start, most)
        _check(out, lse, ref, dt)
        assert not out[5:].any() and (lse[5:] == -math.inf).all()
        held = torch.full_like(q, 3.0).cuda()
        _attend(q, cache, table, lens, start, most, out=held)
        assert (held[5:] == 3.0).all() and torch.equal(held[:5], out[:5])


def test_in_place_and_aliased():
    """The output may be the query itself; the keys and values may be views of one tensor."""
    dt = torch.bfloat16
    q, cache, table, lens, start = _problem([(4, 90), (1, 300)], 4, 2, 16, dt, 21)
    want, _ = _attend(q, cache, table, lens, start, 4)
    own = q.cuda()
    assert P.attention_kv8(own, cache.cuda(), table.cuda(), lens.cuda(), start.cuda(), 4,
                           out=own) is own
    assert torch.equal(own, want)
    kv = torch.randn((20, 2, 128), generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    a = P.kv8_cache(4, 2)
    P.append_kv(a, kv, kv, torch.arange(20).cuda())
    both = P.read_kv8(a, torch.arange(20).cuda(), dt)
    assert torch.equal(both[0], both[1])


def test_a_captured_append_reads_its_inputs_again():
    cache = P.kv8_cache(2, 1)
    k = torch.ones((4, 1, 128), dtype=torch.bfloat16, device="cuda")
    slots = torch.arange(4).cuda()
    P.append_kv(cache, k, k, slots)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        P.append_kv(cache, k, k, slots)
    k.mul_(4)
    graph.replay()
    assert (P.read_kv8(cache, slots, torch.bfloat16) == 4).all()


def test_component_speed_times_the_8bit_stages():
    from kvserve_hpdps_b200.offline import component_speed as CS
    rows = {r["stage"]: r for r in CS.run_serving(tokens=500, requests=5, chunk=40, q_heads=8,
                                                  heads=2, iters=2, warmup=1)}
    for stage in ("append8", "read8", "attn8_decode", "attn8_chunk", "attn8_cross"):
        assert rows[stage]["ms"] > 0
    # e4m3 below 448 2^e: half a step of 2^-4 at most, and exact powers of two between
    assert rows["summary"]["cosine_8bit"] > 1 - 2 ** -8 and rows["summary"]["device_error"] == 0
    assert rows["summary"]["rel_mse_8bit"] < rows["summary"]["rel_mse"]
