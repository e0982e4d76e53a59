"""attention_kv4, many rows: CTAs that go from pieces with one query tile to pieces with two, over
heads whose keys and values have different scales, against the 64-bit form."""

import pytest
import torch

import paged_oracle as O
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P

pytestmark = pytest.mark.gpu

# query rows, cached tokens, query heads, kv heads, group size
SHAPES = {
    "drafts": ([48] * 8, [4000] * 8, 28, 4, 64),
    "two_chunks": ([896] * 2, [3000] * 2, 28, 4, 128),
    "one_chunk": ([330], [8192], 32, 8, 32),
    "decodes_and_chunk": ([1] * 48 + [512], [4000] * 48 + [4096], 28, 4, 64),
    "ragged": ([20] * 12 + [100, 20, 20, 20, 100], [2500 + 7 * i for i in range(17)], 32, 8, 64),
}


def _call(name, dt, seed):
    """A call's tensors on the CPU; odd heads' keys and values are 2^-8 of the even ones'."""
    queries, lens, hq, h, g_size = SHAPES[name]
    g = torch.Generator().manual_seed(seed)
    nb, bs, ng = 331, 16, 128 // g_size
    codes = torch.randint(0, 16, (2, nb, h, bs, 128), generator=g)
    size = torch.exp2(-8.0 * (torch.arange(h) % 2))[:, None, None]
    step = (0.1 + 0.3 * torch.rand((2, nb, h, bs, ng), generator=g)) * size
    mid = 0.3 * torch.randn((2, nb, h, bs, ng), generator=g) * size
    cache = O.pack(codes, step.to(dt), mid.to(dt))
    table = torch.randint(0, nb, (len(lens), -(-max(lens) // bs)), generator=g).int()
    q = (torch.randn((sum(queries), hq, 128), generator=g) * 0.7).to(dt)
    start = torch.tensor([0] + queries).cumsum(0).int()
    return q, cache, table, torch.tensor(lens).int(), start


def _rows_near(out, lse, q, cache, table, lens, start, picks, gone=0):
    """The picked (sequence, row, kv head) against the 64-bit form, head by head.  The first ``gone``
    blocks of ``table`` are not there for the kernel: the form gets a table without them."""
    dt, h = q.dtype, cache.shape[1]
    G = q.shape[1] // h
    for r, i, head in picks:
        n = int(start[r + 1] - start[r])
        seen = int(lens[r]) - n + i + 1 - 16 * gone
        t, at = int(start[r]) + i, slice(head * G, head * G + G)
        want, wlse, tol, ltol = O.attend(q[t:t + 1, at], cache[:, head:head + 1],
                                         table[r:r + 1, gone:], torch.tensor([seen]), None,
                                         tiles=True)
        bound = tol + O.half_step(dt) * (want.abs() + tol)
        d = (out[t:t + 1, at].double().cpu() - want).abs()
        assert (d <= bound).all(), (r, i, head, float((d / bound).max()))
        assert ((lse[t:t + 1, at].double().cpu() - wlse).abs() <= ltol).all(), (r, i, head)


def _picks(name):
    """Rows of every head: the first, of the second query tile, the last; some sequences."""
    queries, _, hq, h, _ = SHAPES[name]
    G = hq // h
    some = [r for r in range(len(queries)) if queries[r] > 1][-6:] + [0, len(queries) - 2]
    return [(r, i, head) for r in sorted({x for x in some if x >= 0}) for head in range(h)
            for i in sorted({0, 128 // G + 1, 180 // G, 255 // G, queries[r] - 1})
            if i < queries[r]]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("name", sorted(SHAPES))
def test_one_tile_pieces_in_front_of_two_tile_pieces(name, dt):
    q, cache, table, lens, start = _call(name, dt, 5)
    args = [x.cuda() for x in (q, cache, table, lens, start)]
    most = max(SHAPES[name][0])
    out, lse = P.attention_kv4(*args, most, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    _rows_near(out, lse, q, cache, table, lens, start, _picks(name))
    for _ in range(4):
        again, l2 = P.attention_kv4(*args, most, return_lse=True)
        assert torch.equal(out, again) and torch.equal(lse, l2)


@pytest.mark.parametrize("name", sorted(SHAPES))
def test_missing_first_blocks_behind_one_tile_pieces(name):
    """The first two blocks of every sequence do not exist: no row takes anything of them."""
    q, cache, table, lens, start = _call(name, torch.bfloat16, 6)
    bad = table.clone()
    bad[:, 0], bad[:, 1] = -1, cache.shape[0]
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), bad.cuda(), lens.cuda(), start.cuda(),
                               max(SHAPES[name][0]), return_lse=True)
    torch.cuda.synchronize()
    assert K.read_device_error(out.device) == 3  # a bound was recorded
    _rows_near(out, lse, q, cache, table, lens, start, _picks(name), gone=2)
