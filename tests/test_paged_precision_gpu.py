"""attention_kv4, many rows: scores as exact as fp32's in both types, and outputs that are off by
the roundings that the kernel makes and no more."""

import math

import pytest
import torch

import paged_oracle as O
from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import paged as P

pytestmark = pytest.mark.gpu

BF, FP = torch.bfloat16, torch.float16


def one_head(q, k, v, seen, scale):
    """fp64 (out, lse, sum of p |v|, largest score error) of query rows ``q`` [n, 128] of one head
    over keys and values [L, 128]; row i sees the first ``seen[i]``.  The score error is that of
    fp32 sums: 2^-18 of the sum of magnitudes, as in paged_oracle.attend."""
    w = q.double() @ k.T * scale
    mag = q.double().abs() @ k.abs().T * scale * 2 ** -18
    hide = torch.arange(k.shape[0])[None] >= seen[:, None]
    w = w.masked_fill(hide, -math.inf)
    mag = mag.masked_fill(hide, 0.0)
    z = torch.logsumexp(w, -1, keepdim=True)
    p = torch.exp(w - z)
    return p @ v, z[:, 0], p @ v.abs(), mag.amax(-1)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("g_size", [32, 64, 128])
@pytest.mark.parametrize("mids,size", [(0.3, 0.5), (0.3, 4.0), (8.0, 4.0)])
def test_scores_are_those_of_fp32(dt, g_size, mids, size):
    """Steps of all bits, mids of the steps' size and far above them; with large queries one key
    has most of the weight, and lse shows its score's error (keys rounded to fp16: 15 times the
    bound in fp16 caches).  An output is off by the
    weights' rounding, 2^-11 of p |v|, in bf16 caches by the values' as well, twice the scores'
    error, and its own rounding; 2^-17 of p |v| covers the exponentials and fp32's sums."""
    g = torch.Generator().manual_seed(g_size)
    hq, h, bs, n, length, ng = 8, 2, 16, 150, 1100, 128 // g_size
    nb = -(-length // bs)
    codes = torch.randint(0, 16, (2, nb, h, bs, 128), generator=g)
    step = (0.1 + 0.1 * torch.rand((2, nb, h, bs, ng), generator=g)).to(dt)
    mid = (mids * torch.randn((2, nb, h, bs, ng), generator=g)).to(dt)
    cache = O.pack(codes, step, mid)
    table = torch.randperm(nb, generator=g).int()[None]
    q = (torch.randn((n, hq, 128), generator=g) * size).to(dt)
    wide = torch.full((1, (6 << 20) // (n * hq * bs) + 1), -1, dtype=torch.int32)
    wide[:, :nb] = table  # room enough for the kernel for many rows
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), wide.cuda(),
                               torch.tensor([length]).int().cuda(),
                               torch.tensor([0, n]).int().cuda(), n, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    x = O.values(cache, dt)[0][:, table[0].long()].permute(0, 2, 1, 3, 4).flatten(2, 3)
    seen = length - n + 1 + torch.arange(n)
    for head in range(hq):
        k, v = x[0, head // 4, :length], x[1, head // 4, :length]
        want, z, pv, werr = one_head(q[:, head], k, v, seen, 1 / math.sqrt(128))
        got, l = out[:, head].double().cpu(), lse[:, head].double().cpu()
        assert ((l - z).abs() <= werr + 2 ** -20 * (1 + z.abs())).all()
        tol = (2 ** -11 * (2 if dt == BF else 1) + 2 ** -17 + 2 * werr[:, None]) * pv
        tol = tol + O.half_step(dt) * (want.abs() + tol) + 2 ** -24
        assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())
        # on the whole: each rounding is 1 / sqrt 3 of half a step by its root mean square at
        # most, those of the weights are independent and p v has alternating signs, so that they
        # add up to less than the output's own; twice half a step leaves room for both
        off = (got - want).norm() / want.norm()
        assert off <= 2 * O.half_step(dt)


@pytest.mark.parametrize("dt", [BF, FP])
@pytest.mark.parametrize("g_size", [32, 64, 128])
@pytest.mark.parametrize("rows,length", [(1, 900), (1, 40), (7, 500)])
def test_few_rows_weights(dt, g_size, rows, length):
    """The kernel for few rows: in bf16 caches weights times steps are fp16, 2^-11 of p |v - mid|; in
    fp16 ones two parts of fp16, which leave 2^-22 at most."""
    g = torch.Generator().manual_seed(g_size + rows)
    hq, h, bs, ng = 8, 2, 16, 128 // g_size
    nb = -(-length // bs)
    codes = torch.randint(0, 16, (2, nb, h, bs, 128), generator=g)
    step = (0.1 + 0.1 * torch.rand((2, nb, h, bs, ng), generator=g)).to(dt)
    mid = (0.1 * torch.randn((2, nb, h, bs, ng), generator=g)).to(dt)
    cache = O.pack(codes, step, mid)
    table = torch.randperm(nb, generator=g).int()[None]
    q = torch.randn((rows, hq, 128), generator=g).to(dt)
    out, lse = P.attention_kv4(q.cuda(), cache.cuda(), table.cuda(),
                               torch.tensor([length]).int().cuda(),
                               torch.tensor([0, rows]).int().cuda(), rows, return_lse=True)
    torch.cuda.synchronize()
    K.check_device_error(out.device)
    x, mids, _ = O.values(cache, dt)
    x, mids = (y[:, table[0].long()].permute(0, 2, 1, 3, 4).flatten(2, 3) for y in (x, mids))
    seen = length - rows + 1 + torch.arange(rows)
    for head in range(hq):
        k, v = x[0, head // 4, :length], x[1, head // 4, :length]
        want, z, pv, werr = one_head(q[:, head], k, v, seen, 1 / math.sqrt(128))
        dev = one_head(q[:, head], k, v - mids[1, head // 4, :length], seen, 1 / math.sqrt(128))[2]
        got, l = out[:, head].double().cpu(), lse[:, head].double().cpu()
        assert ((l - z).abs() <= werr + 2 ** -20 * (1 + z.abs())).all()
        tol = (2 ** -11 * dev if dt == BF else 2 ** -22 * dev) + (2 ** -17 + 2 * werr[:, None]) * pv
        # steps far below the largest, 2^-24 of it times 8 a weight: none here
        tol = tol + O.half_step(dt) * (want.abs() + tol) + 2 ** -25
        assert ((got - want).abs() <= tol).all(), float(((got - want).abs() / tol).max())
