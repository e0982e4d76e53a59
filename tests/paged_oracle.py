"""Plain 64-bit forms of the paged-cache operators, on the CPU, for the tests."""

import math

import torch

D = 128


def half_step(dt):
    """Largest relative error of one rounding to ``dt``."""
    return torch.finfo(dt).eps / 2


def rotate(x, table, pos, interleaved):
    """(rotated rows, sum of magnitudes that each element was added up from), fp64."""
    x, t = x.double().cpu(), table.double().cpu()[pos.long().cpu()][:, None]
    rd = t.shape[-1]
    y, mag = x.clone(), x.abs()
    c, s = t[..., :rd // 2], t[..., rd // 2:]
    if interleaved:
        i0, i1 = slice(0, rd, 2), slice(1, rd, 2)
    else:
        i0, i1 = slice(0, rd // 2), slice(rd // 2, rd)
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    mag[..., i0] = (a * c).abs() + (b * s).abs()
    mag[..., i1] = (b * c).abs() + (a * s).abs()
    return y, mag


def nibble(value):
    """Place of each channel's code among a row's 128 nibbles."""
    d = torch.arange(D)
    q, r = d // 32, d % 32
    if value:
        return (r // 4) * 16 + q * 4 + r % 4
    return (r // 8) * 32 + q * 8 + r % 8


def unpack(cache, dt):
    """(codes [2, nb, H, bs, 128] int64, step, mid [2, nb, H, bs, ng] in ``dt``) of a
    4-bit cache on the CPU."""
    nb, h, bs, rb = cache.shape
    ng = (rb - 128) // 8
    rec = cache.contiguous().view(nb, h, bs * rb)
    codes, steps, mids = [], [], []
    for v in range(2):
        rows = rec[..., 64 * bs * v:64 * bs * (v + 1)].reshape(nb, h, bs, 64).long()
        nib = torch.stack([rows & 15, rows >> 4], -1).flatten(-2)
        codes.append(nib[..., nibble(v)])
        at = 128 * bs + 4 * ng * bs * v
        m = rec[..., at:at + 4 * ng * bs].contiguous().view(dt).view(nb, h, bs, ng, 2)
        steps.append(m[..., 0])
        mids.append(m[..., 1])
    return torch.stack(codes), torch.stack(steps), torch.stack(mids)


def pack(codes, step, mid):
    """A 4-bit cache (uint8, CPU) of codes and metadata laid out as unpack() returns them."""
    _, nb, h, bs, _ = codes.shape
    ng = step.shape[-1]
    parts, metas = [], []
    for v in range(2):
        nib = torch.empty((nb, h, bs, D), dtype=torch.uint8)
        nib[..., nibble(v)] = codes[v].to(torch.uint8)
        parts.append((nib[..., 0::2] | (nib[..., 1::2] << 4)).reshape(nb, h, -1))
        metas.append(torch.stack([step[v], mid[v]], -1).reshape(nb, h, -1).view(torch.uint8))
    return torch.cat(parts + metas, -1).view(nb, h, bs, 128 + 8 * ng)


def values(cache, dt):
    """fp64 values [2, nb, H, bs, 128] of a 4-bit cache on the CPU, and their mids and steps
    spread over the channels."""
    c, s, m = unpack(cache, dt)
    g = D // s.shape[-1]
    s, m = s.double().repeat_interleave(g, -1), m.double().repeat_interleave(g, -1)
    return m + (c - 8) * s, m, s


def attend(q, cache, table, lens, start, scale=None, tiles=False):
    """fp64 (out, lse, tolerance) of attention over a 4-bit cache; NaN rows where
    no sequence has a row.  Tolerance, element by element, of an implementation that
    takes scores and sums in fp32 and probabilities times steps in fp16, before
    the output's own rounding:
      scores: 128 products and the group terms in fp32, with 2^-23 of the sum of their
        magnitudes an addition at worst and 24 of them in a chain (rounded up: 2^-18), which
        moves each weight by that share;
      weights: fp16's half step, 2^-11, of p |code - 8| step; below fp16's
        normal range half of 2^-24 of the largest step, times 8;
      exponentials, sums and the division: 2^-18 of p |v| together.
    ``tiles``: the kernel for many rows rounds more. Keys and values become fp16, so a
      key's product with the query is off by at most half a step, 2^-11, of each
      |q_d k_d|, which adds to the scores' error; a value by 2^-11 |v|, and p itself
      (there is no step in it) by 2^-11 p: together 2^-10 of p |v| and the
      product of both errors, in the place of 2^-11 of p |code - 8| step.
    """
    dt = q.dtype
    q, cache = q.double().cpu(), cache.cpu()
    table, lens = table.cpu().long(), lens.cpu().long()
    T, hq, _ = q.shape
    h = cache.shape[1]
    G = hq // h
    x, mid, step = values(cache, dt)
    scale = 1 / math.sqrt(D) if scale is None else scale
    starts = list(range(len(lens) + 1)) if start is None else start.cpu().tolist()
    out = torch.full((T, hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, hq), math.nan, dtype=torch.float64)
    tol = torch.zeros((T, hq, D), dtype=torch.float64)
    ltol = torch.zeros((T, hq), dtype=torch.float64)
    for r, n in enumerate(lens.tolist()):
        a, b = starts[r], starts[r + 1]
        used = table[r, :(n + cache.shape[2] - 1) // cache.shape[2]]
        k, v = x[0][used], x[1][used]
        k, v = (y.permute(1, 0, 2, 3).reshape(h, -1, D)[:, :n] for y in (k, v))
        dev = (x[1] - mid[1])[used].abs().permute(1, 0, 2, 3).reshape(h, -1, D)[:, :n]
        kmag = (mid[0].abs() + 15 * step[0])[used].permute(1, 0, 2, 3).reshape(h, -1, D)[:, :n]
        vmag = (mid[1].abs() + (x[1] - mid[1]).abs())[used].permute(1, 0, 2, 3)
        vmag = vmag.reshape(h, -1, D)[:, :n]
        top = step[1][used].max() if n else 0.0
        for i in range(b - a):
            seen = n - (b - a) + i + 1
            qi = q[a + i].view(h, G, D)
            if seen <= 0:
                out[a + i], lse[a + i] = 0.0, -math.inf
                continue
            w = torch.einsum("hgd,hld->hgl", qi, k[:, :seen]) * scale
            werr = torch.einsum("hgd,hld->hgl", qi.abs(), kmag[:, :seen]) * abs(scale) * 2 ** -18
            if tiles:
                werr = werr + 2 ** -11 * abs(scale) * torch.einsum("hgd,hld->hgl", qi.abs(),
                                                                   k[:, :seen].abs())
            z = torch.logsumexp(w, -1, keepdim=True)
            p = torch.exp(w - z)
            out[a + i] = torch.einsum("hgl,hld->hgd", p, v[:, :seen]).reshape(hq, D)
            lse[a + i] = z.reshape(hq)
            e = torch.einsum("hgl,hld->hgd", p * (2 * werr.amax(-1, keepdim=True) + 2 ** -18),
                             vmag[:, :seen])
            if tiles:
                e = e + (2 ** -10 + 2 ** -21) * torch.einsum("hgl,hld->hgd", p, v[:, :seen].abs())
            else:
                e = e + 2 ** -11 * torch.einsum("hgl,hld->hgd", p, dev[:, :seen])
            e = e + 8 * 2 ** -25 * top * seen * torch.exp(w.amax(-1, keepdim=True) - z)
            tol[a + i] = e.reshape(hq, D)
            ltol[a + i] = werr.amax(-1).reshape(hq) + 2 ** -20 * (1 + lse[a + i].abs())
    return out, lse, tol, ltol
