"""Plain forms of the 8-bit paged cache's operators, on the CPU, for the tests."""

import math

import torch

import paged_oracle as O

D, UNIT, LOW = 128, 16, -110

# e4m3 by its definition: sign, 4 bits of exponent (bias 7), 3 of mantissa, 0x7F not a number.
_M = torch.arange(127)
NUMBERS = torch.where(_M < 8, _M.double() / 512,
                      (8 + _M % 8).double() * torch.pow(2.0, (_M // 8 - 10).double()))


def values(codes):
    """fp64 values of uint8 codes."""
    c = codes.long()
    x = torch.cat([NUMBERS, torch.tensor([math.nan], dtype=torch.float64)])[c & 127]
    return torch.where(c >= 128, -x, x)


def codes(x):
    """uint8 codes of fp64 numbers up to 448 in magnitude: nearest, ties to the even code."""
    a = x.abs()
    hi = torch.searchsorted(NUMBERS, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    up, down = NUMBERS[hi] - a, a - NUMBERS[lo]
    pick = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, lo)
    pick = torch.where(torch.isnan(x), 127, pick)
    return (pick + 128 * torch.signbit(x).long() * ~torch.isnan(x)).to(torch.uint8)


def exponent(amax):
    """The smallest e with amax <= 448 * 2^e, at least LOW, of one number."""
    if amax == 0:
        return LOW
    m, e = math.frexp(amax / 448.0)  # amax = 448 m 2^e, m in [0.5, 1); a division by 7 is rounded,
    return max(LOW, e - 1 if m == 0.5 else e)  # but for powers of two times 448 it is exact


def rotate32(x, table, pos, inter):
    """The rotation in fp32, each operation rounded once."""
    rd = table.shape[1]
    x, t = x.float(), table.float()[pos.long()][:, None]
    c, s = t[..., :rd // 2], t[..., rd // 2:]
    y = x.clone()
    i0, i1 = ((slice(0, rd, 2), slice(1, rd, 2)) if inter
              else (slice(0, rd // 2), slice(rd // 2, rd)))
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, b * c + a * s
    return y


def append(cache, k, v, slots, pos=None, table=None, inter=False):
    """The cache (CPU, changed in place) after a call, unit by unit."""
    nb, H, rows, _ = cache.shape
    bs = (rows - 1) // 2
    new = [k.float() if pos is None else rotate32(k, table, pos, inter), v.float()]
    units = {}
    for t, s in enumerate(slots.tolist()):
        if 0 <= s < nb * bs and (pos is None or 0 <= int(pos[t]) < table.shape[0]):
            units.setdefault(s // UNIT, {})[s % UNIT] = t
    for u, toks in units.items():
        b, at = u // (bs // UNIT), u % (bs // UNIT)
        for which in range(2):
            for h in range(H):
                x = new[which][list(toks.values()), h].double()
                fine = torch.isfinite(x)
                amax = float(x[fine].abs().max()) if fine.any() else 0.0
                byte = int(cache[b, h, 2 * bs, 2 * at + which])
                old = LOW if byte > 247 else max(LOW, byte - 127)  # no append writes more
                e = exponent(amax)
                if 0 not in toks:
                    e = max(e, old)
                r = which * bs + at * UNIT
                if 0 not in toks and e > old:
                    y = values(cache[b, h, r:r + UNIT]) * 2.0 ** (old - e)
                    cache[b, h, r:r + UNIT] = codes(y)
                cache[b, h, [r + o for o in toks]] = codes(
                    torch.where(fine, x * 2.0 ** -e, math.nan))
                cache[b, h, 2 * bs, 2 * at + which] = e + 127


def read(cache, slots):
    """fp64 [2, n, H, 128] rows of a cache (CPU); negative slots are zeros."""
    bs = (cache.shape[2] - 1) // 2
    s = slots.long().clamp(min=0)
    out = []
    for which in range(2):
        e = cache[s // bs, :, 2 * bs, 2 * (s % bs // UNIT) + which].double() - 127
        scale = torch.where(e == -127, 0.0, torch.pow(2.0, e))
        x = values(cache[s // bs, :, which * bs + s % bs]) * scale[..., None]
        out.append(torch.where((slots >= 0)[:, None, None], x, 0.0))
    return torch.stack(out)


half_step = O.half_step


def random_cache(g, nb, h, bs, spread=2):
    """Rows like N(0, 1) with outlier key channels, under scales a few powers of two apart (CPU)."""
    x = torch.randn((nb, h, 2 * bs, D), generator=g, dtype=torch.float64) * 40
    x[:, :, :bs, :3] *= 4
    cache = torch.zeros((nb, h, 2 * bs + 1, D), dtype=torch.uint8)
    cache[:, :, :2 * bs] = codes(x.clamp(-448, 448))
    cache[:, :, 2 * bs] = torch.randint(121 - spread, 122 + spread, (nb, h, D), generator=g,
                                        dtype=torch.uint8)
    return cache


def attend(q, cache, table, lens, start, scale=None, causal=True, one_part=None):
    """fp64 (out, lse, tolerance, lse's tolerance) of attention over an 8-bit cache (CPU); NaN rows
    where no sequence has a row.  The tolerance, element by element, of an implementation that takes
    products and sums in fp32 and weights in fp16, before the output's own rounding:
      scores: 128 products summed in fp32, 2^-23 of the sum of their magnitudes an addition and 24 of
        them in a chain (rounded up: 2^-18), which moves each weight by that share;
      weights p 2^e (e the values' exponent): fp16's half step, 2^-11, of p |v|, or 2^-21 where fp16
        takes two parts (fp16 outputs, unless ``one_part``); below fp16's normal range half of
        2^-24 of a unit that is at most 2^-6 of the row's largest weight, times |code|;
      exponentials, sums and the division: 2^-18 of p |v| together.
    """
    q64, table, lens = q.double(), table.long(), lens.long()
    T, hq, _ = q.shape
    bs, h = (cache.shape[2] - 1) // 2, cache.shape[1]
    G = hq // h
    scale = 1 / math.sqrt(D) if scale is None else scale
    part = 2 ** -11 if (q.dtype == torch.bfloat16 if one_part is None else one_part) else 2 ** -21
    starts = list(range(len(lens) + 1)) if start is None else start.tolist()
    out = torch.full((T, hq, D), math.nan, dtype=torch.float64)
    lse = torch.full((T, hq), math.nan, dtype=torch.float64)
    tol, ltol = torch.zeros_like(out), torch.zeros_like(lse)
    for r, n in enumerate(lens.tolist()):
        a, b = starts[r], starts[r + 1]
        t = torch.arange(n)
        kv = read(cache, table[r][t // bs] * bs + t % bs).transpose(1, 2)  # [2, H, n, D]
        k, v = kv[0], kv[1]
        e = cache[table[r][t // bs], :, 2 * bs, 2 * (t % bs // UNIT) + 1].double().T - 127  # [H, n]
        for i in range(b - a):
            seen = max(0, n - (b - a) + i + 1) if causal else n
            if seen == 0:
                out[a + i], lse[a + i] = 0.0, -math.inf
                continue
            qi = q64[a + i].view(h, G, D)
            w = torch.einsum("hgd,hld->hgl", qi, k[:, :seen]) * scale
            werr = torch.einsum("hgd,hld->hgl", qi.abs(), k[:, :seen].abs()) * abs(scale) * 2 ** -18
            z = torch.logsumexp(w, -1, keepdim=True)
            p = torch.exp(w - z)
            out[a + i] = torch.einsum("hgl,hld->hgd", p, v[:, :seen]).reshape(hq, D)
            lse[a + i] = z.reshape(hq)
            share = 2 * werr.amax(-1, keepdim=True) + 2 ** -18 + part
            most = (p * 2.0 ** e[:, None, :seen]).amax(-1)
            mag = (v[:, :seen] * 2.0 ** -e[:, :seen, None]).abs().sum(1)  # of the codes
            tol[a + i] = (torch.einsum("hgl,hld->hgd", p * share, v[:, :seen].abs())
                          + 2 ** -31 * most[..., None] * mag[:, None]).reshape(hq, D)
            ltol[a + i] = (2 * werr.amax(-1) + 2 ** -18 + 2 ** -22 * z[..., 0].abs()).reshape(hq)
    return out, lse, tol, ltol
