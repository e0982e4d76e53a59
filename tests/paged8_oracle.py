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
