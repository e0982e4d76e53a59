"""What the 8-bit paged cache's operators refuse (no GPU needed), and the oracle's numbers."""

import math

import pytest
import torch

import paged8_oracle as O8
from kvserve_hpdps_b200.ops import paged as P

BF, FP = torch.bfloat16, torch.float16


def _kv(t=4, h=2, dt=BF):
    return torch.zeros((t, h, 128), dtype=dt)


def _cache(nb=3, h=2, bs=16):
    return P.kv8_cache(nb, h, bs, device="cpu")


def test_allocation():
    c = P.kv8_cache(3, 2, 32, device="cpu")
    assert c.shape == (3, 2, 65, 128) and c.dtype == torch.uint8 and not c.any()
    for bad in (0, 8, 24, 1040, -16):
        with pytest.raises(ValueError):
            P.kv8_cache(3, 2, bad, device="cpu")


def test_oracle_codes_are_e4m3():
    c = torch.arange(256, dtype=torch.uint8)
    nan = c % 128 == 127
    want = c.view(torch.float8_e4m3fn).double()
    got = O8.values(c)
    assert torch.equal(got[~nan], want[~nan]) and got[nan].isnan().all()
    x = torch.cat([torch.randn(20000).double() * 100, got[~nan],
                   (got[:126] + got[1:127]) / 2]).clamp(-448, 448)  # ties among them
    assert torch.equal(O8.codes(x), x.float().to(torch.float8_e4m3fn).view(torch.uint8))
    for amax, e in ((448, 0), (449, 1), (224, -1), (225, 0), (1.0, -8), (1e-45, -110), (0, -110)):
        assert O8.exponent(amax) == e


def test_oracle_append_and_read():
    g = torch.Generator().manual_seed(1)
    cache = _cache(4, 2, 32)
    k, v = (torch.randn((40, 2, 128), generator=g).to(BF) for _ in range(2))
    slots = torch.arange(50, 90)
    O8.append(cache, k, v, slots)
    for x, y in zip(O8.read(cache, slots), (k, v)):
        y = y.double()
        assert ((x - y).abs() <= 2 ** -4 * y.abs() + 2 ** -17 * y.abs().max()).all()
    assert not O8.read(cache, torch.tensor([-1, 0, 49, 90])).any()


@pytest.mark.parametrize("change,error", [
    (dict(cache=_cache(h=4)), ValueError),
    (dict(cache=torch.zeros(3, 2, 32, 128, dtype=torch.uint8)), ValueError),
    (dict(cache=torch.zeros(3, 2, 49, 128, dtype=torch.uint8)), ValueError),   # blocks of 24
    (dict(cache=torch.zeros(3, 2, 2081, 128, dtype=torch.uint8)), ValueError),  # of 1040
    (dict(cache=torch.zeros(3, 2, 33, 256, dtype=torch.uint8)[..., ::2]), ValueError),
    (dict(cache=torch.zeros(3, 2, 66, 128, dtype=torch.uint8)[:, :, ::2]), ValueError),
    (dict(cache=torch.zeros(3 * 2 * 33 * 128 + 8, dtype=torch.uint8)[8:].view(3, 2, 33, 128)),
     ValueError),
    (dict(cache=torch.zeros(1, 2, 33, 128, dtype=torch.uint8).expand(3, 2, 33, 128)), ValueError),
    (dict(key=_kv(dt=torch.float32)), TypeError),
    (dict(value=_kv(dt=FP)), TypeError),
    (dict(slot_mapping=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(slot_mapping=torch.zeros(4)), TypeError),
    (dict(query=_kv()), ValueError),
    (dict(key=_kv().requires_grad_()), ValueError),
    (dict(), ValueError),  # everything fits, but nothing is on a GPU
])
def test_append_refuses(change, error):
    args = dict(cache=_cache(), key=_kv(), value=_kv(),
                slot_mapping=torch.zeros(4, dtype=torch.int64))
    args.update(change)
    with pytest.raises(error):
        P.append_kv(**args)


@pytest.mark.parametrize("change,error", [
    (dict(cache=torch.zeros(2, 3, 16, 2, 128, dtype=BF)), TypeError),
    (dict(cache=P.kv4_cache(3, 2, device="cpu")), ValueError),
    (dict(dtype=torch.float32), TypeError),
    (dict(slot_mapping=torch.zeros(4)), TypeError),
    (dict(out=torch.zeros(2, 4, 2, 64, dtype=BF)), ValueError),
    (dict(out=torch.zeros(2, 4, 2, 128, dtype=FP)), ValueError),
    (dict(out=torch.zeros(2, 4, 2, 128, dtype=BF).requires_grad_()), ValueError),
    (dict(), ValueError),
])
def test_read_refuses(change, error):
    args = dict(cache=_cache(), dtype=BF, slot_mapping=torch.zeros(4, dtype=torch.int64))
    args.update(change)
    with pytest.raises(error):
        P.read_kv8(**args)


@pytest.mark.parametrize("change,error", [
    (dict(query=_kv(dt=torch.float32)), TypeError),
    (dict(query=_kv(h=3)), ValueError),
    (dict(query=_kv(t=1)), ValueError),
    (dict(query=_kv(h=4).requires_grad_()), ValueError),
    (dict(cache=torch.zeros(2, 3, 16, 2, 128, dtype=BF)), TypeError),
    (dict(cache=P.kv4_cache(3, 2, device="cpu")), ValueError),
    (dict(cache=torch.zeros(1, 2, 33, 128, dtype=torch.uint8).expand(3, 2, 33, 128)), ValueError),
    (dict(block_table=torch.zeros((2, 3), dtype=torch.int64)), TypeError),
    (dict(block_table=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), TypeError),
    (dict(max_query_len=2), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(scale=math.nan), ValueError),
    (dict(query_start=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(query_start=torch.zeros(3, dtype=torch.int32), max_query_len=0), ValueError),
    (dict(out=_kv(t=3, h=4)), ValueError),
    (dict(out=_kv(h=4, dt=FP)), ValueError),
    (dict(out=_kv(t=1, h=4).expand(4, 4, 128)), ValueError),
    (dict(causal=False), ValueError),
    (dict(), ValueError),
])
def test_attention_refuses(change, error):
    args = dict(query=_kv(h=4), cache=_cache(), block_table=torch.zeros((2, 3), dtype=torch.int32),
                seq_lens=torch.zeros(2, dtype=torch.int32))
    args.update(change)
    with pytest.raises(error):
        P.attention_kv8(**args)


def test_the_4_bit_operators_refuse_8_bit_caches():
    with pytest.raises(ValueError):
        P.read_kv4(_cache(), torch.zeros(4, dtype=torch.int64), BF)
    with pytest.raises(ValueError):
        P.attention_kv4(_kv(h=4), _cache(), torch.zeros((2, 3), dtype=torch.int32),
                        torch.zeros(2, dtype=torch.int32))
