"""What the paged-cache operators refuse (no GPU needed), and the oracle's layout."""

import math

import pytest
import torch

import paged_oracle as O
from kvserve_hpdps_b200.ops import paged as P

BF, FP = torch.bfloat16, torch.float16


def _kv(t=4, h=2, dt=BF):
    return torch.zeros((t, h, 128), dtype=dt)


def _layer(h=2, dt=BF):
    return torch.zeros((2, 3, 16, h, 128), dtype=dt)


def test_row_bytes_and_allocation():
    assert [P.kv4_row_bytes(g) for g in (32, 64, 128)] == [160, 144, 136]
    c = P.kv4_cache(3, 2, 32, 128, device="cpu")
    assert c.shape == (3, 2, 32, 136) and c.dtype == torch.uint8 and not c.any()
    for bad in (dict(group_size=16), dict(block_size=8), dict(block_size=0)):
        with pytest.raises(ValueError):
            P.kv4_cache(3, 2, device="cpu", **bad)


def test_oracle_packs_what_it_unpacks():
    g = torch.Generator().manual_seed(0)
    for ng in (1, 2, 4):
        codes = torch.randint(0, 16, (2, 3, 2, 16, 128), generator=g)
        step = torch.rand((2, 3, 2, 16, ng), generator=g).to(BF)
        mid = torch.randn((2, 3, 2, 16, ng), generator=g).to(BF)
        c = O.pack(codes, step, mid)
        assert c.shape[3] == P.kv4_row_bytes(128 // ng)
        assert all(torch.equal(a, b) for a, b in zip(O.unpack(c, BF), (codes, step, mid)))
    for v in (0, 1):
        assert sorted(O.nibble(v).tolist()) == list(range(128))


@pytest.mark.parametrize("change,error", [
    (dict(key=_kv(dt=torch.float32)), TypeError),
    (dict(value=_kv(dt=FP)), TypeError),
    (dict(value=_kv(t=5)), ValueError),
    (dict(key=torch.zeros(4, 2, 64, dtype=BF)), ValueError),
    (dict(cache=_layer(dt=FP)), TypeError),
    (dict(cache=_layer(h=4)), ValueError),
    (dict(cache=torch.zeros(3, 3, 16, 2, 128, dtype=BF)), ValueError),
    (dict(cache=torch.zeros(2, 3, 16, 2, 132, dtype=BF)[..., 4:]), ValueError),
    (dict(cache=torch.zeros(3, 2, 16, 150, dtype=torch.uint8)), ValueError),
    (dict(cache=torch.zeros(3, 2, 24, 144, dtype=torch.uint8)), ValueError),
    (dict(cache=torch.zeros(3, 16, 2, 144, dtype=torch.uint8).transpose(1, 2)), ValueError),
    (dict(slot_mapping=torch.zeros(5, dtype=torch.int64)), ValueError),
    (dict(slot_mapping=torch.zeros(4)), TypeError),
    (dict(slot_mapping=torch.zeros((4, 1), dtype=torch.int64)), TypeError),
    (dict(positions=torch.zeros(4, dtype=torch.int64)), ValueError),
    (dict(cos_sin=torch.zeros(8, 128)), ValueError),
    (dict(positions=torch.zeros(3, dtype=torch.int64), cos_sin=torch.zeros(8, 128)), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64), cos_sin=torch.zeros(8, 120)), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64), cos_sin=torch.zeros(8, 144)), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64), cos_sin=torch.zeros(8, 0)), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64),
          cos_sin=torch.zeros(8, 128, dtype=torch.float64)), TypeError),
    (dict(query=_kv()), ValueError),
    (dict(query_out=_kv()), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64), cos_sin=torch.zeros(8, 128),
          query=_kv(t=3)), ValueError),
    (dict(positions=torch.zeros(4, dtype=torch.int64), cos_sin=torch.zeros(8, 128),
          query=_kv(), query_out=_kv(t=3)), ValueError),
    (dict(), ValueError),  # everything fits, but nothing is on a GPU
])
def test_append_refuses(change, error):
    args = dict(cache=_layer(), key=_kv(), value=_kv(),
                slot_mapping=torch.zeros(4, dtype=torch.int64))
    args.update(change)
    with pytest.raises(error):
        P.append_kv(**args)


@pytest.mark.parametrize("change,error", [
    (dict(cache=_layer()), TypeError),
    (dict(dtype=torch.float32), TypeError),
    (dict(slot_mapping=torch.zeros(4)), TypeError),
    (dict(out=torch.zeros(2, 4, 2, 64, dtype=BF)), ValueError),
    (dict(out=torch.zeros(2, 4, 2, 128, dtype=FP)), ValueError),
    (dict(), ValueError),
])
def test_read_refuses(change, error):
    args = dict(cache=P.kv4_cache(3, 2, device="cpu"), dtype=BF,
                slot_mapping=torch.zeros(4, dtype=torch.int64))
    args.update(change)
    with pytest.raises(error):
        P.read_kv4(**args)


@pytest.mark.parametrize("change,error", [
    (dict(query=_kv(dt=torch.float32)), TypeError),
    (dict(query=_kv(h=3)), ValueError),
    (dict(query=_kv(t=1)), ValueError),
    (dict(cache=_layer()), TypeError),
    (dict(block_table=torch.zeros((2, 3), dtype=torch.int64)), TypeError),
    (dict(block_table=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(seq_lens=torch.zeros(2, dtype=torch.int64)), TypeError),
    (dict(seq_lens=torch.zeros(3, dtype=torch.int32)), TypeError),
    (dict(max_query_len=2), ValueError),
    (dict(scale=0.0), ValueError),
    (dict(scale=math.inf), ValueError),
    (dict(query_start=torch.zeros(2, dtype=torch.int32)), TypeError),
    (dict(query_start=torch.zeros(3, dtype=torch.int32), max_query_len=0), ValueError),
    (dict(out=_kv(t=3, h=4)), ValueError),
    (dict(out=_kv(h=4, dt=FP)), ValueError),
    (dict(), ValueError),
])
def test_attention_refuses(change, error):
    args = dict(query=_kv(h=4), cache=P.kv4_cache(3, 2, device="cpu"),
                block_table=torch.zeros((2, 3), dtype=torch.int32),
                seq_lens=torch.zeros(2, dtype=torch.int32))
    args.update(change)
    with pytest.raises(error):
        P.attention_kv4(**args)


def test_oracle_attention_is_softmax():
    g = torch.Generator().manual_seed(1)
    cache = O.pack(torch.randint(0, 16, (2, 2, 1, 16, 128), generator=g),
                   torch.rand((2, 2, 1, 16, 2), generator=g).to(BF),
                   torch.randn((2, 2, 1, 16, 2), generator=g).to(BF))
    q = torch.randn((1, 3, 128), generator=g).to(BF)
    out, lse, tol, _ = O.attend(q, cache, torch.tensor([[1, 0]]).int(),
                                torch.tensor([20]).int(), None)
    x = O.values(cache, BF)[0]
    k, v = (y[[1, 0], 0].flatten(0, 1)[:20] for y in x)
    w = q[0].double() @ k.T / math.sqrt(128)
    assert torch.allclose(out[0], torch.softmax(w, -1) @ v, atol=1e-12)
    assert torch.allclose(lse[0], torch.logsumexp(w, -1), atol=1e-12)
    assert (tol > 0).all()
