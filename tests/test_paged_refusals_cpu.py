"""More calls that the paged-cache operators refuse, told before anything runs (no GPU needed)."""

import pytest
import torch

from kvserve_hpdps_b200.ops import paged as P

BF = torch.bfloat16


def _append(**change):
    args = dict(cache=torch.zeros((2, 3, 16, 2, 128), dtype=BF),
                key=torch.zeros((4, 2, 128), dtype=BF), value=torch.zeros((4, 2, 128), dtype=BF),
                slot_mapping=torch.zeros(4, dtype=torch.int64),
                positions=torch.zeros(4, dtype=torch.int64), cos_sin=torch.zeros(8, 128),
                query=torch.zeros((4, 4, 128), dtype=BF))
    args.update(change)
    return P.append_kv(**args)


def _attend(**change):
    args = dict(query=torch.zeros((4, 4, 128), dtype=BF), cache=P.kv4_cache(3, 2, device="cpu"),
                block_table=torch.zeros((2, 3), dtype=torch.int32),
                seq_lens=torch.zeros(2, dtype=torch.int32))
    args.update(change)
    return P.attention_kv4(**args)


def _read(**change):
    args = dict(cache=P.kv4_cache(3, 2, device="cpu"), dtype=BF,
                slot_mapping=torch.zeros(4, dtype=torch.int64))
    args.update(change)
    return P.read_kv4(**args)


def _grad(*shape, dtype=BF):
    return torch.zeros(shape, dtype=dtype, requires_grad=True)


@pytest.mark.parametrize("call,name,t", [
    (_append, "key", _grad(4, 2, 128)), (_append, "value", _grad(4, 2, 128)),
    (_append, "query", _grad(4, 4, 128)), (_append, "cos_sin", _grad(8, 128, dtype=torch.float32)),
    (_append, "cache", _grad(2, 3, 16, 2, 128)), (_append, "query_out", _grad(4, 4, 128)),
    (_attend, "query", _grad(4, 4, 128)), (_attend, "out", _grad(4, 4, 128)),
    (_read, "out", _grad(2, 4, 2, 128)),
])
def test_gradients_are_not_lost_without_a_word(call, name, t):
    with pytest.raises(ValueError, match="backward"):
        call(**{name: t})
    for ok in (t.detach(), t):
        with torch.no_grad(), pytest.raises(ValueError, match="CUDA"):  # all else fits
            call(**{name: ok})


@pytest.mark.parametrize("call,name,t", [
    (_append, "query_out", torch.zeros((1, 4, 128), dtype=BF).expand(4, 4, 128)),
    (_append, "query_out", torch.zeros((4, 1, 128), dtype=BF).expand(4, 4, 128)),
    (_append, "query_out", torch.zeros(2048, dtype=BF).as_strided((4, 4, 128), (384, 128, 1))),
    (_append, "cache", torch.zeros((2, 1, 16, 2, 128), dtype=BF).expand(2, 3, 16, 2, 128)),
    (_append, "cache", torch.zeros((1, 3, 16, 2, 128), dtype=BF).expand(2, 3, 16, 2, 128)),
    (_append, "cache", P.kv4_cache(1, 2, device="cpu").expand(3, 2, 16, 144)),
    (_append, "cache", P.kv4_cache(3, 1, device="cpu").expand(3, 2, 16, 144)),
    (_attend, "out", torch.zeros((1, 4, 128), dtype=BF).expand(4, 4, 128)),
])
def test_what_is_written_does_not_overlap_itself(call, name, t):
    with pytest.raises(ValueError, match="overlap"):
        call(**{name: t})


@pytest.mark.parametrize("call,out", [(_append, "query_out"), (_attend, "out")])
def test_outputs_are_the_query_or_apart_from_it(call, out):
    buf = torch.zeros((5, 4, 128), dtype=BF)
    with pytest.raises(ValueError, match="overlap"):
        call(query=buf[:4], **{out: buf[1:]})
    for ok in (buf[:4], torch.zeros((4, 4, 128), dtype=BF)):
        with pytest.raises(ValueError, match="CUDA"):
            call(query=buf[:4], **{out: ok})


def test_layouts_that_do_not_overlap_are_taken():
    """Slices of wider buffers, head-major blocks, one layer of several, blocks of one token."""
    for cache in (torch.zeros((2, 3, 2, 16, 128), dtype=BF).transpose(2, 3),
                  torch.zeros((3, 2, 16, 2, 128), dtype=BF),
                  torch.zeros((3, 5, 2, 16, 2, 128), dtype=BF)[:, 1],
                  torch.zeros((2, 3, 1, 2, 128), dtype=BF),
                  torch.zeros((3, 4, 2, 16, 144), dtype=torch.uint8)[:, 1],
                  P.kv4_cache(0, 2, device="cpu")):
        with pytest.raises(ValueError, match="CUDA"):
            _append(cache=cache)
    wide = torch.zeros((4, 9, 128), dtype=BF)
    with pytest.raises(ValueError, match="CUDA"):
        _append(query=wide[:, :4], query_out=wide[:, 4:8])
    with pytest.raises(ValueError, match="CUDA"):
        _attend(query=wide[:, :4], out=wide[:, 5:])
