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
