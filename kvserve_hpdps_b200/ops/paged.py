"""Operators on the paged KV caches of a serving step.

* :func:`append_kv`: a step's new keys and values into a paged cache (16-bit,
  or held in 8 or 4 bits), the position rotation of keys and queries applied in
  the same launch;
* :func:`attention_kv8`, :func:`attention_kv4`: attention over an 8-bit or 4-bit
  cache without unpacking it first (one token, several draft tokens or a
  prefill chunk per sequence; over 8 bits also cross attention);
* :func:`read_kv8`, :func:`read_kv4`: rows of such a cache as 16-bit values, e.g.
  to hand them to the paths that take 16-bit KV.

A 4-bit cache of one layer is a uint8 tensor ``[num_blocks, heads, block_size,
row_bytes]`` (:func:`kv4_cache`), ``row_bytes = 128 + 1024 / group_size``: 64
bytes of codes for the key and the value of a token each, and per group of
``group_size`` (32, 64 or 128) channels a (step, mid) pair of 16-bit floats
for each of them.  A channel's value is ``mid + (code - 8) * step``.  Inside a
(block, head) the bytes are ordered ``[K codes][V codes][K meta][V meta]``,
each part over the block's tokens (``csrc/kv4.cuh`` has the order of the
codes in a row), so a block's record is contiguous and can be moved whole.  The metadata
has the dtype of the keys, values and queries the cache is used with: one
dtype for the life of a cache.

An 8-bit cache of one layer is a uint8 tensor ``[num_blocks, heads, 2 * block_size + 1,
128]`` (:func:`kv8_cache`): in each (block, head) ``block_size`` rows of key codes, as
many of value codes and a row of scales, contiguous too.  Codes are e4m3 numbers
(``cache[:, :, :block_size].view(torch.float8_e4m3fn)``).  Each unit of 16 tokens has two
bytes in the last row, for its keys and its values; a channel's value is
``code * 2 ** (byte - 127)``.  It has no dtype: keys of either 16-bit type can be
appended and queries of either can attend.

All functions run on the current CUDA stream and never synchronise the host.
They have no backward pass and refuse tensors that require a gradient outside
``torch.no_grad()``.
Indices that only the device sees (slots, positions, block ids, lengths) are
checked there: one out of range records ERR_BOUNDS in the device error word
(:func:`kernels.check_device_error`), and its row, or the part of it that the
index names, is left out.  The first call on a device creates that word and
has to come before any stream capture on it.
"""

from __future__ import annotations

from typing import Optional

import torch

from kvserve_hpdps_b200.ops import kernels as K

HEAD_DIM = K.HEAD_DIM
GROUP_SIZES = (32, 64, 128)

_ops = None


def _native():
    """The binding module (raises with a build hint when missing)."""
    global _ops
    if _ops is None:
        try:
            from kvserve_hpdps_b200.ops import _paged_ops
        except ImportError as e:
            raise RuntimeError(f"native module _paged_ops cannot be loaded ({e}); build it with "
                               "`python -m kvserve_hpdps_b200.ops.build`") from e
        if _paged_ops.torch_version != torch.__version__:
            raise RuntimeError(f"native module _paged_ops is built for torch "
                               f"{_paged_ops.torch_version}, this is {torch.__version__}; build it "
                               "again with `python -m kvserve_hpdps_b200.ops.build`")
        _ops = _paged_ops
    return _ops


def _call(name: str, tensor: torch.Tensor, args: tuple):
    """Run a native operator; the first on ``tensor``'s device hands it the error word."""
    ops = _ops or _native()
    try:
        return getattr(ops, name)(*args)
    except ops.NoErrorWord:
        device = tensor.device
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first call on a device has to come before a stream "
                               "capture") from None
        with torch.cuda.device(device):
            ops.set_error_word(device.index, K.workspace(device).err.data_ptr())
        return getattr(ops, name)(*args)


# ------------------------------------------------------------------- caches
def kv4_row_bytes(group_size: int) -> int:
    """Bytes of one (token, head) of a 4-bit cache, key and value together."""
    if group_size not in GROUP_SIZES:
        raise ValueError(f"group_size must be one of {GROUP_SIZES}, got {group_size}")
    return HEAD_DIM + 8 * (HEAD_DIM // group_size)


def kv4_cache(num_blocks: int, num_heads: int, block_size: int = 16, group_size: int = 64,
              device="cuda") -> torch.Tensor:
    """A zeroed 4-bit cache of one layer (every row reads as zeros)."""
    if block_size <= 0 or block_size % 16:
        raise ValueError("block_size must be a multiple of 16")
    return torch.zeros((num_blocks, num_heads, block_size, kv4_row_bytes(group_size)),
                       dtype=torch.uint8, device=device)


def kv8_cache(num_blocks: int, num_heads: int, block_size: int = 16,
              device="cuda") -> torch.Tensor:
    """A zeroed 8-bit cache of one layer (every row reads as zeros)."""
    if block_size <= 0 or block_size % 16 or block_size > 1024:
        raise ValueError("block_size must be a multiple of 16 up to 1024")
    return torch.zeros((num_blocks, num_heads, 2 * block_size + 1, HEAD_DIM), dtype=torch.uint8,
                       device=device)


# ------------------------------------------------------------------- append
def append_kv(cache: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
              slot_mapping: torch.Tensor, positions: Optional[torch.Tensor] = None,
              cos_sin: Optional[torch.Tensor] = None, query: Optional[torch.Tensor] = None,
              *, interleaved: bool = False,
              query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Append a step's keys and values to a paged cache, rotating on the way.

    ``cache``: a 16-bit layer ``[2, nb, bs, H, 128]`` or ``[nb, 2, bs, H, 128]``
    (any block, slot and head strides, so token-major and head-major blocks)
    in the keys' dtype, an 8-bit cache (:func:`kv8_cache`) or a 4-bit one
    (:func:`kv4_cache`).
    ``key`` / ``value``: ``[T, H, 128]`` bf16 or fp16, any token and head
    strides.  ``slot_mapping`` ``[n <= T]``: slot of each token
    (``block * block_size + offset``); a negative slot's token is not appended,
    rows of ``key`` behind ``n`` are not read.  Slots of one call are distinct
    (of two tokens with one slot either may be kept, in parts; in an 8-bit cache the
    slot's unit of 16 may hold anything).

    In an 8-bit cache the 16 tokens of a unit share a scale, keys and values apart, per head: the
    smallest power of two that holds the largest of them in e4m3.  It grows as tokens
    come, and the codes of those before are moved to it (exact but for what falls into
    e4m3's subnormals).  A call that has the token at offset 0 of a unit begins the unit anew:
    the unit's slots that the call does not name lose what they held.  An infinity or NaN
    is held as NaN and has no say in the scale.

    With ``positions`` ``[>= n]`` and ``cos_sin`` ``[max_position, rotary_dim]``
    (cosines, then sines; fp32 or the keys' dtype) the first ``rotary_dim``
    channels of keys and queries are rotated: channel i with i + rotary_dim/2,
    or 2i with 2i + 1 when ``interleaved``.  Computed in fp32 and rounded once.
    ``query`` ``[T, Hq, 128]``: returned rotated, in ``query_out`` when given
    (it may be ``query``); rows behind ``n`` are not written there, and zeros
    without it.  A position
    outside the table records an error: its token is not appended and its
    query row is returned as it is.  Without ``positions`` nothing is rotated
    and ``query`` must be None.
    """
    args = (cache, key, value, slot_mapping, positions, cos_sin, query, interleaved, query_out)
    return _call("append_kv", key, args)


# --------------------------------------------------------------------- read
def read_kv4(cache: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of a 4-bit cache: ``[2, n, H, 128]`` keys and values at the slots.

    ``dtype``: the 16-bit type the cache was written with; the values are
    rounded to it once.  A negative slot reads zeros."""
    args = (cache, slot_mapping, dtype, out)
    return _call("read_kv4", cache, args)


def read_kv8(cache: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of an 8-bit cache: ``[2, n, H, 128]`` keys and values at the slots.

    ``dtype``: bf16 or fp16; the values are rounded to it once (bf16 holds all of
    them), those past its largest number to that.  A negative slot reads zeros."""
    args = (cache, slot_mapping, dtype, out)
    return _call("read_kv8", cache, args)


# ---------------------------------------------------------------- attention
def attention_kv4(query: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                  seq_lens: torch.Tensor, query_start: Optional[torch.Tensor] = None,
                  max_query_len: int = 1, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Causal attention of ``query`` ``[T, Hq, 128]`` over a 4-bit cache.

    ``block_table`` int32 ``[R, columns]``: block ids of each sequence;
    ``seq_lens`` int32 ``[R]``: tokens of it in the cache (up to 2^31 - 2^16), those
    of the query rows among them (append first).  ``query_start`` int32 ``[R + 1]``: sequence r's
    query rows are ``query_start[r]..query_start[r + 1]``, at most
    ``max_query_len`` of them; row i of n sees the first
    ``seq_lens[r] - n + i + 1`` tokens.  Without it sequence r has the one row
    r.  ``Hq`` is a multiple of the cache's heads (consecutive query heads
    share one).  ``scale`` defaults to 1/sqrt(128).

    ``max_query_len`` and the room in the table choose the kernel, for the call as a whole: give
    sequences of one or a few rows and prefill chunks calls of their own (48 decodes
    beside a chunk of 512: 327 us together, 149 apart), each with its own bound.

    Returns the output in the query's dtype (``out`` when given) and with
    ``return_lse`` also the fp32 logarithm of each row's sum of exponentials
    ``[T, Hq]``.  A row that sees no token is zeros with -inf.  A sequence
    whose extents do not fit the arrays records an error and is left out; so is
    a block id outside the cache, with its tokens.  Rows of no sequence and of
    one left out keep what a given ``out`` holds (which saves writing them, in a
    batch padded far), without one they are zeros; their logarithm is -inf.  Scratch is allocated per call from torch's
    allocator, so captured graphs do not share it.
    """
    args = (query, cache, block_table, seq_lens, query_start, max_query_len, scale, out,
            return_lse, True)
    out, lse = _call("attention_kv4", query, args)
    return (out, lse) if return_lse else out


def attention_kv8(query: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                  seq_lens: torch.Tensor, query_start: Optional[torch.Tensor] = None,
                  max_query_len: int = 1, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, return_lse: bool = False, *,
                  causal: bool = True):
    """Attention of ``query`` ``[T, Hq, 128]`` (bf16 or fp16) over an 8-bit cache.

    Arguments, results and errors are :func:`attention_kv4`'s.  With ``causal=False``
    every query row sees all ``seq_lens[r]`` tokens of its sequence: cross attention to an
    encoder's states, whose keys and values :func:`append_kv` has put into the cache (without
    positions) and whose number has nothing to do with that of the query rows.

    Both kernels take scores and sums in fp32.  That for many rows rounds weights to 11 bits in
    both types, that for few rows in bf16 alone: an fp16 row's error is up to a third larger where
    ``max_query_len`` and the room in the table choose the first.  Scales and scores may lie as far
    apart as fp32 holds them.  A query row with an element that is not finite, and a token to see,
    is NaN.
    """
    args = (query, cache, block_table, seq_lens, query_start, max_query_len, scale, out,
            return_lse, causal)
    out, lse = _call("attention_kv8", query, args)
    return (out, lse) if return_lse else out
