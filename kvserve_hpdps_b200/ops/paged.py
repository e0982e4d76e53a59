"""Operators on the paged KV caches of a serving step.

* :func:`append_kv`: a step's new keys and values into a paged cache (16-bit,
  or held in 4 bits), the position rotation of keys and queries applied in the
  same launch;
* :func:`attention_kv4`: attention over a 4-bit cache without unpacking it
  first (one token, several draft tokens or a prefill chunk per sequence);
* :func:`read_kv4`: rows of a 4-bit cache as 16-bit values, e.g. to hand them
  to the paths that take 16-bit KV.

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

All functions run on the current CUDA stream and never synchronise the host.
Indices that only the device sees (slots, positions, block ids, lengths) are
checked there: one out of range records ERR_BOUNDS in the device error word
(:func:`kernels.check_device_error`), and its row, or the part of it that the
index names, is left out.  The first call on a device creates that word and
has to come before any stream capture on it.
"""

from __future__ import annotations

import ctypes
import math
from typing import Optional

import torch

from kvserve_hpdps_b200.ops import kernels as K
from kvserve_hpdps_b200.ops import _lib
from kvserve_hpdps_b200.ops._lib import check, lib

HEAD_DIM = K.HEAD_DIM
GROUP_SIZES = (32, 64, 128)
_INT = (torch.int32, torch.int64)
_HALF = (torch.bfloat16, torch.float16)


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


def _groups4(cache: torch.Tensor) -> int:
    """Channel groups of a 4-bit cache's rows; raises on what is not one."""
    if cache.dtype != torch.uint8 or cache.dim() != 4:
        raise TypeError("a 4-bit cache is a uint8 [blocks, heads, block_size, row_bytes] tensor")
    nb, h, bs, rb = cache.shape
    if rb not in (136, 144, 160):
        raise ValueError(f"a 4-bit cache's row has 136, 144 or 160 bytes, got {rb}")
    if bs <= 0 or bs % 16:
        raise ValueError("block_size must be a multiple of 16")
    st = cache.stride()
    if st[3] != 1 or st[2] != rb or st[0] % 16 or st[1] % 16 or cache.data_ptr() % 16:
        raise ValueError("a 4-bit cache's records must be contiguous and 16-byte aligned, "
                         f"got strides {st}")
    return (rb - 128) // 8


def _cuda(what: str, device: torch.device, *tensors: Optional[torch.Tensor]) -> None:
    if device.type != "cuda":
        raise ValueError(f"{what} needs CUDA tensors")
    for t in tensors:
        if t is not None and t.device != device:
            raise ValueError(f"{what}: tensors on {t.device} and {device}")


def _rows(t: torch.Tensor) -> torch.Tensor:
    """``t`` [rows, heads, 128] as the kernels read it: 16-byte aligned rows,
    copied only when it is not."""
    st = t.stride()
    if st[2] == 1 and not st[0] % 8 and not st[1] % 8 and not t.data_ptr() % 16:
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _index(name: str, t: torch.Tensor, n: Optional[int] = None) -> torch.Tensor:
    if t.dtype not in _INT or t.dim() != 1:
        raise TypeError(f"{name} must be a one-dimensional int32 or int64 tensor")
    if n is not None and t.shape[0] < n:
        raise ValueError(f"{name} has {t.shape[0]} entries for {n} tokens")
    return t if t.is_contiguous() else t.contiguous()


def _heads3(name: str, t: torch.Tensor, dtype=None) -> None:
    if t.dtype not in _HALF or (dtype is not None and t.dtype != dtype):
        raise TypeError(f"{name} must be bf16 or fp16, one dtype for all, got {t.dtype}")
    if t.dim() != 3 or t.shape[2] != HEAD_DIM:
        raise ValueError(f"{name} must be [tokens, heads, {HEAD_DIM}], got {tuple(t.shape)}")


def _out3(name: str, t: torch.Tensor, like: torch.Tensor) -> None:
    if t.dtype != like.dtype or t.shape != like.shape:
        raise ValueError(f"{name} must match the query's shape and dtype")
    st = t.stride()
    if st[2] != 1 or st[0] % 8 or st[1] % 8 or t.data_ptr() % 16:
        raise ValueError(f"{name} must have 16-byte aligned rows")


class _On:
    """Makes a tensor's device current for a launch (nothing when it is)."""

    def __init__(self, device: torch.device):
        idx = device.index
        self._guard = None if idx == torch.cuda.current_device() else torch.cuda.device(idx)

    def __enter__(self):
        if self._guard is not None:
            self._guard.__enter__()

    def __exit__(self, *exc):
        if self._guard is not None:
            self._guard.__exit__(*exc)


def _err_ptr(device: torch.device) -> int:
    err = K._err_words.get(device.index)
    if err is None:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("the first call on a device has to come before a stream capture")
        err = K.workspace(device).err
    return err.data_ptr()


# ------------------------------------------------------------------- append
def append_kv(cache: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
              slot_mapping: torch.Tensor, positions: Optional[torch.Tensor] = None,
              cos_sin: Optional[torch.Tensor] = None, query: Optional[torch.Tensor] = None,
              *, interleaved: bool = False,
              query_out: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """Append a step's keys and values to a paged cache, rotating on the way.

    ``cache``: a 16-bit layer ``[2, nb, bs, H, 128]`` or ``[nb, 2, bs, H, 128]``
    (any block, slot and head strides, so token-major and head-major blocks)
    in the keys' dtype, or a 4-bit cache (:func:`kv4_cache`).
    ``key`` / ``value``: ``[T, H, 128]`` bf16 or fp16, any token and head
    strides.  ``slot_mapping`` ``[n <= T]``: slot of each token
    (``block * block_size + offset``); a negative slot's token is not appended,
    rows of ``key`` behind ``n`` are not read.  Slots of one call are distinct
    (of two tokens with one slot either may be kept, in parts).

    With ``positions`` ``[>= n]`` and ``cos_sin`` ``[max_position, rotary_dim]``
    (cosines, then sines; fp32 or the keys' dtype) the first ``rotary_dim``
    channels of keys and queries are rotated: channel i with i + rotary_dim/2,
    or 2i with 2i + 1 when ``interleaved``.  Computed in fp32 and rounded once.
    ``query`` ``[T, Hq, 128]``: returned rotated, in ``query_out`` when given
    (it may be ``query``); rows behind ``n`` are not written.  A position
    outside the table records an error: its token is not appended and its
    query row is returned as it is.  Without ``positions`` nothing is rotated
    and ``query`` must be None.
    """
    _heads3("key", key)
    dt = key.dtype
    _heads3("value", value, dt)
    if value.shape != key.shape:
        raise ValueError(f"key {tuple(key.shape)} and value {tuple(value.shape)} differ")
    dev = key.device
    slots = _index("slot_mapping", slot_mapping)
    T, H = key.shape[0], key.shape[1]
    n = slots.shape[0]
    if n > T:
        raise ValueError(f"{n} slots for {T} tokens")
    L = _lib.AppendLaunch()
    if cache.dtype == torch.uint8:
        L.groups = _groups4(cache)
        nb, hc, bs = cache.shape[0], cache.shape[1], cache.shape[2]
        L.block_stride, L.head_stride = cache.stride(0), cache.stride(1)
    else:
        if cache.dtype != dt:
            raise TypeError(f"cache is {cache.dtype}, keys are {dt}")
        if cache.dim() != 5 or cache.shape[4] != HEAD_DIM or 2 not in cache.shape[:2]:
            raise ValueError(f"expected a [2, nb, bs, H, {HEAD_DIM}] layer, "
                             f"got {tuple(cache.shape)}")
        st = cache.stride()
        if st[4] != 1 or any(x % 8 for x in st[:4]) or cache.data_ptr() % 16:
            raise ValueError(f"the cache's rows must be 16-byte aligned, got strides {st}")
        if cache.shape[1] == 2 and cache.shape[0] != 2:
            L.block_stride, L.kv_stride = st[0], st[1]
        else:
            L.kv_stride, L.block_stride = st[0], st[1]
        nb, bs, hc = K._num_blocks(cache), cache.shape[2], cache.shape[3]
        L.slot_stride, L.head_stride = st[2], st[3]
    if hc != H:
        raise ValueError(f"the cache has {hc} heads, the keys {H}")
    L.num_slots, L.block_size = nb * bs, bs
    key, value = _rows(key), _rows(value)
    L.key, L.value, L.slots, L.cache = (key.data_ptr(), value.data_ptr(), slots.data_ptr(),
                                        cache.data_ptr())
    L.key_ts, L.key_hs = key.stride(0), key.stride(1)
    L.val_ts, L.val_hs = value.stride(0), value.stride(1)
    L.tokens, L.heads = n, H
    L.fp16, L.slots64 = dt == torch.float16, slots.dtype == torch.int64
    if (positions is None) != (cos_sin is None):
        raise ValueError("positions and cos_sin go together")
    if positions is None and query is not None:
        raise ValueError("query is only taken to be rotated (positions and cos_sin)")
    if positions is not None:
        pos = _index("positions", positions, n)
        if cos_sin.dim() != 2 or cos_sin.dtype not in (torch.float32, dt):
            raise TypeError("cos_sin must be [max_position, rotary_dim], fp32 or the keys' dtype")
        rd = cos_sin.shape[1]
        if rd <= 0 or rd > HEAD_DIM or rd % 16:
            raise ValueError(f"rotary_dim must be a multiple of 16 up to {HEAD_DIM}, got {rd}")
        if cos_sin.stride(1) != 1 or cos_sin.stride(0) * cos_sin.element_size() % 16 \
                or cos_sin.data_ptr() % 16:
            raise ValueError("cos_sin's rows must be 16-byte aligned")
        L.pos, L.table, L.pos64 = pos.data_ptr(), cos_sin.data_ptr(), pos.dtype == torch.int64
        L.max_pos, L.table_stride, L.rotary = cos_sin.shape[0], cos_sin.stride(0), rd
        L.table32, L.interleaved = cos_sin.dtype == torch.float32, bool(interleaved)
    if query is None:
        if query_out is not None:
            raise ValueError("query_out without query")
    else:
        _heads3("query", query, dt)
        if query.shape[0] != T:
            raise ValueError(f"query has {query.shape[0]} rows, key {T}")
        if query_out is None:
            query_out = torch.empty(query.shape, dtype=dt, device=dev)
        else:
            _out3("query_out", query_out, query)
        src = _rows(query)
        L.query, L.query_out, L.q_heads = src.data_ptr(), query_out.data_ptr(), src.shape[1]
        L.q_ts, L.q_hs = src.stride(0), src.stride(1)
        L.qo_ts, L.qo_hs = query_out.stride(0), query_out.stride(1)
    _cuda("append_kv", dev, cache, value, slot_mapping, positions, cos_sin, query, query_out)
    if n == 0 or H == 0:
        return query_out
    with _On(dev):
        L.err = _err_ptr(dev)
        check(lib().kvs_append_kv(ctypes.byref(L), K._stream(dev)), "append_kv")
    return query_out


# --------------------------------------------------------------------- read
def read_kv4(cache: torch.Tensor, slot_mapping: torch.Tensor, dtype: torch.dtype,
             out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Rows of a 4-bit cache: ``[2, n, H, 128]`` keys and values at the slots.

    ``dtype``: the 16-bit type the cache was written with; the values are
    rounded to it once.  A negative slot reads zeros."""
    groups = _groups4(cache)
    if dtype not in _HALF:
        raise TypeError(f"dtype must be bf16 or fp16, got {dtype}")
    slots = _index("slot_mapping", slot_mapping)
    dev = cache.device
    nb, H, bs, _ = cache.shape
    n = slots.shape[0]
    if out is None:
        out = torch.empty((2, n, H, HEAD_DIM), dtype=dtype, device=dev)
    elif (out.shape != (2, n, H, HEAD_DIM) or out.dtype != dtype or not out.is_contiguous()
          or out.data_ptr() % 16):
        raise ValueError(f"out must be a contiguous {dtype} [2, {n}, {H}, {HEAD_DIM}] tensor")
    _cuda("read_kv4", dev, slots, out)
    if n == 0 or H == 0:
        return out
    L = _lib.Read4Launch()
    L.cache, L.slots, L.out = cache.data_ptr(), slots.data_ptr(), out.data_ptr()
    L.block_stride, L.head_stride, L.num_slots = cache.stride(0), cache.stride(1), nb * bs
    L.tokens, L.heads, L.block_size, L.groups = n, H, bs, groups
    L.fp16, L.slots64 = dtype == torch.float16, slots.dtype == torch.int64
    with _On(dev):
        L.err = _err_ptr(dev)
        check(lib().kvs_read_kv4(ctypes.byref(L), K._stream(dev)), "read_kv4")
    return out


# ---------------------------------------------------------------- attention
def attention_kv4(query: torch.Tensor, cache: torch.Tensor, block_table: torch.Tensor,
                  seq_lens: torch.Tensor, query_start: Optional[torch.Tensor] = None,
                  max_query_len: int = 1, scale: Optional[float] = None,
                  out: Optional[torch.Tensor] = None, return_lse: bool = False):
    """Causal attention of ``query`` ``[T, Hq, 128]`` over a 4-bit cache.

    ``block_table`` int32 ``[R, columns]``: block ids of each sequence;
    ``seq_lens`` int32 ``[R]``: tokens of it in the cache, those of the query
    rows among them (append first).  ``query_start`` int32 ``[R + 1]``: sequence r's
    query rows are ``query_start[r]..query_start[r + 1]``, at most
    ``max_query_len`` of them; row i of n sees the first
    ``seq_lens[r] - n + i + 1`` tokens.  Without it sequence r has the one row
    r.  ``Hq`` is a multiple of the cache's heads (consecutive query heads
    share one).  ``scale`` defaults to 1/sqrt(128).

    Returns the output in the query's dtype (``out`` when given) and with
    ``return_lse`` also the fp32 logarithm of each row's sum of exponentials
    ``[T, Hq]``.  A row that sees no token is zeros with -inf.  Rows of no
    sequence are left as they are.  A sequence whose extents do not fit the
    arrays records an error and is left out; so is a block id outside the
    cache, with its tokens.  Scratch is allocated per call from torch's
    allocator, so captured graphs do not share it.
    """
    _heads3("query", query)
    groups = _groups4(cache)
    dev = query.device
    if block_table.dtype != torch.int32 or block_table.dim() != 2:
        raise TypeError("block_table must be an int32 [sequences, columns] tensor")
    R = block_table.shape[0]
    if seq_lens.dtype != torch.int32 or seq_lens.shape != (R,):
        raise TypeError(f"seq_lens must be an int32 [{R}] tensor")
    T, Hq = query.shape[0], query.shape[1]
    nb, H, bs, _ = cache.shape
    if H == 0 or Hq % H:
        raise ValueError(f"{Hq} query heads are no multiple of the cache's {H}")
    if query_start is None:
        if T < R:
            raise ValueError(f"{T} query rows for {R} sequences")
        if max_query_len != 1:
            raise ValueError("max_query_len needs query_start")
    else:
        if query_start.dtype != torch.int32 or query_start.shape != (R + 1,):
            raise TypeError(f"query_start must be an int32 [{R + 1}] tensor")
        if max_query_len < 1:
            raise ValueError("max_query_len must be positive")
        query_start = query_start.contiguous()
    if out is None:
        out = torch.empty(query.shape, dtype=query.dtype, device=dev)
    else:
        _out3("out", out, query)
    lse = torch.empty((T, Hq), dtype=torch.float32, device=dev) if return_lse else None
    _cuda("attention_kv4", dev, cache, block_table, seq_lens, query_start, out)
    if R and T and Hq:
        q = _rows(query)
        if block_table.stride(1) != 1:
            block_table = block_table.contiguous()
        seq_lens = seq_lens.contiguous()
        L = _lib.Attn4Launch()
        L.q, L.out, L.cache = q.data_ptr(), out.data_ptr(), cache.data_ptr()
        L.table, L.lens = block_table.data_ptr(), seq_lens.data_ptr()
        if lse is not None:
            L.lse = lse.data_ptr()
        if query_start is not None:
            L.start = query_start.data_ptr()
        L.q_ts, L.q_hs = q.stride(0), q.stride(1)
        L.o_ts, L.o_hs = out.stride(0), out.stride(1)
        L.block_stride, L.head_stride = cache.stride(0), cache.stride(1)
        L.table_stride, L.table_cols = block_table.stride(0), block_table.shape[1]
        L.seqs, L.tokens, L.num_blocks, L.q_heads, L.heads = R, T, nb, Hq, H
        L.block_size, L.groups, L.fp16 = bs, groups, query.dtype == torch.float16
        L.max_q = min(max_query_len, T)
        L.scale = 1.0 / math.sqrt(HEAD_DIM) if scale is None else float(scale)
        with _On(dev):
            L.err = _err_ptr(dev)
            n = lib().kvs_attn4_scratch_bytes(ctypes.byref(L))
            scratch = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
            L.scratch = K._ptr(scratch)
            check(lib().kvs_attention_kv4(ctypes.byref(L), K._stream(dev)), "attention_kv4")
    return (out, lse) if return_lse else out
