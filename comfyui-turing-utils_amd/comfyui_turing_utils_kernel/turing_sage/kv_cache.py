"""A paged key/value cache in 8 bits and the attention that reads it.

A video model that makes its frames chunk by chunk, or a served prompt, attends
to the keys and values of tokens that were computed before.  They are kept as
int8 codes in pages of 64 tokens, with one scale a page and head for the keys and
one for the values: half the memory, and half the reads of a decoding step.

* ``QuantizedKVCache``: the pool of pages;
* ``kv_cache_append``: quantizes new tokens behind the ends of their sequences;
* ``kv_cache_read``: cached tokens in 16 bits;
* ``kv_cache_attention``: attention of query tokens over their sequences;
* ``SequenceKVCache``: a pool with the block table and lengths of a batch, and
  the three calls on it, as the Wan block takes it.

No counterpart in the reference's facade (its attention sees whole sequences).
"""
from __future__ import annotations

import dataclasses
from typing import Optional

import torch

from .. import _lib
from .core import _compute_units, _sage_head_dim
from .quant import _layout_dims
from .sparse import _check_lengths, _require_gpu

PAGE_TOKENS = 64
_FLOATS = (torch.bfloat16, torch.float16)


@dataclasses.dataclass(frozen=True)
class QuantizedKVCache:
    """A pool of pages: ``key_codes`` int8 [pages, heads, 64, width],
    ``value_codes`` int8 [pages, heads, width, 64] (transposed, as the attention
    reads them), ``key_scale`` and ``value_scale`` fp32 [pages, heads]; width 64
    or 128.  What stands in a page's free places is never read."""

    key_codes: torch.Tensor
    value_codes: torch.Tensor
    key_scale: torch.Tensor
    value_scale: torch.Tensor

    @classmethod
    def allocate(cls, pages: int, heads: int, head_dim: int, device=None) -> "QuantizedKVCache":
        """Room for 64 * ``pages`` tokens; a head_dim up to 128 takes 64 or 128 channels."""
        if pages < 1 or heads < 1 or not 1 <= head_dim <= 128:
            raise ValueError(f"a cache needs pages, heads and a head_dim up to 128, got {pages}, {heads}, {head_dim}")
        width = _sage_head_dim(head_dim)
        return cls(torch.zeros((pages, heads, PAGE_TOKENS, width), dtype=torch.int8, device=device),
                   torch.zeros((pages, heads, width, PAGE_TOKENS), dtype=torch.int8, device=device),
                   torch.zeros((pages, heads), dtype=torch.float32, device=device),
                   torch.zeros((pages, heads), dtype=torch.float32, device=device))

    @property
    def tensors(self) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
        return self.key_codes, self.value_codes, self.key_scale, self.value_scale


def _check_cache(key_codes, value_codes, key_scale, value_scale, block_table, lengths):
    """(pages, heads, width, batch, pages of a sequence)"""
    if key_codes.dtype != torch.int8 or value_codes.dtype != torch.int8:
        raise TypeError("cache codes must be int8")
    if key_scale.dtype != torch.float32 or value_scale.dtype != torch.float32:
        raise TypeError("cache scales must be float32")
    if key_codes.dim() != 4 or key_codes.size(2) != PAGE_TOKENS or key_codes.size(3) not in (64, 128) \
            or min(key_codes.shape) < 1:
        raise ValueError(f"key codes must be [pages, heads, {PAGE_TOKENS}, 64 or 128], got {tuple(key_codes.shape)}")
    pages, heads, _, width = key_codes.shape
    if value_codes.shape != (pages, heads, width, PAGE_TOKENS):
        raise ValueError(f"value codes must be {(pages, heads, width, PAGE_TOKENS)}, got {tuple(value_codes.shape)}")
    if key_scale.shape != (pages, heads) or value_scale.shape != (pages, heads):
        raise ValueError(f"cache scales must be {(pages, heads)}")
    tensors = (key_codes, value_codes, key_scale, value_scale)
    if not all(t.is_contiguous() for t in tensors):
        raise ValueError("the cache's tensors must be contiguous")
    if block_table.dtype != torch.int32 or lengths.dtype != torch.int32:
        raise TypeError("block_table and lengths must be int32")
    if block_table.dim() != 2 or block_table.size(1) < 1 or lengths.shape != (block_table.size(0),):
        raise ValueError(f"block_table must be [batch, pages of a sequence] and lengths [batch], got "
                         f"{tuple(block_table.shape)} and {tuple(lengths.shape)}")
    if {t.device for t in (*tensors, block_table, lengths)} != {key_codes.device}:
        raise ValueError("the cache, block_table and lengths must be on one device")
    return pages, heads, width, block_table.size(0), block_table.size(1)


def _check_aligned(key_codes, value_codes) -> None:
    if key_codes.data_ptr() % 16 or value_codes.data_ptr() % 16:
        raise ValueError("the cache's codes must start on 16 bytes")


def _check_tokens(x, name, tensor_layout, batch, heads, width) -> int:
    """The token count of x, [batch, heads, tokens, head_dim] or NHD."""
    if tensor_layout not in ("HND", "NHD"):
        raise ValueError(f"Unsupported tensor_layout: {tensor_layout}")
    if x.dim() != 4 or not 1 <= x.size(3) <= width:
        raise ValueError(f"{name} must be four-dimensional with a head_dim up to the cache's {width}, got {tuple(x.shape)}")
    h, tokens = (x.size(1), x.size(2)) if tensor_layout == "HND" else (x.size(2), x.size(1))
    if x.size(0) != batch or (heads is not None and h != heads):
        raise ValueError(f"{name} must have the batch {batch} of the block table and the cache's {heads} heads, got "
                         f"{tuple(x.shape)} as {tensor_layout}")
    return tokens


def _rows(x: torch.Tensor, width: int) -> torch.Tensor:
    """x with the cache's channels, contiguous ones, in rows that start on 16 bytes."""
    if x.size(-1) != width:
        x = torch.nn.functional.pad(x, (0, width - x.size(-1)))
    piece = 16 // x.element_size()
    if x.stride(-1) != 1 or x.data_ptr() % 16 or any(s % piece for s in x.stride()[:-1]):
        # (contiguous() and clone() would keep any stride of an axis of one)
        x = torch.empty(x.shape, dtype=x.dtype, device=x.device).copy_(x)
    return x


def _check_mean(key_mean, batch, heads, width, device) -> None:
    if key_mean is None:
        return
    if key_mean.dtype != torch.bfloat16:
        raise TypeError("key_mean must be bfloat16")
    if key_mean.dim() != 3 or key_mean.shape[:2] != (batch, heads) or not 1 <= key_mean.size(2) <= width:
        raise ValueError(f"key_mean must be [{batch}, {heads}, head_dim], got {tuple(key_mean.shape)}")
    if key_mean.device != device:
        raise ValueError("key_mean must be on the cache's device")


def _mean_rows(key_mean, width):
    return None if key_mean is None else _rows(key_mean.contiguous(), width)


# ---------------------------------------------------------------------------
# Writing
# ---------------------------------------------------------------------------

def _check_append(key, value, key_codes, value_codes, key_scale, value_scale, block_table, lengths, tensor_layout,
                  new_lengths, key_in_scale, key_mean):
    cache = _check_cache(key_codes, value_codes, key_scale, value_scale, block_table, lengths)
    _, heads, width, batch, _ = cache
    tokens = _check_tokens(key, "key", tensor_layout, batch, heads, width)
    if value.shape != key.shape:
        raise ValueError("key and value must have one shape")
    if value.dtype not in _FLOATS:
        raise TypeError("value must be bfloat16 or float16")
    if key_in_scale is None:
        if key.dtype != value.dtype:
            raise TypeError("key must have value's type, or be int8 codes with a key_scale")
    else:
        if key.dtype != torch.int8 or key_in_scale.dtype != torch.float32:
            raise TypeError("a key_scale is float32 and belongs to int8 keys")
        blocks = (tokens + PAGE_TOKENS - 1) // PAGE_TOKENS
        if key_in_scale.shape != (batch, heads, blocks):
            raise ValueError(f"key_scale must be {(batch, heads, blocks)}, one for {PAGE_TOKENS} tokens, got "
                             f"{tuple(key_in_scale.shape)}")
    _check_mean(key_mean, batch, heads, width, key_codes.device)
    if {key.device, value.device} != {key_codes.device} \
            or (key_in_scale is not None and key_in_scale.device != key_codes.device):
        raise ValueError("key, value and the cache must be on one device")
    _check_lengths(new_lengths, batch, key_codes.device, "new_lengths")
    return (*cache, tokens)


@torch.library.custom_op("turing_utils::kv_cache_append",
                         mutates_args=("key_codes", "value_codes", "key_scale", "value_scale"))
def _append_op(
    key: torch.Tensor,
    value: torch.Tensor,
    key_codes: torch.Tensor,
    value_codes: torch.Tensor,
    key_scale: torch.Tensor,
    value_scale: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    tensor_layout: str,
    new_lengths: torch.Tensor | None = None,
    key_in_scale: torch.Tensor | None = None,
    key_mean: torch.Tensor | None = None,
) -> torch.Tensor:
    _require_gpu(key_codes, "the key/value cache")
    pages, heads, width, batch, row, tokens = _check_append(
        key, value, key_codes, value_codes, key_scale, value_scale, block_table, lengths, tensor_layout, new_lengths,
        key_in_scale, key_mean)
    _check_aligned(key_codes, value_codes)
    device = key_codes.device
    with torch.cuda.device(device):
        after = torch.empty(batch, dtype=torch.int32, device=device)
        if batch == 0:
            return after
        if tokens == 0:
            return torch.clamp(lengths, 0, row * PAGE_TOKENS, out=after)
        key, value, key_mean = _rows(key, width), _rows(value, width), _mean_rows(key_mean, width)
        block_table, lengths = block_table.contiguous(), lengths.contiguous()
        new_lengths = None if new_lengths is None else new_lengths.contiguous()
        key_in_scale = None if key_in_scale is None else key_in_scale.contiguous()
        _, _, *k_strides = _layout_dims(key, tensor_layout)
        _, _, *v_strides = _layout_dims(value, tensor_layout)
        _lib.call("tu_kv_cache_append", key.data_ptr(), _lib.ptr(key_in_scale), value.data_ptr(),
                  int(value.dtype == torch.float16), batch, heads, tokens, width, *k_strides, *v_strides,
                  _lib.ptr(key_mean), block_table.data_ptr(), row, lengths.data_ptr(), _lib.ptr(new_lengths),
                  key_codes.data_ptr(), value_codes.data_ptr(), key_scale.data_ptr(), value_scale.data_ptr(), pages,
                  after.data_ptr(), _lib.stream_of(device))
    return after


@_append_op.register_fake
def _append_fake(key, value, key_codes, value_codes, key_scale, value_scale, block_table, lengths, tensor_layout,
                 new_lengths=None, key_in_scale=None, key_mean=None):
    _check_append(key, value, key_codes, value_codes, key_scale, value_scale, block_table, lengths, tensor_layout,
                  new_lengths, key_in_scale, key_mean)
    return torch.empty_like(lengths, memory_format=torch.contiguous_format)


def kv_cache_append(
    key: torch.Tensor,
    value: torch.Tensor,
    cache: QuantizedKVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    tensor_layout: str = "HND",
    new_lengths: Optional[torch.Tensor] = None,
    key_scale: Optional[torch.Tensor] = None,
    key_mean: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """Quantizes ``key`` and ``value`` (bf16 or fp16, [B, Hkv, L, D] or NHD) into
    the pages behind each sequence's end, and returns the lengths afterwards
    (int32 [B]; ``lengths`` stays as it is).

    Sequence b holds ``lengths[b]`` tokens, token t in page ``block_table[b, t //
    64]`` (int32 [B, n]); it gets the first ``new_lengths[b]`` of the L tokens (all
    when None), as many as its n pages have room for.  Lengths are taken within
    [0, 64 n].  A table entry that is no page of the pool drops its tokens.

    Per page and head, K and V apart, in 32 bits: the scale is the largest of that
    of the page's earlier tokens, max |new x| / 127 and 1e-7 / 127, a code is
    round(x * (1 / scale)); where the scale grows, the earlier codes are made again
    from the values they stand for.  A page keeps its scale until it is begun anew
    (written from its first place on).  A NaN or infinite x makes the scale of its
    page and head NaN or infinite and the codes zero: every row that attends to the
    page is NaN, and no other.

    ``key`` may be int8 codes with ``key_scale`` fp32 [B, Hkv, ceil(L / 64)], as
    ``prequantize_rms_rope_qk`` gives them.  ``key_mean`` (bf16 [B, Hkv, D]) is
    subtracted from the keys before they are quantized: a constant of a head moves
    all scores of a query alike, which the softmax cancels, and keys around zero
    are quantized more finely; give it to every call of the sequence.

    Pages that are written must be named once among those of the call; what a page
    named twice holds is unspecified.  The op is
    ``torch.ops.turing_utils.kv_cache_append``; it has no backward."""
    args = (new_lengths, key_scale, key_mean)
    if tensor_layout in ("HND", "NHD") and key.is_cuda and not torch.compiler.is_compiling():
        after = _lib.host_calls().kv_cache_append(key, value, *cache.tensors, block_table, lengths,
                                                  tensor_layout == "NHD", *args, _lib.raw_stream(key.get_device()))
        if after is not None:
            return after
    return _append_op(key, value, *cache.tensors, block_table, lengths, tensor_layout, *args)


# ---------------------------------------------------------------------------
# Reading back
# ---------------------------------------------------------------------------

def _check_read(key_codes, value_codes, key_scale, value_scale, block_table, lengths, max_length, tensor_layout, dtype,
                starts, key_mean):
    cache = _check_cache(key_codes, value_codes, key_scale, value_scale, block_table, lengths)
    _, heads, width, batch, _ = cache
    if tensor_layout not in ("HND", "NHD"):
        raise ValueError(f"Unsupported tensor_layout: {tensor_layout}")
    if dtype not in _FLOATS:
        raise TypeError("a cache is read as bfloat16 or float16")
    if not 0 <= max_length <= 0x7fffff00:
        raise ValueError(f"max_length must not be negative, got {max_length}")
    _check_lengths(starts, batch, key_codes.device, "starts")
    _check_mean(key_mean, batch, heads, width, key_codes.device)
    return cache, ((batch, heads, max_length, width) if tensor_layout == "HND" else (batch, max_length, heads, width))


@torch.library.custom_op("turing_utils::kv_cache_read", mutates_args=())
def _read_op(
    key_codes: torch.Tensor,
    value_codes: torch.Tensor,
    key_scale: torch.Tensor,
    value_scale: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    max_length: int,
    tensor_layout: str,
    dtype: torch.dtype,
    starts: torch.Tensor | None = None,
    key_mean: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    _require_gpu(key_codes, "the key/value cache")
    (pages, heads, width, batch, row), shape = _check_read(
        key_codes, value_codes, key_scale, value_scale, block_table, lengths, max_length, tensor_layout, dtype, starts,
        key_mean)
    _check_aligned(key_codes, value_codes)
    device = key_codes.device
    with torch.cuda.device(device):
        key, value = (torch.empty(shape, dtype=dtype, device=device) for _ in range(2))
        if batch == 0 or max_length == 0:
            return key, value
        key_mean = _mean_rows(key_mean, width)
        block_table, lengths = block_table.contiguous(), lengths.contiguous()
        starts = None if starts is None else starts.contiguous()
        _, _, *strides = _layout_dims(key, tensor_layout)
        _lib.call("tu_kv_cache_read", key_codes.data_ptr(), value_codes.data_ptr(), key_scale.data_ptr(),
                  value_scale.data_ptr(), pages, block_table.data_ptr(), row, lengths.data_ptr(), _lib.ptr(starts),
                  _lib.ptr(key_mean), key.data_ptr(), value.data_ptr(), int(dtype == torch.float16), batch, heads,
                  max_length, width, *strides, *strides, _lib.stream_of(device))
    return key, value


@_read_op.register_fake
def _read_fake(key_codes, value_codes, key_scale, value_scale, block_table, lengths, max_length, tensor_layout, dtype,
               starts=None, key_mean=None):
    _, shape = _check_read(key_codes, value_codes, key_scale, value_scale, block_table, lengths, max_length,
                           tensor_layout, dtype, starts, key_mean)
    return tuple(torch.empty(shape, dtype=dtype, device=key_codes.device) for _ in range(2))


def kv_cache_read(
    cache: QuantizedKVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    max_length: int,
    starts: Optional[torch.Tensor] = None,
    tensor_layout: str = "HND",
    dtype: torch.dtype = torch.bfloat16,
    key_mean: Optional[torch.Tensor] = None,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Cached keys and values in 16 bits: of each sequence the ``max_length``
    tokens from ``starts[b]`` on (int32 [B], 0 when None), as [B, Hkv, max_length,
    width] or NHD; zeros at and past ``lengths[b]`` and where the table names no
    page.  A value is code * scale, a key also plus ``key_mean`` (what was given to
    ``kv_cache_append``), in 32 bits, rounded once."""
    args = (int(max_length), tensor_layout, dtype, starts, key_mean)
    if tensor_layout in ("HND", "NHD") and dtype in _FLOATS and cache.key_codes.is_cuda \
            and not torch.compiler.is_compiling():
        out = _lib.host_calls().kv_cache_read(*cache.tensors, block_table, lengths, args[0], tensor_layout == "NHD",
                                              dtype == torch.float16, starts, key_mean,
                                              _lib.raw_stream(cache.key_codes.get_device()))
        if out is not None:
            return out
    return _read_op(*cache.tensors, block_table, lengths, *args)


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def _check_attend(query, key_codes, value_codes, key_scale, value_scale, block_table, lengths, tensor_layout,
                  query_scale, blkq, query_lengths, max_length):
    cache = _check_cache(key_codes, value_codes, key_scale, value_scale, block_table, lengths)
    _, heads, width, batch, _ = cache
    tokens = _check_tokens(query, "query", tensor_layout, batch, None, width)
    hq = query.size(1) if tensor_layout == "HND" else query.size(2)
    if hq < 1 or hq % heads:
        raise ValueError(f"the query's {hq} heads must be a multiple of the cache's {heads}")
    if query_scale is None:
        if query.dtype not in _FLOATS:
            raise TypeError("query must be bfloat16 or float16, or int8 codes with a query_scale")
    else:
        if query.dtype != torch.int8 or query_scale.dtype != torch.float32:
            raise TypeError("a query_scale is float32 and belongs to int8 queries")
        if blkq < 1 or query_scale.shape != (batch, hq, (tokens + blkq - 1) // blkq):
            raise ValueError(f"query_scale must be [{batch}, {hq}, ceil({tokens} / blkq)] with blkq > 0, got "
                             f"{tuple(query_scale.shape)} and {blkq}")
    if query.device != key_codes.device or (query_scale is not None and query_scale.device != key_codes.device):
        raise ValueError("query and the cache must be on one device")
    if max_length < 1:
        raise ValueError(f"max_length must be positive, got {max_length}")
    _check_lengths(query_lengths, batch, key_codes.device, "query_lengths")
    return (*cache, hq, tokens)


@torch.library.custom_op("turing_utils::kv_cache_attention", mutates_args=())
def _attend_op(
    query: torch.Tensor,
    key_codes: torch.Tensor,
    value_codes: torch.Tensor,
    key_scale: torch.Tensor,
    value_scale: torch.Tensor,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    tensor_layout: str,
    is_causal: bool,
    sm_scale: float,
    max_length: int,
    query_scale: torch.Tensor | None = None,
    blkq: int = 128,
    query_lengths: torch.Tensor | None = None,
) -> torch.Tensor:
    _require_gpu(key_codes, "the key/value cache")
    pages, heads, width, batch, row, hq, tokens = _check_attend(
        query, key_codes, value_codes, key_scale, value_scale, block_table, lengths, tensor_layout, query_scale, blkq,
        query_lengths, max_length)
    _check_aligned(key_codes, value_codes)
    device, head_dim = key_codes.device, query.size(-1)
    scale = float(sm_scale) if sm_scale > 0.0 else head_dim ** -0.5
    dtype = torch.bfloat16 if query_scale is not None else query.dtype
    with torch.cuda.device(device):
        shape = (batch, hq, tokens, width) if tensor_layout == "HND" else (batch, tokens, hq, width)
        out = torch.empty(shape, dtype=dtype, device=device)
        if out.numel() == 0:
            return out[..., :head_dim].contiguous()
        query, block_table, lengths = _rows(query, width), block_table.contiguous(), lengths.contiguous()
        query_lengths = None if query_lengths is None else query_lengths.contiguous()
        query_scale = None if query_scale is None else query_scale.contiguous()
        _, _, *q_strides = _layout_dims(query, tensor_layout)
        _, _, *o_strides = _layout_dims(out, tensor_layout)
        cus = _compute_units(device)
        max_length = min(max_length, row * PAGE_TOKENS)
        kind = 2 if query_scale is not None else int(query.dtype == torch.float16)
        nbytes = int(_lib.load().tu_kv_cache_attn_workspace(batch, hq, heads, tokens, width, max_length, kind,
                                                            int(bool(is_causal)), cus))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _lib.call("tu_kv_cache_attn", query.data_ptr(), _lib.ptr(query_scale), kind, int(blkq), key_codes.data_ptr(),
                  value_codes.data_ptr(), key_scale.data_ptr(), value_scale.data_ptr(), pages, block_table.data_ptr(),
                  row, lengths.data_ptr(), _lib.ptr(query_lengths), out.data_ptr(), batch, hq, heads, tokens, width,
                  *q_strides, *o_strides, scale, int(bool(is_causal)), max_length, cus, _lib.ptr(workspace), nbytes,
                  _lib.stream_of(device))
    return out if head_dim == width else out[..., :head_dim].contiguous()


@_attend_op.register_fake
def _attend_fake(query, key_codes, value_codes, key_scale, value_scale, block_table, lengths, tensor_layout, is_causal,
                 sm_scale, max_length, query_scale=None, blkq=128, query_lengths=None):
    _check_attend(query, key_codes, value_codes, key_scale, value_scale, block_table, lengths, tensor_layout,
                  query_scale, blkq, query_lengths, max_length)
    return torch.empty(query.shape, dtype=torch.bfloat16 if query_scale is not None else query.dtype,
                       device=query.device)


def kv_cache_attention(
    query: torch.Tensor,
    cache: QuantizedKVCache,
    block_table: torch.Tensor,
    lengths: torch.Tensor,
    *,
    tensor_layout: str = "HND",
    is_causal: bool = False,
    sm_scale: Optional[float] = None,
    query_scale: Optional[torch.Tensor] = None,
    blkq: int = 128,
    query_lengths: Optional[torch.Tensor] = None,
    max_length: Optional[int] = None,
) -> torch.Tensor:
    """Attention of ``query`` ([B, Hq, Lq, D] or NHD, Hq a multiple of the cache's
    heads) over the cached tokens of its sequences, the ``lengths[b]`` tokens in
    the pages of ``block_table[b]`` (as ``kv_cache_append`` returns them).

    Sequence b has ``query_lengths[b]`` = n query tokens (int32 [B], Lq when None).
    They see every cached token, or with ``is_causal``, as the sequence's last n
    tokens, those up to their own: query i the keys j <= lengths[b] - n + i.  Rows
    that see no key, and rows at or past n, are zeros.

    ``query`` is bf16 or fp16, or int8 codes with ``query_scale`` fp32 [B, Hq,
    ceil(Lq / blkq)], the framework's own form, which needs half of the products
    with the keys.  A float row is taken as integers of 16 bits with one scale: each
    element is off by at most max |row| / 65024 (of a row below 1e-33, 1e-33 /
    65024).  Elements below 1/128 of the row's largest lose bits of a bf16, those
    below 1/16 of an fp16.  The result has the query's type and shape, bf16 for
    codes.  ``sm_scale`` is head_dim^-0.5 unless given.  Scores are held in 32 bits: a
    row whose largest is infinite there is NaN.

    ``max_length``: a bound of the lengths, where it is known to be less than the
    64 n of the block table; the split of long sequences over the GPU is made for
    it.  The op is ``torch.ops.turing_utils.kv_cache_attention``; it has no
    backward."""
    if sm_scale is not None and not 0.0 < float(sm_scale) < float("inf"):
        raise ValueError("sm_scale must be a positive finite number")
    if max_length is None:
        max_length = max(1, block_table.size(-1) * PAGE_TOKENS) if block_table.dim() else 1
    args = (bool(is_causal), -1.0 if sm_scale is None else float(sm_scale), int(max_length), query_scale, int(blkq),
            query_lengths)
    if tensor_layout in ("HND", "NHD") and query.is_cuda and not torch.compiler.is_compiling():
        out = _lib.host_calls().kv_cache_attention(query, *cache.tensors, block_table, lengths, tensor_layout == "NHD",
                                                   *args, _compute_units(query.device),
                                                   _lib.raw_stream(query.get_device()))
        if out is not None:
            return out
    return _attend_op(query, *cache.tensors, block_table, lengths, tensor_layout, *args)


# ---------------------------------------------------------------------------
# A batch's sequences
# ---------------------------------------------------------------------------

@dataclasses.dataclass
class SequenceKVCache:
    """A pool with the block table and the lengths of a batch of sequences.

    ``append`` moves ``lengths`` on, in place, so that a captured step that appends
    and attends can be replayed.  To write tokens again (a chunk at its next
    denoising step), set ``lengths`` back in place first."""

    cache: QuantizedKVCache
    block_table: torch.Tensor
    lengths: torch.Tensor

    @classmethod
    def allocate(cls, batch: int, max_length: int, heads: int, head_dim: int, device=None) -> "SequenceKVCache":
        """Empty sequences of up to ``max_length`` tokens each, with pages of their own."""
        if batch < 1 or max_length < 1:
            raise ValueError(f"a cache needs a batch and a length, got {batch} and {max_length}")
        row = (max_length + PAGE_TOKENS - 1) // PAGE_TOKENS
        return cls(QuantizedKVCache.allocate(batch * row, heads, head_dim, device),
                   torch.arange(batch * row, dtype=torch.int32, device=device).view(batch, row),
                   torch.zeros(batch, dtype=torch.int32, device=device))

    @property
    def max_length(self) -> int:
        """Tokens that a sequence has places for."""
        return self.block_table.size(1) * PAGE_TOKENS

    def append(self, key: torch.Tensor, value: torch.Tensor, **kwargs) -> None:
        """``kv_cache_append`` behind the sequences' ends; ``lengths`` grow."""
        self.lengths.copy_(kv_cache_append(key, value, self.cache, self.block_table, self.lengths, **kwargs))

    def read(self, *, max_length: int, **kwargs) -> tuple[torch.Tensor, torch.Tensor]:
        """``kv_cache_read`` of the sequences."""
        return kv_cache_read(self.cache, self.block_table, self.lengths, max_length=max_length, **kwargs)

    def attend(self, query: torch.Tensor, **kwargs) -> torch.Tensor:
        """``kv_cache_attention`` over the sequences."""
        return kv_cache_attention(query, self.cache, self.block_table, self.lengths, **kwargs)
