"""Block-sparse Sage attention: each block of 128 queries attends to the key
blocks of 64 that a cheap score selects.

Three calls, each on the quantized state of ``prequantize_sageattn`` (or of
the fused producer, ``prequantize_sageattn_from_qk``) or its tensors:

* ``select_key_blocks``: the product of the blocks' mean rows, and for each
  query block the ``keep`` key blocks where it is largest;
* ``key_block_attention``: Sage attention over the listed key blocks;
* ``sparse_sageattn``: quantize, select, attend in one call from bf16 / fp16.

The reference's sparse router (Sol / SLA, comfyui_turing_utils/attention/
sparse.py) picks blocks by a threshold on its own score; this is another
selection with a fixed count per query block, built for this package.
"""
from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from .core import (
    PrequantizedSageAttention,
    _check_qk,
    _compute_units,
    prequantize_sageattn,
)
from .quant import _layout_dims

QUERY_BLOCK = 128
KEY_BLOCK = 64


def _blocks(length: int, block: int) -> int:
    return (length + block - 1) // block


def _check_lengths(lengths: Optional[torch.Tensor], batch: int, device, what: str) -> Optional[torch.Tensor]:
    if lengths is None:
        return None
    if lengths.dtype != torch.int32 or lengths.shape != (batch,):
        raise ValueError(f"{what} must be int32 [{batch}], got {lengths.dtype} {tuple(lengths.shape)}")
    if lengths.device != device:
        raise ValueError(f"{what} must be on the Q/K device")
    return lengths.contiguous()


def _require_gpu(t: torch.Tensor, what: str) -> None:
    if t.device.type != "cuda":
        raise RuntimeError(f"{what} requires CUDA (HIP) tensors")
    if not _lib.device_supported(t.device):
        raise RuntimeError(f"{what} requires a gfx950 (MI355X-class) GPU")


def _row_aligned(x: torch.Tensor) -> torch.Tensor:
    """Codes whose rows start on 16 bytes."""
    return x.contiguous() if x.data_ptr() % 16 or any(s % 16 for s in x.stride()[:-1]) else x


def _check_select(keep, sink_blocks, local_blocks) -> None:
    if keep < 1 or sink_blocks < 0 or local_blocks < 0:
        raise ValueError("keep must be at least 1, sink_blocks and local_blocks not negative")


def _select(query_int8, query_scale, key_int8, key_scale, tensor_layout, keep, is_causal, sink_blocks, local_blocks,
            blkq, blkk, query_lengths, key_lengths):
    _require_gpu(query_int8, "Sage block selection")
    batch, hq, hkv, lq, lk = _check_qk(query_int8, query_scale, key_int8, key_scale, tensor_layout, blkq, blkk)
    if lq == 0 or lk == 0 or batch == 0:
        raise ValueError("Sage block selection requires non-empty Q/K sequences")
    _check_select(keep, sink_blocks, local_blocks)
    device, dim = query_int8.device, query_int8.size(-1)
    query_lengths = _check_lengths(query_lengths, batch, device, "query_lengths")
    key_lengths = _check_lengths(key_lengths, batch, device, "key_lengths")
    query_int8, key_int8 = _row_aligned(query_int8), _row_aligned(key_int8)
    _, _, *q_strides = _layout_dims(query_int8, tensor_layout)
    _, _, *k_strides = _layout_dims(key_int8, tensor_layout)
    query_scale, key_scale = query_scale.contiguous(), key_scale.contiguous()
    nkb = _blocks(lk, KEY_BLOCK)
    limit = 0x3fffffff
    with torch.cuda.device(device):
        index = torch.empty((batch, hq, _blocks(lq, QUERY_BLOCK), min(keep, nkb)), dtype=torch.int32, device=device)
        nbytes = int(_lib.load().tu_sage_block_select_workspace(batch, hq, hkv, lq, lk, dim))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _lib.call("tu_sage_block_select", query_int8.data_ptr(), query_scale.data_ptr(), blkq, key_int8.data_ptr(),
                  key_scale.data_ptr(), blkk, batch, hq, hkv, lq, lk, dim, *q_strides, *k_strides,
                  _lib.ptr(query_lengths), _lib.ptr(key_lengths), min(keep, nkb), min(sink_blocks, limit),
                  min(local_blocks, limit), int(bool(is_causal)), workspace.data_ptr(), nbytes, index.data_ptr(),
                  _lib.stream_of(device))
    return index


@torch.library.custom_op("turing_utils::sage_block_select", mutates_args=())
def sage_block_select(
    query_int8: torch.Tensor,
    query_scale: torch.Tensor,
    key_int8: torch.Tensor,
    key_scale: torch.Tensor,
    tensor_layout: str,
    keep: int,
    is_causal: bool,
    sink_blocks: int,
    local_blocks: int,
    blkq: int,
    blkk: int,
    query_lengths: torch.Tensor | None = None,
    key_lengths: torch.Tensor | None = None,
) -> torch.Tensor:
    return _select(query_int8, query_scale, key_int8, key_scale, tensor_layout, keep, is_causal, sink_blocks,
                   local_blocks, blkq, blkk, query_lengths, key_lengths)


@sage_block_select.register_fake
def _sage_block_select_fake(query_int8, query_scale, key_int8, key_scale, tensor_layout, keep, is_causal, sink_blocks,
                            local_blocks, blkq, blkk, query_lengths=None, key_lengths=None):
    batch, hq, _, lq, lk = _check_qk(query_int8, query_scale, key_int8, key_scale, tensor_layout, blkq, blkk)
    _check_select(keep, sink_blocks, local_blocks)
    return torch.empty((batch, hq, _blocks(lq, QUERY_BLOCK), min(keep, _blocks(lk, KEY_BLOCK))), dtype=torch.int32,
                       device=query_int8.device)


def select_key_blocks(
    query_int8: torch.Tensor,
    query_scale: torch.Tensor,
    key_int8: torch.Tensor,
    key_scale: torch.Tensor,
    *,
    keep: int,
    tensor_layout: str = "HND",
    is_causal: bool = False,
    sink_blocks: int = 0,
    local_blocks: int = 0,
    blkq: int = 128,
    blkk: int = 128,
    query_lengths: Optional[torch.Tensor] = None,
    key_lengths: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """The key blocks each query block attends to: int32 [B, Hq,
    ceil(Lq / 128), min(keep, ceil(Lk / 64))], ascending, -1 behind the last.

    Query block i (rows 128 i ..) sees key block j (keys 64 j ..) if the block
    has rows below ``query_lengths[b]``, the key block starts below
    ``key_lengths[b]`` and, when causal, at or below the query block's last
    row.  Of those it takes the first ``keep``: the forced blocks (the first
    ``sink_blocks``, and with ``local_blocks`` = w the two on the diagonal, 2 i
    and 2 i + 1, and w - 1 more on each side) in the order of j, whatever their
    products; then the others by the larger product of the blocks' mean rows
    (64-bit, over the rows in front of the sample's end), NaN last, the lower j
    first among equals."""
    args = (tensor_layout, int(keep), bool(is_causal), int(sink_blocks), int(local_blocks), int(blkq), int(blkk),
            query_lengths, key_lengths)
    if tensor_layout in ("HND", "NHD") and query_int8.is_cuda and not torch.compiler.is_compiling():
        index = _lib.host_calls().select_key_blocks(query_int8, query_scale, key_int8, key_scale,
                                                    tensor_layout == "NHD", *args[1:],
                                                    _lib.raw_stream(query_int8.get_device()))
        if index is not None:
            return index
    return sage_block_select(query_int8, query_scale, key_int8, key_scale, *args)


def _check_attend(query_int8, query_scale, key_int8, key_scale, value_t, block_index, tensor_layout, blkq, blkk):
    batch, hq, hkv, lq, lk = _check_qk(query_int8, query_scale, key_int8, key_scale, tensor_layout, blkq, blkk)
    if lq == 0 or lk == 0 or batch == 0:
        raise ValueError("block attention requires non-empty Q/K sequences")
    if blkk // KEY_BLOCK & (blkk // KEY_BLOCK - 1):
        raise ValueError("block attention needs blkk = 64 * 2^n")
    width = query_int8.size(-1)
    lpad = _blocks(lk, KEY_BLOCK) * KEY_BLOCK
    if value_t.dtype != torch.bfloat16 or value_t.shape != (batch, hkv, width, lpad):
        raise ValueError(f"V^T must be bf16 [{batch}, {hkv}, {width}, {lpad}]")
    if block_index.dtype != torch.int32 or block_index.dim() != 4 \
            or block_index.shape[:3] != (batch, hq, _blocks(lq, QUERY_BLOCK)):
        raise ValueError(f"block_index must be int32 [{batch}, {hq}, {_blocks(lq, QUERY_BLOCK)}, n], got "
                         f"{block_index.dtype} {tuple(block_index.shape)}")
    if len({value_t.device, block_index.device, query_int8.device}) != 1:
        raise ValueError("V^T and block_index must be on the Q/K device")
    return batch, hq, hkv, lq, lk, lpad


def _attend(query_int8, query_scale, key_int8, key_scale, value_t, block_index, tensor_layout, is_causal, sm_scale,
            blkq, blkk, query_lengths, key_lengths):
    _require_gpu(query_int8, "Sage block attention")
    batch, hq, hkv, lq, lk, lpad = _check_attend(query_int8, query_scale, key_int8, key_scale, value_t, block_index,
                                                 tensor_layout, blkq, blkk)
    device, dim, width = query_int8.device, query_int8.size(-1), block_index.size(-1)
    scale = float(sm_scale) if sm_scale > 0.0 else dim ** -0.5
    query_lengths = _check_lengths(query_lengths, batch, device, "query_lengths")
    key_lengths = _check_lengths(key_lengths, batch, device, "key_lengths")
    query_int8, key_int8 = _row_aligned(query_int8), _row_aligned(key_int8)
    value_t = value_t.contiguous()
    if value_t.data_ptr() % 16:
        value_t = value_t.clone()
    block_index, query_scale, key_scale = block_index.contiguous(), query_scale.contiguous(), key_scale.contiguous()
    with torch.cuda.device(device):
        shape = (batch, lq, hq, dim) if tensor_layout == "NHD" else (batch, hq, lq, dim)
        if width == 0:  # nothing is listed
            return torch.zeros(shape, dtype=torch.bfloat16, device=device)
        output = torch.empty(shape, dtype=torch.bfloat16, device=device)
        _, _, *q_strides = _layout_dims(query_int8, tensor_layout)
        _, _, *k_strides = _layout_dims(key_int8, tensor_layout)
        _, _, *o_strides = _layout_dims(output, tensor_layout)
        cus = _compute_units(device)
        nbytes = int(_lib.load().tu_sage_block_attn_workspace(batch, hq, lq, dim, width, cus))
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None
        _lib.call("tu_sage_block_attn", query_int8.data_ptr(), query_scale.data_ptr(), blkq, key_int8.data_ptr(),
                  key_scale.data_ptr(), blkk, value_t.data_ptr(), lpad, block_index.data_ptr(), width,
                  output.data_ptr(), batch, hq, hkv, lq, lk, dim, *q_strides, *k_strides, *o_strides,
                  _lib.ptr(query_lengths), _lib.ptr(key_lengths), scale, int(bool(is_causal)), cus,
                  _lib.ptr(workspace), nbytes, _lib.stream_of(device))
    return output


@torch.library.custom_op("turing_utils::sage_block_attention", mutates_args=())
def sage_block_attention(
    query_int8: torch.Tensor,
    query_scale: torch.Tensor,
    key_int8: torch.Tensor,
    key_scale: torch.Tensor,
    value_t: torch.Tensor,
    block_index: torch.Tensor,
    tensor_layout: str,
    is_causal: bool,
    sm_scale: float,
    blkq: int,
    blkk: int,
    query_lengths: torch.Tensor | None = None,
    key_lengths: torch.Tensor | None = None,
) -> torch.Tensor:
    return _attend(query_int8, query_scale, key_int8, key_scale, value_t, block_index, tensor_layout, is_causal,
                   sm_scale, blkq, blkk, query_lengths, key_lengths)


@sage_block_attention.register_fake
def _sage_block_attention_fake(query_int8, query_scale, key_int8, key_scale, value_t, block_index, tensor_layout,
                               is_causal, sm_scale, blkq, blkk, query_lengths=None, key_lengths=None):
    _check_attend(query_int8, query_scale, key_int8, key_scale, value_t, block_index, tensor_layout, blkq, blkk)
    return torch.empty(query_int8.shape, dtype=torch.bfloat16, device=query_int8.device)


def key_block_attention(
    query_int8: torch.Tensor,
    query_scale: torch.Tensor,
    key_int8: torch.Tensor,
    key_scale: torch.Tensor,
    value_t: torch.Tensor,
    block_index: torch.Tensor,
    *,
    tensor_layout: str = "HND",
    is_causal: bool = False,
    sm_scale: Optional[float] = None,
    blkq: int = 128,
    blkk: int = 128,
    query_lengths: Optional[torch.Tensor] = None,
    key_lengths: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``attention_from_vt`` over listed key blocks: the queries of block i
    (rows 128 i .. 128 i + 127) attend to the keys of the blocks
    ``block_index[b, h, i]`` names (int32 [B, Hq, ceil(Lq / 128), n]).

    An entry counts if it lies in [0, ceil(Lk / 64)) and is larger than every
    entry before it, so lists are ascending and -1 (or anything else) names
    nothing.  Keys at or past ``key_lengths[b]`` are not seen, whatever codes
    and values stand there; rows at or past ``query_lengths[b]``, and rows that
    see no key, are zeros.  Causal masks are aligned at the first row and key.
    Scales are not negative (a quantizer's are not); one that is NaN, or infinite
    with codes of zero as a quantizer leaves them, makes NaN of the rows that see
    its keys, or that have it, and of no others.
    Values of the listed blocks in front of the sample's end must be finite, as
    in the dense attention: 0 times infinity is a NaN in every row of the tile.
    Output: bf16 in the layout and shape of ``query_int8``."""
    if sm_scale is not None and not 0.0 < float(sm_scale) < float("inf"):
        raise ValueError("sm_scale must be a positive finite number")
    tensors = (query_int8, query_scale, key_int8, key_scale, value_t, block_index)
    args = (tensor_layout, bool(is_causal), -1.0 if sm_scale is None else float(sm_scale), int(blkq), int(blkk),
            query_lengths, key_lengths)
    if tensor_layout in ("HND", "NHD") and query_int8.is_cuda and not torch.compiler.is_compiling():
        out = _lib.host_calls().key_block_attention(*tensors, tensor_layout == "NHD", *args[1:],
                                                    _compute_units(query_int8.device),
                                                    _lib.raw_stream(query_int8.get_device()))
        if out is not None:
            return out
    return sage_block_attention(*tensors, *args)


def sparse_sageattn_from_prequantized(
    quantized: PrequantizedSageAttention,
    *,
    keep: int,
    sink_blocks: int = 0,
    local_blocks: int = 0,
    query_lengths: Optional[torch.Tensor] = None,
    key_lengths: Optional[torch.Tensor] = None,
) -> torch.Tensor:
    """``sageattn_from_prequantized`` over the ``keep`` key blocks that
    ``select_key_blocks`` picks for each query block."""
    qk = (quantized.query_int8, quantized.query_scale, quantized.key_int8, quantized.key_scale)
    common = dict(tensor_layout=quantized.tensor_layout, is_causal=quantized.is_causal, blkq=quantized.blkq,
                  blkk=quantized.blkk, query_lengths=query_lengths, key_lengths=key_lengths)
    index = select_key_blocks(*qk, keep=keep, sink_blocks=sink_blocks, local_blocks=local_blocks, **common)
    out = key_block_attention(*qk, quantized.value_t, index, sm_scale=quantized.sm_scale, **common)
    out = out[..., : quantized.original_head_dim]
    return out if quantized.output_dtype == torch.bfloat16 else out.to(quantized.output_dtype)


def sparse_sageattn(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    tensor_layout: str = "HND",
    is_causal: bool = False,
    sm_scale: Optional[float] = None,
    smooth_k: bool = True,
    *,
    keep: int,
    sink_blocks: int = 0,
    local_blocks: int = 0,
    query_lengths: Optional[torch.Tensor] = None,
    key_lengths: Optional[torch.Tensor] = None,
    BLKQ: int = 128,
    BLKK: int = 128,
) -> torch.Tensor:
    """``sageattn`` over ``keep`` key blocks of 64 per query block of 128.
    Rows behind a sample's length must hold finite values (the quantizer's
    block scales and K's mean see them); they are not attended to."""
    quantized = prequantize_sageattn(q, k, v, tensor_layout=tensor_layout, is_causal=is_causal, sm_scale=sm_scale,
                                     smooth_k=smooth_k, BLKQ=BLKQ, BLKK=BLKK)
    return sparse_sageattn_from_prequantized(quantized, keep=keep, sink_blocks=sink_blocks, local_blocks=local_blocks,
                                             query_lengths=query_lengths, key_lengths=key_lengths)
