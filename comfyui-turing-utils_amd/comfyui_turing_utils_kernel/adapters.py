"""Low-rank adapters (LoRA) of many requests at once beside a W8A8 projection.

An adapter adds ``scaling * (x A^T) B^T`` to a projection ``x W^T``.  Merged
into W it would need W quantized again, and one W could serve one adapter; here
it stays apart, and every row of a batch names its own (or none).

The projection's input exists only as ConvRot INT8 codes of the rotated
activation ``x R`` (R the block-Hadamard group transform, symmetric and
orthonormal), so A is rotated once when it is loaded: ``(x R)(A R)^T = x A^T``.
The adapter then sees the same quantized activation as the projection, and a
fused norm + quantizer feeds both.  The product with A is a kernel of its own
(one byte per activation read); the product with B runs in the epilogue of the
INT8 GEMM and joins its fp32 value before the one rounding to bf16.

No counterpart in the reference's kernel package: ComfyUI merges LoRAs into
weights, and the plugin's quantized layers take none.
"""
from __future__ import annotations

from typing import Optional, Sequence

import torch

from . import _lib, ops
from .ops import _check_residual, _linear_args
from .turing_sage.core import _compute_units

RANK_MULTIPLE = 8  # the kernels read 16-byte pieces of a rank
MAX_RANK = 4096

def _check_adapters(m, n, k, down, up, scaling, adapter_ids, adapter_rows, parts=1) -> None:
    if down.dtype != torch.bfloat16 or up.dtype != torch.bfloat16:
        raise TypeError("adapter weights must be bfloat16")
    if parts < 1 or (parts > 1 and n % (16 * parts)):
        raise ValueError(f"{n} columns do not make {parts} equal parts of a multiple of 16")
    if down.dim() != 3 or up.dim() != 3 or down.shape[2] != k \
            or up.shape != (down.shape[0], n, down.shape[1] // parts) or down.shape[1] % parts:
        raise ValueError(f"adapters must be down [count, rank, {k}] and up [count, {n}, "
                         f"{'rank' if parts == 1 else f'rank / {parts}'}], got {tuple(down.shape)} and {tuple(up.shape)}")
    rank = down.shape[1]
    if down.shape[0] < 1 or rank // parts % RANK_MULTIPLE or not 0 < rank <= MAX_RANK:
        raise ValueError(f"adapters need a count of at least 1 and a rank that is a multiple of {RANK_MULTIPLE} up to "
                         f"{MAX_RANK} (zero ranks pad), got {tuple(down.shape)}")
    if scaling.dtype != torch.float32 or scaling.shape != (down.shape[0],):
        raise ValueError("adapter scaling must be one float32 per adapter")
    if adapter_ids.dtype != torch.int32 or adapter_ids.dim() != 1:
        raise TypeError("adapter_ids must be a 1D int32 tensor")
    if adapter_rows < 1 or adapter_ids.numel() != (m + adapter_rows - 1) // adapter_rows:
        raise ValueError(f"adapter_ids must hold one adapter per {adapter_rows} of {m} rows, got {adapter_ids.numel()}")


def _aligned(t: Optional[torch.Tensor]) -> Optional[torch.Tensor]:
    """Contiguous and on 16 bytes, as the kernels read."""
    if t is None:
        return None
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _linear_adapters(activation, weight, activation_scale, weight_scale, bias, down, up, scaling, adapter_ids,
                     adapter_rows, residual, gate, gate_rows, parts):
    activation, weight, activation_scale, weight_scale, bias, m, n, k = _linear_args(
        activation, weight, activation_scale, weight_scale, bias)
    _check_adapters(m, n, k, down, up, scaling, adapter_ids, adapter_rows, parts)
    if residual is not None:
        _check_residual(residual, gate, gate_rows, m, n)
    elif gate is not None:
        raise ValueError("a gate needs a residual")
    others = [down, up, scaling, adapter_ids] + [t for t in (residual, gate) if t is not None]
    if {t.device for t in others} != {activation.device}:
        raise ValueError("INT8 linear tensors must use the same CUDA device")
    if gate is not None:
        gate = gate.to(torch.bfloat16).reshape(-1, n)
    down, up, residual, gate = (_aligned(t) for t in (down, up, residual, gate))
    # (names of their own: a copy has to live until the launch)
    scaling, adapter_ids = scaling.contiguous(), adapter_ids.contiguous()
    device = activation.device
    out = torch.empty((m, n), dtype=torch.bfloat16, device=device)
    if m == 0:
        return out
    cus, (count, rank, _) = _compute_units(device), down.shape
    nbytes = int(_lib.load().tu_int8_gemm_adapters_workspace(m, rank))
    with torch.cuda.device(device):
        workspace = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _lib.call(
            "tu_int8_gemm_adapters", activation.data_ptr(), weight.data_ptr(), activation_scale.data_ptr(),
            weight_scale.data_ptr(), _lib.ptr(bias), down.data_ptr(), up.data_ptr(), scaling.data_ptr(),
            adapter_ids.data_ptr(), int(adapter_rows), rank, count, int(parts), _lib.ptr(residual), _lib.ptr(gate),
            int(gate_rows) if gate is not None else 1, out.data_ptr(), m, n, k, cus, workspace.data_ptr(), nbytes,
            _lib.stream_of(device))
    return out


@torch.library.custom_op("turing_utils::int8_linear_adapters", mutates_args=())
def _int8_linear_adapters_op(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: torch.Tensor | None,
    down: torch.Tensor,
    up: torch.Tensor,
    scaling: torch.Tensor,
    adapter_ids: torch.Tensor,
    adapter_rows: int = 1,
    residual: torch.Tensor | None = None,
    gate: torch.Tensor | None = None,
    gate_rows: int = 1,
    parts: int = 1,
) -> torch.Tensor:
    return _linear_adapters(activation, weight, activation_scale, weight_scale, bias, down, up, scaling, adapter_ids,
                            adapter_rows, residual, gate, gate_rows, parts)


@_int8_linear_adapters_op.register_fake
def _int8_linear_adapters_fake(activation, weight, activation_scale, weight_scale, bias, down, up, scaling,
                               adapter_ids, adapter_rows=1, residual=None, gate=None, gate_rows=1,
                               parts=1):
    (m, k), n = activation.shape, weight.size(0)
    _check_adapters(m, n, k, down, up, scaling, adapter_ids, adapter_rows, parts)
    if residual is not None:
        _check_residual(residual, gate, gate_rows, m, n)
    return torch.empty((m, n), dtype=torch.bfloat16, device=activation.device)


def turing_int8_linear_adapters(
    activation: torch.Tensor,
    weight: torch.Tensor,
    activation_scale: torch.Tensor,
    weight_scale: torch.Tensor,
    bias: Optional[torch.Tensor],
    down: torch.Tensor,
    up: torch.Tensor,
    scaling: torch.Tensor,
    adapter_ids: torch.Tensor,
    adapter_rows: int = 1,
    residual: Optional[torch.Tensor] = None,
    gate: Optional[torch.Tensor] = None,
    gate_rows: int = 1,
    parts: int = 1,
) -> torch.Tensor:
    """``int8_linear`` (or, with ``residual``, ``int8_linear_residual``) whose
    fp32 value gains each row's adapter before it is rounded:

        y[m] = int8_linear value + scaling[a] * as[m] * (codes[m] . down[a]^T) . up[a]^T

    with ``a = adapter_ids[m // adapter_rows]``; a row whose id lies outside
    [0, count) has no adapter and gets int8_linear's bits.  ``down`` bf16
    [count, rank, K] holds rotated rows (``LinearAdapters`` makes them), ``up``
    bf16 [count, N, rank], ``scaling`` fp32 [count], ``adapter_ids`` int32
    [ceil(M / adapter_rows)]; the rank is a multiple of 8.  With ``parts`` the
    columns and the ranks are so many equal parts (of a multiple of 16 columns
    and 8 ranks each), the columns of a part see its own ranks alone, and ``up``
    is [count, N, rank / parts]: the projections of a fused q / k / v have
    adapters of their own.  Infinite or NaN weights make infinity or NaN of their
    own adapter's rows alone.  The op is
    ``torch.ops.turing_utils.int8_linear_adapters``; it has no backward."""
    args = (activation, weight, activation_scale, weight_scale, bias, down, up, scaling, adapter_ids, adapter_rows,
            residual, gate, gate_rows, parts)
    if not torch.compiler.is_compiling() and activation.is_cuda:
        out = _lib.host_calls().int8_linear_adapters(*args, _compute_units(activation.device),
                                                     _lib.raw_stream(activation.get_device()))
        if out is not None:
            return out
    return _int8_linear_adapters_op(*args)


_R4 = ((1, 1, 1, -1), (1, 1, -1, 1), (1, -1, 1, 1), (-1, 1, 1, 1))


def _rotation(group: int, device) -> torch.Tensor:
    """The ConvRot group transform as an fp64 matrix [group, group]: R4 on the
    radix-4 digits of strides 1, 4 and 16, on stride 64 another R4 (group 256)
    or the orthonormal H2 (group 128)."""
    r4 = torch.tensor(_R4, dtype=torch.float64) / 2
    top = r4 if group == 256 else torch.tensor(((1, 1), (1, -1)), dtype=torch.float64) * 0.5 ** 0.5
    m = top
    for _ in range(3):
        m = torch.kron(m, r4)
    return m.to(device)


class LinearAdapters:
    """The adapters of one W8A8 linear, laid out for the kernels: ``down`` bf16
    [count, rank, K] (rotated), ``up`` bf16 [count, N, rank / parts], ``scaling``
    fp32 [count]; ``parts`` as in ``turing_int8_linear_adapters``.  Adapters of
    different ranks share the largest, padded with zeros."""

    def __init__(self, down: torch.Tensor, up: torch.Tensor, scaling: torch.Tensor, group: int = 128, parts: int = 1):
        if group not in ops.SUPPORTED_GROUP_SIZES:
            raise ValueError(f"ConvRot group must be one of {ops.SUPPORTED_GROUP_SIZES}, got {group}")
        if down.dim() != 3 or up.dim() != 3:
            raise ValueError("adapters must be down [count, rank, K] and up [count, N, rank / parts]")
        # an empty list of rows: the shapes alone
        _check_adapters(0, up.shape[1], down.shape[2], down, up, scaling,
                        torch.empty(0, dtype=torch.int32, device=down.device), 1, parts)
        self.down, self.up, self.scaling, self.group = _aligned(down), _aligned(up), scaling.contiguous(), group
        self.parts = parts

    @property
    def count(self) -> int:
        return self.down.shape[0]

    @property
    def rank(self) -> int:
        return self.down.shape[1]

    @classmethod
    def from_float(cls, adapters: Sequence[tuple[torch.Tensor, torch.Tensor, float]], group: int = 128,
                   device=None) -> "LinearAdapters":
        """From (A [r, K], B [N, r], scaling) of each adapter, ``scaling`` being
        alpha / r where a file has an alpha.  A is rotated in fp64 and rounded
        to bf16 once."""
        if not adapters:
            raise ValueError("at least one adapter is needed")
        k, n = adapters[0][0].shape[-1], adapters[0][1].shape[0]
        if group not in ops.SUPPORTED_GROUP_SIZES or k % group:
            raise ValueError(f"ConvRot group {group} must be 128 or 256 and divide K={k}")
        for a, b, _ in adapters:
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != k or b.shape != (n, a.shape[0]) or a.shape[0] < 1:
                raise ValueError(f"each adapter needs A [rank, {k}] and B [{n}, rank], got {tuple(a.shape)} and "
                                 f"{tuple(b.shape)}")
        rank = (max(a.shape[0] for a, _, _ in adapters) + RANK_MULTIPLE - 1) // RANK_MULTIPLE * RANK_MULTIPLE
        device = adapters[0][0].device if device is None else torch.device(device)
        down = torch.zeros((len(adapters), rank, k), dtype=torch.bfloat16, device=device)
        up = torch.zeros((len(adapters), n, rank), dtype=torch.bfloat16, device=device)
        for i, (a, b, _) in enumerate(adapters):
            r = a.shape[0]
            rotated = a.to(device, torch.float64).reshape(r, k // group, group) @ _rotation(group, device)
            down[i, :r] = rotated.reshape(r, k).to(torch.bfloat16)
            up[i, :, :r] = b.to(device, torch.bfloat16)
        scaling = torch.tensor([float(s) for _, _, s in adapters], dtype=torch.float32, device=device)
        return cls(down, up, scaling, group)

    @staticmethod
    def concat(parts: "Sequence[LinearAdapters]") -> "LinearAdapters":
        """The adapters of ``W8A8Linear.concat``'s linear from those of its
        parts (adapter i of each part together): each part's output columns
        see its own ranks only.  Equal parts of a multiple of 16 columns stay
        parts, of the largest's rank; of others, ``up`` is padded with zeros.
        Every part needs the same scalings, as one file gives a model's layers."""
        if not parts or len({(p.count, p.down.shape[2], p.group) for p in parts}) != 1:
            raise ValueError("concatenated adapters need one count, K and ConvRot group")
        if any(not torch.equal(p.scaling, parts[0].scaling) for p in parts[1:]):
            raise ValueError("concatenated adapters need the same scalings")
        if any(p.parts != 1 for p in parts):
            raise ValueError("concatenated adapters cannot be concatenated again")
        count, n = parts[0].count, sum(p.up.shape[1] for p in parts)
        scaling, group = parts[0].scaling, parts[0].group
        if len({p.up.shape[1] for p in parts}) == 1 and n % (16 * len(parts)) == 0:
            most = max(p.rank for p in parts)
            pad = torch.nn.functional.pad
            return LinearAdapters(torch.cat([pad(p.down, (0, 0, 0, most - p.rank)) for p in parts], 1),
                                  torch.cat([pad(p.up, (0, most - p.rank)) for p in parts], 1), scaling, group, len(parts))
        up = torch.zeros((count, n, sum(p.rank for p in parts)), dtype=torch.bfloat16, device=parts[0].up.device)
        row = col = 0
        for p in parts:
            up[:, row:row + p.up.shape[1], col:col + p.rank] = p.up
            row, col = row + p.up.shape[1], col + p.rank
        return LinearAdapters(torch.cat([p.down for p in parts], 1), up, scaling, group)
