"""GPU: the adapters in the epilogue of each of the GEMM's seven tiles, within
the bound of tests/operator_reference.py: ranks of one chunk of 32, two and
three, rows of one adapter, of two with a border inside a wave, of any, and
columns of several parts with their borders inside a wave."""
from __future__ import annotations

import pytest
import torch

import comfyui_turing_utils_kernel as kernel
from comfyui_turing_utils_kernel import _lib
from tests import test_gpu_adapters as adapters

K = 272
# (rows, columns) at which the launch takes the tile on 256 compute units
SIZES = {(64, 64): (61, 528), (128, 64): (2051, 528), (128, 128): (2051, 1056), (128, 192): (2051, 2064),
         (128, 256): (5503, 1008), (256, 192): (4103, 2064), (256, 256): (1407, 8208)}


def test_the_sizes_take_all_seven_tiles():
    found = {tile: _lib.load().tu_int8_gemm_tile(m, n, K, 256) for tile, (m, n) in SIZES.items()}
    assert {tile: (t >> 16, t & 0xffff) for tile, t in found.items()} == {tile: tile for tile in SIZES}
    assert len(SIZES) == 7


def _inputs(dev, tile, rank, rows, **kw):
    if torch.cuda.get_device_properties(dev).multi_processor_count != 256:
        pytest.skip("the sizes take these tiles on 256 compute units")
    m, n = SIZES[tile]
    print(f"[adapter tiles] {tile}", flush=True)
    # one request, three with borders inside a wave's rows, rows of any
    ids = {"one": [1], "three": [2, 0, 1], "any": None}[rows]
    per = {"one": m, "three": (m + 2) // 3, "any": 1}[rows]
    return adapters._inputs(dev, m, K, n, rank, 3, per, ids=ids, seed=rank + m, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("tile", SIZES)
@pytest.mark.parametrize("rank", [8, 32, 64, 96])
@pytest.mark.parametrize("rows", ["one", "three", "any"])
def test_ranks_and_rows(gpu_device, tile, rank, rows):
    adapters._check(_inputs(gpu_device, tile, rank, rows))


@pytest.mark.gpu
@pytest.mark.parametrize("tile", SIZES)
@pytest.mark.parametrize("rank", [32, 64, 96])
@pytest.mark.parametrize("rows", ["one", "three", "any"])
def test_gated_residual(gpu_device, tile, rank, rows):
    adapters._check(_inputs(gpu_device, tile, rank, rows, residual=True, gate=True))


@pytest.mark.gpu
@pytest.mark.parametrize("tile", SIZES)
@pytest.mark.parametrize("rank", [24, 96, 192, 240])
@pytest.mark.parametrize("rows", ["one", "three", "any"])
def test_parts(gpu_device, tile, rank, rows):
    """Three parts of 8 to 80 ranks, alternately with a residual."""
    a = _inputs(gpu_device, tile, rank, rows, residual=rank % 64 == 32)
    a["up"], a["parts"] = a["up"][..., :rank // 3].contiguous(), 3
    got = adapters._check(a)
    assert torch.equal(got, kernel.turing_int8_linear_adapters(**a))
