"""GPU: ``turing_int8_linear_adapters`` where the down-projection's result, or a
weight, leaves the range of bf16: infinities and NaN as the formula has them."""
from __future__ import annotations

import pytest
import torch

import comfyui_turing_utils_kernel as kernel
from tests import operator_reference as ref
from tests import test_gpu_adapters as adapters

pytestmark = pytest.mark.gpu

INF = float("inf")
# rows, K, columns, rank, adapters: one row, mixed rows, rows sorted by adapter, several fragments of one adapter
SIZES = [(1, 64, 32, 8, 1), (61, 256, 200, 40, 3), (300, 128, 72, 24, 8), (2050, 128, 256, 64, 1)]


def _inputs(dev, m, k, n, rank, count, **kw):
    """Codes and down weights above zero, so that h is, up weights of both signs."""
    a = adapters._inputs(dev, m, k, n, rank, count, ids=[i % (count + 1) - 1 for i in range(m)] if count > 1 else [0] * m,
                         seed=m, **kw)
    a["activation"] = a["activation"].abs().clamp_min(1)  # -128 stays below zero: as 1
    a["activation"][a["activation"] < 0] = 1
    a["down"] = a["down"].abs().clamp_min(2.0 ** -10)
    return a


def _compare(a):
    print(f"[adapters] {tuple(a['activation'].shape)} rank {a['down'].shape[1]} count {a['down'].shape[0]}", flush=True)
    got = kernel.turing_int8_linear_adapters(**a)
    want, bound = ref.linear(a["activation"], a["weight"], a["activation_scale"], a["weight_scale"], a["bias"],
                             a["down"], a["up"], a["scaling"], a["adapter_ids"], a["adapter_rows"])
    finite = want.isfinite()
    assert torch.equal(got.isnan(), want.isnan()), (int(got.isnan().sum()), int(want.isnan().sum()))
    assert torch.equal(got.double()[want.isinf()], want[want.isinf()])
    assert bool(((got.double() - want).abs() <= bound)[finite].all())
    return want


@pytest.mark.parametrize("size", SIZES)
@pytest.mark.parametrize("signs", ["one", "both"])
def test_an_infinite_adapter(gpu_device, size, signs):
    """Infinite scaling: columns whose weights have one sign are infinite, those of both signs NaN."""
    a = _inputs(gpu_device, *size)
    a["scaling"][-1] = INF
    if signs == "one":
        column = torch.arange(size[2], device=gpu_device) % 3 - 1
        a["up"] = a["up"].abs().clamp_min(2.0 ** -6) * torch.where(column == 0, 1, column)[:, None]
    want = _compare(a)
    assert want.isinf().any() if signs == "one" else want.isnan().any()


@pytest.mark.parametrize("size", SIZES)
def test_results_past_the_largest_bf16(gpu_device, size):
    """Finite in fp32, infinite if rounded to bf16 alone."""
    m, k, n, rank, count = size
    a = _inputs(gpu_device, *size)
    a["activation"].fill_(1)
    a["activation_scale"].fill_(1.0)
    a["down"].fill_(1.0)
    a["scaling"].fill_(3.4e38 / k)
    a["up"] = (a["up"].float() * 2.0 ** -100).to(torch.bfloat16)
    h = torch.tensor(3.4e38 / k, dtype=torch.float32) * k
    assert h.isfinite() and h.to(torch.bfloat16).isinf()
    assert _compare(a).isfinite().all()
