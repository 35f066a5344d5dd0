"""GPU: calls of the adapters that their documentation allows and no ordinary
program makes."""
from __future__ import annotations

import pytest
import torch

import comfyui_turing_utils_kernel as kernel
from tests import test_gpu_adapters as adapters

pytestmark = pytest.mark.gpu


def _column(t):
    """The same values as a column of a table."""
    table = torch.zeros(t.numel(), 3, dtype=t.dtype, device=t.device)
    table[:, 1] = t
    return table[:, 1]


@pytest.mark.parametrize("m,count", [(3, 3), (64, 64), (700, 5)])
def test_strided_scaling_and_ids(gpu_device, m, count):
    """Scalings and ids that are columns of a table, or one value for all."""
    a = adapters._inputs(gpu_device, m, 256, 128, 16, count, seed=m)
    want = kernel.turing_int8_linear_adapters(**a)
    b = dict(a, scaling=_column(a["scaling"]), adapter_ids=_column(a["adapter_ids"]))
    for _ in range(4):
        assert torch.equal(kernel.turing_int8_linear_adapters(**b), want)
    same = dict(a, scaling=a["scaling"][:1].clone().expand(count), adapter_ids=_column(a["adapter_ids"]))
    full = dict(a, scaling=same["scaling"].contiguous())
    assert torch.equal(kernel.turing_int8_linear_adapters(**same), kernel.turing_int8_linear_adapters(**full))
