"""GPU: attention over the key/value cache in 8 bits with queries at the edges of what
bf16 and fp16 hold."""
from __future__ import annotations

import pytest
import torch

from tests.test_gpu_cache_attn import _check, _ints, _pool, _query

pytestmark = pytest.mark.gpu

# (query tokens, K/V heads of the two sequences): few rows, and so many that they are taken in blocks of 128 and of 256
ROWS = [(1, 2), (40, 2), (140, 33), (256, 66)]


@pytest.mark.parametrize("lq,heads", ROWS)
@pytest.mark.parametrize("size", [1e-33, 1e-31, 1e-20, 1e20, 1e33])
def test_rows_of_any_size(gpu_device, lq, heads, size):
    """Small queries of large keys, and the other way about: the same scores."""
    pool, table, g = _pool(gpu_device, 2, heads, 64, 4, 43)
    q, kw = _query(gpu_device, 2, heads, lq, 64, "bf16", "HND", g)
    q = (q.double() * size).to(torch.bfloat16)
    pool[2].copy_(pool[2].double() / size)
    _check(q, pool, table, _ints([200, 256], gpu_device), causal=True, **kw)


@pytest.mark.parametrize("lq,heads", ROWS)
def test_rows_of_next_to_nothing(gpu_device, lq, heads):
    """Rows below 1e-33 are held to half a unit of 1e-33 / 32512, zeros exactly: weights all alike."""
    pool, table, g = _pool(gpu_device, 2, heads, 64, 4, 45)
    q, kw = _query(gpu_device, 2, heads, lq, 64, "bf16", "HND", g)
    for size in (0.0, 1e-36, 9.2e-41):
        _check(q * size, pool, table, _ints([200, 256], gpu_device), causal=True, **kw)
