"""GPU: attention over the key/value cache in 8 bits with queries at the edges of what
bf16 and fp16 hold: rows with channels far above the others, rows of any size, scores so
far apart that one key takes all."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import _lib, turing_sage
from tests import cache_reference as ref
from tests.test_gpu_cache_attn import _check, _ints, _pool, _query

# (query tokens, K/V heads of the two sequences): rows a workgroup
ROWS = {(1, 2): 16, (40, 2): 16, (140, 33): 128, (260, 100): 256}


def test_the_sizes_take_the_forms():
    for (lq, heads), rows in ROWS.items():
        for kind in (0, 1):
            assert _lib.load().tu_kv_cache_attn_plan(2, heads, heads, lq, 64, 256, kind, 1, 256) == rows << 16 | 1


@pytest.mark.gpu
@pytest.mark.parametrize("lq,heads", ROWS)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("times", [30.0, 1000.0])
def test_channels_far_above_the_others(gpu_device, lq, heads, kind, times):
    """The other channels are held to half a unit of 16 bits of the largest, and no better: the bound counts that."""
    pool, table, g = _pool(gpu_device, 2, heads, 64, 4, 41)
    q, kw = _query(gpu_device, 2, heads, lq, 64, kind, "HND", g)
    q[..., 9] *= times
    pool[0][..., 9] = 1  # (scores that the other channels still decide)
    _check(q, pool, table, _ints([200, 256], gpu_device), causal=True, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,heads", ROWS)
@pytest.mark.parametrize("size", [1e-33, 1e-31, 1e-20, 1e20, 1e33])
def test_rows_of_any_size(gpu_device, lq, heads, size):
    """Small queries of large keys, and the other way about: the same scores."""
    pool, table, g = _pool(gpu_device, 2, heads, 64, 4, 43)
    q, kw = _query(gpu_device, 2, heads, lq, 64, "bf16", "HND", g)
    q = (q.double() * size).to(torch.bfloat16)
    pool[2].copy_(pool[2].double() / size)
    _check(q, pool, table, _ints([200, 256], gpu_device), causal=True, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,heads", ROWS)
def test_rows_of_next_to_nothing(gpu_device, lq, heads):
    """Rows below 1e-33 are held to half a unit of 1e-33 / 32512, zeros exactly: weights all alike."""
    pool, table, g = _pool(gpu_device, 2, heads, 64, 4, 45)
    q, kw = _query(gpu_device, 2, heads, lq, 64, "bf16", "HND", g)
    for size in (0.0, 1e-36, 9.2e-41):
        _check(q * size, pool, table, _ints([200, 256], gpu_device), causal=True, **kw)


@pytest.mark.gpu
@pytest.mark.parametrize("lq,heads", ROWS)
@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("size", [1e4, 1e12, 1e30])
def test_far_scores_of_floats(gpu_device, lq, heads, kind, size):
    """A key whose score is ahead of the others' by more than twice their error, that of a query's elements (half a unit
    of 16 bits of the row's largest, times the key's elements) and ten roundings of 32 bits, and by 200 besides, which is
    a weight of no size, takes all: the row is that key's value, a product of a code and two factors of 32 bits, rounded
    once.  Any other row is a mean of values."""
    pool, table, g = _pool(gpu_device, 2, heads, 64, 4, 47)
    pool[2].mul_(size)
    q, _ = _query(gpu_device, 2, heads, lq, 64, kind, "HND", g)
    got = turing_sage.kv_cache_attention(q, turing_sage.QuantizedKVCache(*pool), table, _ints([200, 256], gpu_device),
                                         is_causal=True).double()
    assert torch.isfinite(got).all()
    clear, half = 0, ref.HALF[q.dtype]
    for b, length in enumerate((200, 256)):
        k, v, ks, vs, _ = ref.sequence(pool, table, length, b)
        for h in range(heads):
            x = q[b, h].double()
            s = (x @ k[h].t()) * 0.125 * ks[h]
            off = x.abs().amax(1, keepdim=True) / 65024 * k[h].abs().sum(1) * 0.125 * ks[h] + 10 * 2.0 ** -24 * s.abs()
            hidden = torch.arange(length, device=s.device) > length - lq + torch.arange(lq, device=s.device)[:, None]
            seen = ~hidden.all(1)
            s.masked_fill_(hidden, -torch.inf)
            two, at = s.topk(2, 1)
            wins = seen & (two[:, 0] - two[:, 1] > 2 * off.masked_fill(hidden, 0).amax(1) + 200)
            want = (v[h] * vs[h][:, None])[at[:, 0]]
            assert bool(((got[b, h] - want).abs() <= (half + 2.0 ** -20) * want.abs() + 2.0 ** -25)[wins].all()), (b, h)
            most = (v[h] * vs[h][:, None]).abs().amax(0) * (1 + 2 * half + 2.0 ** -11)
            assert bool((got[b, h].abs() <= most).all()), (b, h)
            clear += int(wins.sum())
    assert clear > 0.9 * 2 * heads * min(lq, 200)
