"""GPU: attention over the key/value cache in 8 bits at calls of so many rows that the
launch takes them in blocks of 128, or, with more of those than compute units, of 256,
with and without a split of the keys.  The same properties and bounds as at small calls."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import _lib, turing_sage
from tests import cache_reference as ref
from tests.test_gpu_cache_attn import _check, _ints, _pool, _query

pytestmark = pytest.mark.gpu



@pytest.fixture(params=[33, 66])
def heads(request):
    """K/V heads of two sequences: of two blocks of 128 rows each 132 blocks, taken as they are, or 264, taken as 132 of
    256."""
    return request.param


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["bf16", "f16", "int8"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lq,lengths,counts", [(256, [256, 130], None), (131, [131, 576], [131, 7]), (250, [2, 500], [2, 250])])
def test_chunks(gpu_device, heads, d, kind, causal, lq, lengths, counts):
    pool, table, g = _pool(gpu_device, 2, heads, d, 9, d + lq)
    layout = "NHD" if lq % 2 else "HND"
    q, kw = _query(gpu_device, 2, heads, lq, d, kind, layout, g)
    got = _check(q, pool, table, _ints(lengths, gpu_device), layout, causal, query_lengths=_ints(counts, gpu_device), **kw)
    again = turing_sage.kv_cache_attention(q, turing_sage.QuantizedKVCache(*pool), table, _ints(lengths, gpu_device),
                                           tensor_layout=layout, is_causal=causal, query_lengths=_ints(counts, gpu_device), **kw)
    assert torch.equal(got, again)


@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_shared_heads(gpu_device, heads, kind):
    pool, table, g = _pool(gpu_device, 2, heads, 64, 4, 3)
    q, kw = _query(gpu_device, 2, 3 * heads, 70, 64, kind, "NHD", g)
    _check(q, pool, table, _ints([200, 70], gpu_device), "NHD", True, **kw)


def test_pages_that_are_none(gpu_device, heads):
    pool, table, g = _pool(gpu_device, 2, heads, 64, 9, 7)
    table[0, 2], table[0, 3], table[0, 8], table[1, 0] = -1, 10 ** 6, -5, -(10 ** 9)
    q, kw = _query(gpu_device, 2, heads, 200, 64, "int8", "HND", g)
    for causal in (False, True):
        _check(q, pool, table, _ints([570, 300], gpu_device), causal=causal, **kw)


@pytest.mark.parametrize("which,value", [(2, float("nan")), (3, float("inf")), (3, float("nan"))])
def test_scales_that_are_no_numbers(gpu_device, heads, which, value):
    """NaN in the rows that see the page, nothing elsewhere."""
    pool, table, g = _pool(gpu_device, 2, heads, 64, 6, 9)
    lengths = _ints([380, 384], gpu_device)
    q, _ = _query(gpu_device, 2, heads, 200, 64, "bf16", "HND", g)
    want = _check(q, pool, table, lengths, causal=True)
    pool[which][int(table[0, 4]), 5] = value  # keys 256 .. 319: of rows 76 on
    got = turing_sage.kv_cache_attention(q, turing_sage.QuantizedKVCache(*pool), table, lengths, is_causal=True)
    assert bool(got[0, 5, 76:].isnan().all())
    rest = torch.ones_like(got, dtype=torch.bool)
    rest[0, 5, 76:] = False
    assert torch.equal(got[rest], want[rest])


@pytest.mark.parametrize("ratio", [1e-9, 1e-25, 0.0])
def test_pages_of_unlike_value_scales(gpu_device, heads, ratio):
    pool, table, g = _pool(gpu_device, 2, heads, 64, 6, 9)
    scales = pool[3].clone()
    scales[table[0, ::2].long()] *= ratio
    scales[table[1, 1:3].long()] *= ratio
    q, _ = _query(gpu_device, 2, heads, 140, 64, "bf16", "HND", g)
    _check(q, [*pool[:3], scales], table, _ints([384, 250], gpu_device))


@pytest.mark.parametrize("size", [1e-6, 50.0, 1e4, 1e30])
def test_scores_of_any_size(gpu_device, heads, size):
    pool, table, g = _pool(gpu_device, 2, heads, 64, 4, 11)
    q, kw = _query(gpu_device, 2, heads, 140, 64, "int8", "HND", g)
    kw["query_scale"] = kw["query_scale"] * size
    lengths = _ints([200, 256], gpu_device)
    if size < 1e30:
        _check(q, pool, table, lengths, causal=True, **kw)
        return
    # A score of 1e30 is off by 1e24, and the bound of a weight is no number.  A row whose largest score is ahead of the
    # others by more than twice its error (10 * 2^-24 of it, as the bound counts) has that key's value, once rounded
    # to bf16 from the product of a code (times a weight of one power of two, exactly) and two factors of 32 bits; any
    # other row has a mean of values.
    got = turing_sage.kv_cache_attention(q, turing_sage.QuantizedKVCache(*pool), table, lengths, is_causal=True, **kw).double()
    clear = 0
    for b, length in enumerate((200, 256)):
        k, v, ks, vs, _ = ref.sequence(pool, table, length, b)
        for h in range(heads):
            x = q[b, h].double() * kw["query_scale"][b, h].double().repeat_interleave(16)[:140, None]
            s = (x @ k[h].t()) * 0.125 * ks[h]
            s.masked_fill_(torch.arange(length, device=s.device) > length - 140 + torch.arange(140, device=s.device)[:, None], -torch.inf)
            two, at = s.topk(2, 1)
            wins = two[:, 0] - two[:, 1] > 20 * 2.0 ** -24 * two.abs().amax(1)
            want = (v[h] * vs[h][:, None])[at[:, 0]]
            off = (got[b, h] - want).abs()
            assert bool((off <= (2.0 ** -8 + 2.0 ** -20) * want.abs())[wins].all()), (b, h)
            assert bool((got[b, h].abs() <= (v[h] * vs[h][:, None]).abs().amax(0) * (1 + 2.0 ** -8 + 2.0 ** -9)).all()), (b, h)
            clear += int(wins.sum())
    assert clear > 0.99 * 2 * heads * 140


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("d,heads,lq,kind", [(64, 18, 1020, "int8"), (64, 12, 1020, "bf16"), (128, 12, 1020, "int8"),
                                             (128, 8, 120, "f16")])
def test_a_split_of_many_rows(gpu_device, causal, d, heads, lq, kind):
    """Long keys and too few blocks of rows for the chip (of 128 rows in the first and last case, of 256 in the others):
    ranges of keys, past the pages that a wave knows at once."""
    pool, table, g = _pool(gpu_device, 1, heads, d, 400, 5)
    q, kw = _query(gpu_device, 1, heads, lq, d, kind, "NHD", g)
    most, cus = 25600, torch.cuda.get_device_properties(gpu_device).multi_processor_count
    code = dict(bf16=0, f16=1, int8=2)[kind]
    assert _lib.load().tu_kv_cache_attn_workspace(1, heads, heads, lq, d, most, code, int(causal), cus) > 0
    for length in (25555, 9000, lq):
        _check(q, pool, table, _ints([length], gpu_device), "NHD", causal, **kw)


@pytest.mark.parametrize("count", [60, 120])
def test_windows_of_pages(gpu_device, count):
    """One range of more pages than a wave knows at once, at 128 and at 256 rows a block."""
    pool, table, g = _pool(gpu_device, 1, count, 64, 150, 6)
    q, kw = _query(gpu_device, 1, count, 260, 64, "int8", "HND", g)
    table[0, 70] = -1
    for causal in (False, True):
        _check(q, pool, table, _ints([9570], gpu_device), causal=causal, **kw)
