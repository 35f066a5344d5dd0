"""GPU: attention over the key/value cache in 8 bits against its definition in 64
bits, with a bound derived from the kernel's arithmetic."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import turing_sage
from tests import cache_reference as ref

pytestmark = pytest.mark.gpu


def _pool(device, batch, heads, d, row, seed, spread=1.0):
    """(pool, table, generator): every page holds codes and scales that tokens could have."""
    g = torch.Generator().manual_seed(seed)
    table, pages = ref.tables(batch, row, g, device)
    codes = [torch.randn(pages, heads, *shape, generator=g).mul(40).round().clamp(-127, 127).to(torch.int8).to(device)
             for shape in ((64, d), (d, 64))]
    scales = [((0.5 + torch.rand(pages, heads, generator=g)) * 0.03 * spread).to(device) for _ in range(2)]
    return [*codes, *scales], table, g


def _query(device, b, hq, lq, d, kind, layout, g, blkq=16):
    x = torch.randn(b, hq, lq, d, generator=g)
    if kind == "int8":
        x = x.mul(40).round().clamp(-127, 127).to(torch.int8)
        scale = ((0.5 + torch.rand(b, hq, (lq + blkq - 1) // blkq, generator=g)) * 0.03).to(device)
        kw = dict(query_scale=scale, blkq=blkq)
    else:
        x, kw = x.to(dict(bf16=torch.bfloat16, f16=torch.float16)[kind]), {}
    return (x if layout == "HND" else x.transpose(1, 2).contiguous()).to(device), kw


def _ints(values, device):
    return None if values is None else torch.tensor(values, dtype=torch.int32, device=device)


def _check(query, pool, table, lengths, layout="HND", causal=False, max_length=None, **kw):
    cache = turing_sage.QuantizedKVCache(*pool)
    got = turing_sage.kv_cache_attention(query, cache, table, lengths, tensor_layout=layout, is_causal=causal,
                                         max_length=max_length, **kw)
    want, bound = ref.attend(query, pool, table, lengths, layout, causal, **kw)
    assert got.shape == query.shape and got.dtype == (torch.bfloat16 if "query_scale" in kw else query.dtype)
    off = (got.double() - want).abs()
    assert bool((off <= bound).all()), f"{float((off - bound).max()):.3g} past the bound, {int((off > bound).sum())} of {off.numel()}"
    return got


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["bf16", "f16", "int8"])
@pytest.mark.parametrize("hq,hkv", [(3, 3), (8, 2), (40, 2), (5, 1)])
@pytest.mark.parametrize("lengths", [[1, 0, 63, 64, 65], [700, 1, 0, 513, 300]])
def test_single_tokens(gpu_device, d, kind, hq, hkv, lengths):
    pool, table, g = _pool(gpu_device, 5, hkv, d, 11, d + hq)
    for layout in ("HND", "NHD"):
        q, kw = _query(gpu_device, 5, hq, 1, d, kind, layout, g)
        for causal in (False, True):
            got = _check(q, pool, table, _ints(lengths, gpu_device), layout, causal, **kw)
        assert not got[lengths.index(0)].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", ["bf16", "f16", "int8"])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("hq,hkv,lq,lengths,counts", [
    (4, 4, 2, [2, 300, 1], None), (4, 4, 7, [7, 64, 0], [7, 3, 0]), (8, 1, 3, [100, 130, 64], None),
    (2, 2, 17, [17, 500, 16], [17, 16, 17]), (6, 2, 33, [300, 65, 640], [33, 1, 20]),
    (2, 1, 130, [130, 700, 129], None), (3, 3, 300, [300, 704, 20], [300, 257, 300]), (1, 1, 128, [128, 1, 704], None),
])
def test_chunks(gpu_device, d, kind, causal, hq, hkv, lq, lengths, counts):
    """Few and many rows, ends inside tiles, sequences shorter than their queries, rows without keys."""
    pool, table, g = _pool(gpu_device, 3, hkv, d, 11, d + lq)
    layout = "NHD" if lq % 2 else "HND"
    q, kw = _query(gpu_device, 3, hq, lq, d, kind, layout, g)
    got = _check(q, pool, table, _ints(lengths, gpu_device), layout, causal, query_lengths=_ints(counts, gpu_device), **kw)
    rows = ref.hnd(got, layout)
    for b, n in enumerate(counts or []):
        assert not rows[b, :, n:].any()


@pytest.mark.parametrize("kind,blkq", [("int8", 1), ("int8", 128), ("int8", 48)])
def test_query_blocks(gpu_device, kind, blkq):
    pool, table, g = _pool(gpu_device, 2, 2, 64, 4, blkq)
    for lq in (1, 70, 200):
        q, kw = _query(gpu_device, 2, 4, lq, 64, kind, "HND", g, blkq)
        _check(q, pool, table, _ints([200, 256], gpu_device), causal=True, **kw)


@pytest.mark.parametrize("lq", [1, 40])
@pytest.mark.parametrize("d", [64, 128])
def test_long_sequences(gpu_device, d, lq):
    """Many pages a unit: past the pages that a wave knows at once, whatever length the split was made for."""
    pool, table, g = _pool(gpu_device, 2, 1, d, 700, 5)
    q, kw = _query(gpu_device, 2, 2, lq, d, "bf16", "HND", g)
    lengths = _ints([44700, 20001], gpu_device)
    for most in (None, 1, 64 * 3, 64 * 300):
        _check(q, pool, table, lengths, causal=True, max_length=most, **kw)


@pytest.mark.parametrize("lq", [1, 50, 130])
def test_pages_that_are_none(gpu_device, lq):
    """Table entries outside the pool: their keys are not seen."""
    pool, table, g = _pool(gpu_device, 3, 2, 64, 9, 7)
    table[0, 2], table[0, 3], table[1, 0], table[2] = -1, 10 ** 6, -(10 ** 9), -1
    q, _ = _query(gpu_device, 3, 4, lq, 64, "bf16", "HND", g)
    got = _check(q, pool, table, _ints([570, 64 if lq == 1 else 200, 300], gpu_device), causal=True)
    assert not got[2].any()


@pytest.mark.parametrize("lq", [1, 20, 140])
@pytest.mark.parametrize("d", [64, 128])
def test_what_is_not_seen_changes_nothing(gpu_device, d, lq):
    """Codes behind the ends, pages of no table, and rows behind a sequence's queries: any bytes, the same bits."""
    pool, table, g = _pool(gpu_device, 2, 2, d, 6, 3)
    q, _ = _query(gpu_device, 2, 4, lq, d, "bf16", "HND", g)
    lengths, counts = _ints([200, 333], gpu_device), _ints([lq, max(1, lq - 5)], gpu_device)
    cache = turing_sage.QuantizedKVCache(*pool)
    kw = dict(is_causal=True, query_lengths=counts)
    want = turing_sage.kv_cache_attention(q, cache, table, lengths, **kw)
    for b, length in enumerate((200, 333)):
        page, rest = int(table[b, length // 64]), length % 64
        pool[0][page, :, rest:] = -128
        pool[1][page, :, :, rest:] = -128
        behind = table[b, length // 64 + 1:].long()
        pool[2][behind], pool[3][behind] = float("nan"), float("inf")
    if lq > 5:
        q[1, :, lq - 5:] = float("nan")
    got = turing_sage.kv_cache_attention(q, cache, table, lengths, **kw)
    assert torch.equal(got, want) and torch.isfinite(got).all()


@pytest.mark.parametrize("lq", [1, 30, 200])
@pytest.mark.parametrize("which,value", [(2, float("nan")), (2, float("inf")), (3, float("nan")), (3, float("inf"))])
def test_scales_that_are_no_numbers(gpu_device, lq, which, value):
    """NaN of the rows that see the page, and of no others."""
    pool, table, g = _pool(gpu_device, 2, 2, 64, 6, lq)
    q, _ = _query(gpu_device, 2, 2, lq, 64, "bf16", "HND", g)
    lengths = _ints([300, 300], gpu_device)
    clean = turing_sage.kv_cache_attention(q, turing_sage.QuantizedKVCache(*pool), table, lengths, is_causal=True)
    pool[which][int(table[0, 3]), 1] = value  # keys 192 .. 255
    if which == 2 and value == float("inf"):
        pool[0][int(table[0, 3]), 1] = 0
    got = turing_sage.kv_cache_attention(q, turing_sage.QuantizedKVCache(*pool), table, lengths, is_causal=True)
    sees = torch.arange(300 - lq, 300, device=gpu_device) >= 192
    assert torch.isnan(got[0, 1][sees]).all()
    assert torch.equal(got[0, 1][~sees], clean[0, 1][~sees])
    assert torch.equal(got[0, 0], clean[0, 0]) and torch.equal(got[1], clean[1])


@pytest.mark.parametrize("lq", [1, 20, 140])
def test_queries_that_are_no_numbers(gpu_device, lq):
    pool, table, g = _pool(gpu_device, 1, 1, 64, 4, 2)
    q, _ = _query(gpu_device, 1, 2, lq, 64, "bf16", "HND", g)
    lengths = _ints([200], gpu_device)
    cache = turing_sage.QuantizedKVCache(*pool)
    want = turing_sage.kv_cache_attention(q, cache, table, lengths)
    q[0, 1, lq // 2, 5] = float("nan")
    q[0, 0, lq - 1, 60] = float("inf")
    got = turing_sage.kv_cache_attention(q, cache, table, lengths)
    bad = torch.zeros(1, 2, lq, dtype=torch.bool, device=gpu_device)
    bad[0, 1, lq // 2] = bad[0, 0, lq - 1] = True
    assert torch.isnan(got[bad]).all()
    off = (got[~bad].double() - want[~bad].double()).abs()
    # (a wave's rows share one form of the exponent)
    assert bool((off <= 2.0 ** -7 * want[~bad].double().abs() + 2.0 ** -10).all())


@pytest.mark.parametrize("lq", [1, 40])
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("size", [1e-6, 1e-3, 50.0, 1e4, 1e12, 1e30])
def test_scores_of_any_size(gpu_device, lq, kind, size):
    """From all weights alike to one key that takes all, past the exponent's fine range."""
    pool, table, g = _pool(gpu_device, 2, 2, 64, 5, 11)
    pool[2].mul_(size)
    q, kw = _query(gpu_device, 2, 2, lq, 64, kind, "HND", g)
    cache = turing_sage.QuantizedKVCache(*pool)
    lengths = _ints([300, 65], gpu_device)
    if size <= 50.0:
        _check(q, pool, table, lengths, **kw)
        return
    got = turing_sage.kv_cache_attention(q, cache, table, lengths, **kw).double()
    # the largest score takes all, by a distance that no rounding reaches
    want, _ = ref.attend(q, pool, table, lengths, "HND", False, **kw)
    if kind == "int8":
        assert bool(((got - want).abs() <= ref.HALF[torch.bfloat16] * want.abs() + 1e-6).all())
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("lq", [1, 20, 140])
@pytest.mark.parametrize("ratio", [1e-3, 1e-9, 1e-25, 0.0])
def test_pages_of_unlike_value_scales(gpu_device, lq, ratio):
    """Pages whose values are far smaller than others' still count in the sum of weights."""
    pool, table, g = _pool(gpu_device, 2, 1, 64, 6, 13)
    for order in ((0, 2), (3,)):
        scales = pool[3].clone()
        for j in order:
            scales[table[:, j].long()] *= ratio
        q, _ = _query(gpu_device, 2, 1, lq, 64, "bf16", "HND", g)
        _check(q, [*pool[:3], scales], table, _ints([384, 250], gpu_device))
    _check(q, [*pool[:3], pool[3] * ratio], table, _ints([384, 250], gpu_device))


def test_narrow_heads(gpu_device):
    for head_dim in (24, 72):
        width = 64 if head_dim <= 64 else 128
        pool, table, g = _pool(gpu_device, 2, 2, width, 4, head_dim)
        pool[0][..., head_dim:] = 0
        pool[1][:, :, head_dim:] = 0
        for lq in (1, 70):
            q, _ = _query(gpu_device, 2, 4, lq, head_dim, "bf16", "NHD", g)
            _check(q, pool, table, _ints([200, 256], gpu_device), "NHD")


def test_one_page_of_many_sequences(gpu_device):
    """Tables that share their first pages, as prompts with a common beginning do."""
    pool, table, g = _pool(gpu_device, 3, 2, 64, 5, 17)
    table[1:, :3] = table[0, :3]
    for lq in (1, 90):
        q, _ = _query(gpu_device, 3, 4, lq, 64, "bf16", "HND", g)
        _check(q, pool, table, _ints([320, 200, 250], gpu_device), causal=True)


def test_strided_queries(gpu_device):
    pool, table, g = _pool(gpu_device, 2, 2, 64, 4, 19)
    qkv = torch.randn(2, 50, 3, 4, 64, generator=g).to(torch.bfloat16).to(gpu_device)
    wide = torch.randn(2, 50, 4, 67, generator=g).to(torch.bfloat16).to(gpu_device)[..., 1:65]
    lengths = _ints([200, 256], gpu_device)
    for q in (qkv[:, :, 0], wide, qkv[:, :, 0].transpose(1, 2)):
        layout = "NHD" if q.size(1) == 50 else "HND"
        got = _check(q, pool, table, lengths, layout)
        again = _check(q.contiguous(), pool, table, lengths, layout)
        assert torch.equal(got, again)


def test_past_32_bits(gpu_device):
    """Pages whose bytes lie past 2^31 and 2^32 in the pool."""
    pages, heads, d = 70000, 8, 128  # 4.6 GB of codes each
    pool = [torch.zeros(pages, heads, 64, d, dtype=torch.int8, device=gpu_device),
            torch.zeros(pages, heads, d, 64, dtype=torch.int8, device=gpu_device),
            torch.full((pages, heads), 0.5, device=gpu_device), torch.full((pages, heads), 0.5, device=gpu_device)]
    cache = turing_sage.QuantizedKVCache(*pool)
    table = _ints([[69999, 3, 40000], [32768, 65536, 0]], gpu_device)
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, heads, 150, d, generator=g).to(torch.bfloat16).to(gpu_device)
    lengths = turing_sage.kv_cache_append(x, -x, cache, table, _ints([0, 0], gpu_device))
    k, v = turing_sage.kv_cache_read(cache, table, lengths, max_length=150)
    assert torch.equal(k, -v) and bool(((k - x).abs().double() <= 0.04).all())
    for lq in (1, 130):
        q, _ = _query(gpu_device, 2, heads, lq, d, "bf16", "HND", g)
        _check(q, pool, table, lengths, causal=True)
