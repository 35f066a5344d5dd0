"""GPU: writing the key/value cache in 8 bits and reading it back, bit for bit
against the formula in 32 bits, and the values in 64."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import turing_sage
from tests import cache_reference as ref

pytestmark = pytest.mark.gpu


def _tokens(b, heads, tokens, d, gen, dtype, layout, device):
    x = torch.randn(b, heads, tokens, d, generator=gen) + torch.randn(b, heads, 1, d, generator=gen)
    x = x.to(dtype)
    return (x if layout == "HND" else x.transpose(1, 2).contiguous()).to(device)


def _same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(a.cpu().nan_to_num(7777.0), b.nan_to_num(7777.0))


def _write(device, d, dtype, layout, tokens, held, new=None, codes=False, mean=False, heads=3, seed=0, row=5):
    g = torch.Generator().manual_seed(seed)
    b = len(held)
    table, pages = ref.tables(b, row, g, device)
    pool = ref.rubbish_pool(pages, heads, d, g, device)
    lengths = torch.tensor(held, dtype=torch.int32, device=device)
    for i, had in enumerate(held):  # (pages that hold earlier tokens have a scale)
        if had % 64:
            for scale in pool[2:]:
                scale[int(table[i, had // 64])] = torch.tensor([0.004, 0.02, 1.0])[:heads].to(device)
    key, value = (_tokens(b, heads, tokens, d, g, dtype, layout, device) for _ in range(2))
    kw = dict(new_lengths=None if new is None else torch.tensor(new, dtype=torch.int32, device=device))
    if codes:
        key = torch.randint(-127, 128, key.shape, generator=g, dtype=torch.int8).to(device)
        kw["key_scale"] = (0.01 + 0.03 * torch.rand(b, heads, ref.blocks(tokens), generator=g)).to(device)
    if mean:
        kw["key_mean"] = torch.randn(b, heads, d, generator=g).to(torch.bfloat16).to(device)
    want, after = ref.append(key, value, pool, table, lengths, layout, **kw)
    cache = turing_sage.QuantizedKVCache(*pool)
    got = turing_sage.kv_cache_append(key, value, cache, table, lengths, tensor_layout=layout, **kw)
    assert torch.equal(got.cpu(), after) and lengths.tolist() == held
    _same(cache.tensors, want)
    return cache, table, after.to(device), key, value, kw


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,codes,mean", [(torch.bfloat16, False, False), (torch.float16, False, True),
                                              (torch.bfloat16, True, False), (torch.float16, True, True)])
@pytest.mark.parametrize("tokens,held,new", [
    (1, [0, 1, 62, 63, 64, 130, 319, 320], None),           # single tokens; the last sequence is full
    (2, [63, 0, 126], [2, 0, 1]),
    (64, [0, 64, 1], None),
    (65, [0, 63, 200], [65, 64, 7]),
    (300, [0, 5, 64, 319], [300, 300, 129, 300]),           # past the last page's end
])
def test_append(gpu_device, d, dtype, codes, mean, layout, tokens, held, new):
    _write(gpu_device, d, dtype, layout, tokens, held, new, codes, mean, seed=tokens + d)


@pytest.mark.parametrize("d", [64, 128])
def test_values_are_within_half_a_step(gpu_device, d):
    """In 64 bits: what a page's codes stand for is half a scale from the inputs (and the rounding of the product)."""
    cache, table, after, key, value, _ = _write(gpu_device, d, torch.bfloat16, "HND", 200, [0, 64], seed=3)
    for b, first in ((0, 0), (1, 64)):
        k, v, ks, vs, _ = ref.sequence(cache.tensors, table, int(after[b]), b)
        for codes, scale, x in ((k, ks, key), (v, vs, value)):
            scale = scale[:, first:, None]
            off = (codes[:, first:] * scale - x[b].double()).abs()
            assert bool((off <= scale * (0.5 + 128 * 2.0 ** -22)).all())
            # a page's largest is a code of 127
            tops = codes[:, first:first + 192].view(3, 3, 64 * d).abs().amax(2)
            assert bool((tops == 127).all())


def test_token_by_token(gpu_device):
    """A page filled one token at a time: each step is the formula's, and the codes stay
    within the sum of half the scales they went through."""
    g = torch.Generator().manual_seed(1)
    table, pages = ref.tables(2, 2, g, gpu_device)
    pool = ref.rubbish_pool(pages, 2, 64, g, gpu_device)
    cache = turing_sage.QuantizedKVCache(*pool)
    lengths = torch.tensor([0, 40], dtype=torch.int32, device=gpu_device)
    pool[2][table[1, 0].long()] = 0.001
    pool[3][table[1, 0].long()] = 0.001
    x = _tokens(2, 2, 70, 64, g, torch.bfloat16, "HND", gpu_device)
    budget = torch.zeros(2, device=gpu_device, dtype=torch.float64)
    scale = torch.zeros(2, device=gpu_device, dtype=torch.float64)
    for t in range(70):
        want, after = ref.append(x[:, :, t:t + 1], -x[:, :, t:t + 1], cache.tensors, table, lengths, "HND")
        lengths = turing_sage.kv_cache_append(x[:, :, t:t + 1], -x[:, :, t:t + 1], cache, table, lengths)
        assert torch.equal(lengths.cpu(), after)
        _same(cache.tensors, want)
        if t < 64:
            now = cache.key_scale[table[0, 0].long()].double()
            budget += torch.where(now > scale, now / 2, 0.0)
            scale = now
    k, _, ks, _, _ = ref.sequence(cache.tensors, table, 64, 0)
    assert bool(((k * ks[..., None] - x[0, :, :64].double()).abs() <= budget[:, None, None] * 1.001).all())


def test_again_at_the_same_place(gpu_device):
    """A chunk written twice over (its next denoising step), with the lengths set back."""
    g = torch.Generator().manual_seed(2)
    state = turing_sage.SequenceKVCache.allocate(2, 300, 3, 128, gpu_device)
    first = _tokens(2, 3, 70, 128, g, torch.bfloat16, "NHD", gpu_device)
    state.append(first, first, tensor_layout="NHD")
    held = state.lengths.clone()
    for _ in range(3):
        chunk = _tokens(2, 3, 150, 128, g, torch.bfloat16, "NHD", gpu_device)
        want, after = ref.append(chunk, -chunk, state.cache.tensors, state.block_table, held, "NHD")
        state.lengths.copy_(held)
        state.append(chunk, -chunk, tensor_layout="NHD")
        _same(state.cache.tensors, want)
        assert state.lengths.tolist() == after.tolist() == [220, 220]
    k, v = state.read(max_length=220, tensor_layout="NHD")
    assert torch.equal(v[:, 70:], -k[:, 70:])


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3.3e38, 1e-30])
def test_extreme_inputs(gpu_device, bad):
    """Numbers that are none, the largest and tiny ones: the page and head of theirs alone."""
    g = torch.Generator().manual_seed(4)
    table, pages = ref.tables(1, 4, g, gpu_device)
    pool = ref.rubbish_pool(pages, 2, 64, g, gpu_device)
    lengths = torch.zeros(1, dtype=torch.int32, device=gpu_device)
    key, value = (_tokens(1, 2, 200, 64, g, torch.bfloat16, "HND", gpu_device) for _ in range(2))
    key[0, 0, 70, 3] = bad
    value[0, 1, 130, 60] = bad
    if bad == 1e-30:
        key[0, 1, 64:128] = bad
    want, _ = ref.append(key, value, pool, table, lengths, "HND")
    cache = turing_sage.QuantizedKVCache(*pool)
    after = turing_sage.kv_cache_append(key, value, cache, table, lengths)
    _same(cache.tensors, want)
    # a later token of the page leaves a scale that is no number
    key, value = key[:, :, :1], value[:, :, :1]
    back = torch.tensor([100], dtype=torch.int32, device=gpu_device)
    want, _ = ref.append(key, value, cache.tensors, table, back, "HND")
    turing_sage.kv_cache_append(key, value, cache, table, back)
    _same(cache.tensors, want)
    assert after.tolist() == [200]


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("max_length,starts,mean", [(1, None, False), (320, None, True), (333, [0, 63, 64, 300], False),
                                                    (7, [60, 1, 300, 9999], True), (64, [-5, 64, 10, 0], False)])
def test_read(gpu_device, d, dtype, layout, max_length, starts, mean):
    cache, table, after, *_ = _write(gpu_device, d, torch.bfloat16, "HND", 300, [0, 5, 64, 0], [300, 129, 1, 0], seed=9)
    table = table.clone()
    table[0, 1], table[1, 0] = -1, 10 ** 6  # no pages of the pool
    kw = dict(starts=None if starts is None else torch.tensor(starts, dtype=torch.int32, device=gpu_device))
    if mean:
        kw["key_mean"] = torch.randn(4, 3, d).to(torch.bfloat16).to(gpu_device)
    want = ref.read(cache.tensors, table, after, max_length, layout, dtype, **kw)
    got = turing_sage.kv_cache_read(cache, table, after, max_length=max_length, tensor_layout=layout, dtype=dtype, **kw)
    for a, b in zip(got, want):
        assert a.dtype == dtype and a.is_contiguous() and torch.equal(a.cpu().nan_to_num(77.0), b.nan_to_num(77.0))


def test_pages_that_are_none(gpu_device):
    """Tokens of a page outside the pool are dropped; the lengths count them."""
    g = torch.Generator().manual_seed(6)
    table, pages = ref.tables(2, 3, g, gpu_device)
    pool = ref.rubbish_pool(pages, 2, 64, g, gpu_device)
    table[0, 1], table[1, 0] = -7, pages
    lengths = torch.tensor([10, -4], dtype=torch.int32, device=gpu_device)
    pool[2].fill_(0.01), pool[3].fill_(0.01)
    x = _tokens(2, 2, 180, 64, g, torch.bfloat16, "HND", gpu_device)
    want, after = ref.append(x, x, pool, table, lengths, "HND")
    cache = turing_sage.QuantizedKVCache(*pool)
    got = turing_sage.kv_cache_append(x, x, cache, table, lengths)
    assert got.tolist() == after.tolist() == [190, 180]
    _same(cache.tensors, want)


def test_rows_behind_the_new_ones_are_not_read(gpu_device):
    """A padded batch: what stands behind a sequence's new tokens may be anything."""
    a = _write(gpu_device, 64, torch.bfloat16, "HND", 100, [0, 30], [100, 33], seed=8)
    g = torch.Generator().manual_seed(8)
    table, pages = ref.tables(2, 5, g, gpu_device)
    pool = ref.rubbish_pool(pages, 3, 64, g, gpu_device)
    key, value = a[3].clone(), a[4].clone()
    key[1, :, 33:] = float("nan")
    value[1, :, 33:] = float("inf")
    for scale in pool[2:]:
        scale[int(table[1, 0])] = torch.tensor([0.004, 0.02, 1.0]).to(gpu_device)
    cache = turing_sage.QuantizedKVCache(*pool)
    turing_sage.kv_cache_append(key, value, cache, table, torch.tensor([0, 30], dtype=torch.int32, device=gpu_device),
                                **a[5])
    for x, y in zip(cache.tensors, a[0].tensors):
        assert torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))


@pytest.mark.parametrize("head_dim", [8, 40, 72, 100])
def test_narrow_heads(gpu_device, head_dim):
    """A head_dim that is none of the kernel's: channels of zeros."""
    g = torch.Generator().manual_seed(head_dim)
    state = turing_sage.SequenceKVCache.allocate(2, 200, 2, head_dim, gpu_device)
    x = _tokens(2, 2, 130, head_dim, g, torch.bfloat16, "NHD", gpu_device)
    mean = torch.randn(2, 2, head_dim, generator=g).to(torch.bfloat16).to(gpu_device)
    want, _ = ref.append(x, x, state.cache.tensors, state.block_table, state.lengths, "NHD", key_mean=mean)
    state.append(x, x, tensor_layout="NHD", key_mean=mean)
    _same(state.cache.tensors, want)
    k, v = state.read(max_length=130, tensor_layout="NHD", key_mean=mean)
    width = 64 if head_dim <= 64 else 128
    assert k.shape == v.shape == (2, 130, 2, width) and not v[..., head_dim:].any() and not k[..., head_dim:].any()


def test_strided_inputs(gpu_device):
    """Keys and values as views of one fused projection, and ones that need a copy."""
    g = torch.Generator().manual_seed(12)
    qkv = torch.randn(2, 90, 3, 4, 64, generator=g).to(torch.bfloat16).to(gpu_device)
    k, v = qkv[:, :, 1], qkv[:, :, 2]
    odd = torch.randn(2, 90, 4, 67, generator=g).to(torch.bfloat16).to(gpu_device)[..., 1:65]
    for key, value in ((k, v), (odd, v), (k.transpose(1, 2), v.transpose(1, 2))):
        layout = "NHD" if key.size(1) == 90 else "HND"
        both = []
        for contiguous in (False, True):
            state = turing_sage.SequenceKVCache.allocate(2, 100, 4, 64, gpu_device)
            state.append(key.contiguous() if contiguous else key, value, tensor_layout=layout)
            both.append(state.cache.tensors)
        for a, b in zip(*both):
            assert torch.equal(a, b)
