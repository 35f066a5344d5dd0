"""GPU: attention over the key/value cache in 8 bits where both the pages' value scales
and their scores lie far apart, against its definition in 64 bits: the page that takes
the softmax is then one whose values are too small to matter, or zeros."""
from __future__ import annotations

import math

import pytest
import torch

from comfyui_turing_utils_kernel import _lib
from tests.test_gpu_cache_attn import _check, _ints, _pool, _query

# (query tokens, K/V heads of the two sequences): rows a workgroup
ROWS = {(1, 1): 16, (20, 1): 16, (140, 1): 16, (140, 33): 128, (256, 66): 256}


def test_the_sizes_take_the_forms():
    for (lq, heads), rows in ROWS.items():
        for kind in (0, 2):
            for most in (64, 384):
                assert _lib.load().tu_kv_cache_attn_plan(2, heads, heads, lq, 64, most, kind, 0, 256) == rows << 16 | 1


def _leads(device, lq, heads, kind, lead, ratio, order, row=6, page=3):
    """(query, pool, table, kw): scores around 0 but those of page `page`, which are `lead` higher, as log2 of the weight;
    its values' scale is `ratio` of the others'.  order "first": it is the sequence's first page."""
    pool, table, g = _pool(device, 2, heads, 64, row, 31)
    q, kw = _query(device, 2, heads, lq, 64, kind, "HND", g)
    if order == "first":
        table[:, [0, page]] = table[:, [page, 0]]
        page = 0
    high = table[:, page].long()
    q[..., 0] = 40 if kind == "int8" else 1.0
    if kind == "int8":
        kw["query_scale"] = torch.full_like(kw["query_scale"], 1 / 40)
    pool[2].fill_(0.001)
    pool[0][..., 0] = 0
    pool[0][high] = 0
    pool[0][high, :, :, 0] = 100 + torch.randint(-1, 2, (2, heads, 64), generator=g).to(torch.int8).to(device)
    pool[2][high] = lead * math.log(2) * 8 / 100  # (sm_scale is 1 / 8)
    pool[3].fill_(0.01)
    pool[3][high] *= ratio
    return q, pool, table, kw


@pytest.mark.gpu
@pytest.mark.parametrize("lq,heads", ROWS)
@pytest.mark.parametrize("kind", ["bf16", "int8"])
@pytest.mark.parametrize("lead", [60, 68, 75, 85])
@pytest.mark.parametrize("ratio", [1e-25, 0.0])
def test_small_values_of_high_scores(gpu_device, lq, heads, kind, lead, ratio):
    """The sum counts the page whole, its values enter with their own scale.  (With max_length 64 one range has them all,
    and a wave of few rows pages 0 and 4.)"""
    for order, page in (("first", 3), ("later", 3), ("later", 4)):
        q, pool, table, kw = _leads(gpu_device, lq, heads, kind, lead, ratio, order, page=page)
        for most in (None, 64):
            got = _check(q, pool, table, _ints([384, 290], gpu_device), max_length=most, **kw)
            assert torch.isfinite(got).all()


@pytest.mark.gpu
@pytest.mark.parametrize("lq,heads", ROWS)
@pytest.mark.parametrize("order", ["first", "later"])
@pytest.mark.parametrize("lead", [0, 30, 100, 170])
def test_scales_at_both_ends(gpu_device, lq, heads, order, lead):
    """Values of 2^100 and pages of the least scale a cache writes (1e-7 / 127), 2^130 apart."""
    q, pool, table, kw = _leads(gpu_device, lq, heads, "bf16", lead, 1.0, order)
    pool[3].fill_(2.0 ** 100)
    pool[3][table[:, 0 if order == "first" else 3].long()] = 1e-7 / 127
    _check(q, pool, table, _ints([384, 250], gpu_device), **kw)
