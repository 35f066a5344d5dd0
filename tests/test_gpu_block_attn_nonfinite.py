"""GPU: ``key_block_attention`` where scales are no numbers, infinite, tiny or
huge, against the 64-bit reference of tests/operator_reference.py: a row is
NaN where the softmax of the scores it sees is, and nowhere else.  Grids whose
lists are split into ranges and grids whose lists are not."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import _lib, turing_sage
from tests import operator_reference as ref
from tests import test_gpu_block_attn as attn

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")
# query rows, keys, entries of a list: up to six entries are never split
FORMS = {"whole": (300, 700, 5), "split": (150, 9000, 100)}


def _parts(b, hq, lq, d, width):
    return _lib.load().tu_sage_block_attn_workspace(b, hq, lq, d, width, 256) > 0


def _compare(args, index, causal=False, blkq=16, blkk=64, ql=None, kl=None):
    """The call against the reference, NaN for NaN; returns (output, rows that are NaN)."""
    q8, qs, k8, ks, vt = args
    print(f"[block attn] Q{tuple(q8.shape)} K{tuple(k8.shape)} list {index.size(-1)} causal {causal}", flush=True)
    got = turing_sage.key_block_attention(*args, index, is_causal=causal, blkq=blkq, blkk=blkk, query_lengths=ql,
                                          key_lengths=kl)
    want, size = ref.attend(*args, index, "HND", causal, q8.size(-1) ** -0.5, blkq, blkk, ql, kl)
    none = want.isnan()
    assert torch.equal(got.isnan(), none), (int(got.isnan().sum()), int(none.sum()))
    off, bound = (got.double() - want).abs(), ref.attend_bound(want, size)
    assert bool((off <= bound)[~none].all()), float((off / bound)[~none].max())
    return got, none.any(-1)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("value", [NAN, INF])
@pytest.mark.parametrize("side", ["query", "key"])
def test_scales_that_are_no_numbers(gpu_device, d, form, causal, value, side):
    """As the quantizer leaves them: codes of zero where a scale is infinite.
    Every third block of keys, or every fourth group of 16 queries; rows that
    see none of such keys, and no such row itself, keep their values."""
    lq, lk, width = FORMS[form]
    q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 2, 4, 2, lq, lk, d, blkq=16, blkk=64, seed=d + lq)
    assert _parts(2, 4, lq, d, width) == (form == "split")
    index = attn._random_lists(2, 4, lq, lk, width, g, gpu_device)
    if side == "key":
        # few enough that some rows see none
        ks[0, :, 1::(3 if form == "whole" else 60)] = value
        at = (~ks.isfinite()).repeat_interleave(64, 2)[:, :, :lk]
        k8[at] = 0
        index[0, 0] = torch.arange(width, device=gpu_device)  # and the blocks on the diagonal
    else:
        qs[:, 1, ::4] = value
        at = (~qs.isfinite()).repeat_interleave(16, 2)[:, :, :lq]
        q8[at] = 0
    _, rows = _compare((q8, qs, k8, ks, vt), index, causal)
    assert rows.any() and not rows.all()


@pytest.mark.parametrize("form", FORMS)
def test_a_range_that_is_nan_is_not_left_out(gpu_device, form):
    """One NaN block anywhere in a list makes every row of it NaN, however the list is cut."""
    lq, lk, width = FORMS[form]
    *args, _ = attn._inputs(gpu_device, 1, 2, 2, lq, lk, 128, blkq=16, blkk=64, seed=3)
    index = torch.arange(width, dtype=torch.int32, device=gpu_device).expand(1, 2, (lq + 127) // 128, width).contiguous()
    for at in sorted({0, 1, width // 2, width - 1}):
        scales = args[3].clone()
        scales[:, 0, at] = NAN
        got, rows = _compare((args[0], args[1], args[2], scales, args[4]), index)
        assert rows[:, 0].all() and not rows[:, 1].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("value", [NAN, INF, 30.0, 0.0])
def test_queries_behind_the_end_leave_the_others_their_bits(gpu_device, d, causal, value):
    """Rows behind the sample's end that share a wave with rows in front of it:
    any scales, any codes."""
    *args, g = attn._inputs(gpu_device, 1, 2, 2, 300, 300, d, blkq=16, blkk=64, seed=4)
    index = attn._random_lists(1, 2, 300, 300, 5, g, gpu_device)
    ql = torch.tensor([131], dtype=torch.int32, device=gpu_device)
    kw = dict(is_causal=causal, blkq=16, blkk=64, query_lengths=ql)
    clean = turing_sage.key_block_attention(*args, index, **kw)
    args[1][:, :, 9:] = value  # from row 144 on
    args[0][:, :, 131:] = 127
    got = turing_sage.key_block_attention(*args, index, **kw)
    assert torch.equal(got, clean) and torch.isfinite(got).all()


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("power", [-100, -70, 70, 100])
def test_scales_far_apart_whose_product_is_ordinary(gpu_device, form, power):
    """2^-n beside 2^n: every product is the same number, and so is the result."""
    lq, lk, width = FORMS[form]
    q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 1, 2, 1, lq, lk, 128, blkq=16, blkk=64, seed=5)
    index = attn._random_lists(1, 2, lq, lk, width, g, gpu_device)
    for causal in (False, True):
        want, _ = _compare((q8, qs, k8, ks, vt), index, causal)
        got, _ = _compare((q8, qs * 2.0 ** power, k8, ks * 2.0 ** -power, vt), index, causal)
        assert torch.equal(got, want)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("causal", [False, True])
def test_scores_below_every_ordinary_number(gpu_device, form, causal):
    """Finite scores of -1e32 to -1e36 alone: the largest takes the row."""
    lq, lk, width = FORMS[form]
    q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 1, 2, 2, lq, lk, 128, blkq=16, blkk=64, seed=6)
    q8, k8 = q8.abs().clamp_min(1), -k8.abs().clamp_min(1)
    # one scale: scores are one factor times whole numbers, equal or far apart
    qs.fill_(2.0 ** 50), ks.fill_(2.0 ** 50)
    index = attn._random_lists(1, 2, lq, lk, width, g, gpu_device)
    _, rows = _compare((q8, qs, k8, ks, vt), index, causal)
    assert not rows.any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("power", [3, 7, 9, 11, 13, 15, 17, 21, 40, 90])
def test_scores_of_any_size(gpu_device, d, form, power):
    """One factor of 2^power / 8 or so times whole numbers, positive and
    negative: past 2^11 or so the largest score takes the row, and scores that
    are equal share it."""
    lq, lk, width = FORMS[form]
    q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 1, 2, 2, lq, lk, d, blkq=16, blkk=64, seed=7)
    qs.fill_(1.37), ks.fill_(2.0 ** power)
    index = attn._random_lists(1, 2, lq, lk, width, g, gpu_device)
    _, rows = _compare((q8, qs, k8, ks, vt), index)
    assert not rows.any()


@pytest.mark.parametrize("where", ["q", "k"])
@pytest.mark.parametrize("lq,lk", [(300, 300), (1, 9000)])
def test_an_infinite_input_gives_what_the_dense_attention_gives(gpu_device, where, lq, lk):
    """One infinite element of Q (its block of rows is NaN) or, with K's mean
    taken off, of K (its head is): every block kept, the rows that are NaN are
    those of the dense attention."""
    g = torch.Generator().manual_seed(8)
    q = torch.randn(1, 2, lq, 128, generator=g).to(torch.bfloat16).to(gpu_device)
    k, v = (torch.randn(1, 2, lk, 128, generator=g).to(torch.bfloat16).to(gpu_device) for _ in range(2))
    (q if where == "q" else k)[0, 1, min(lq, lk) - 1, 5] = INF
    dense = turing_sage.sageattn(q, k, v)
    got = turing_sage.sparse_sageattn(q, k, v, keep=(lk + 63) // 64)
    assert dense[:, 1].isnan().any() and torch.equal(got.isnan(), dense.isnan())


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_waves_of_ordinary_and_of_far_scores_side_by_side(gpu_device, d, causal):
    """Rows 32 .. 63 of every query block have scores of 2^30 and more, the
    others ordinary ones; 800 query blocks, so that no list is split, with lists
    of up to 280 entries, a segment and some."""
    lq, lk, width = 128 * 40 - 3, 64 * 320, 280
    q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 1, 20, 20, lq, lk, d, blkq=16, blkk=64, seed=9)
    assert not _parts(1, 20, lq, d, width)
    ks.fill_(2.0 ** -6)
    qs.fill_(1.0)
    group = torch.arange(qs.size(2), device=gpu_device) % 8
    qs[:, :, (group == 2) | (group == 3)] = 2.0 ** 24
    index = attn._random_lists(1, 20, lq, lk, width, g, gpu_device)
    got = turing_sage.key_block_attention(q8, qs, k8, ks, vt, index, is_causal=causal, blkq=16, blkk=64)
    assert torch.equal(got, turing_sage.key_block_attention(q8, qs, k8, ks, vt, index, is_causal=causal, blkq=16, blkk=64))
    two = [t[:, 3:5] for t in (q8, qs, k8, ks, vt, index)]
    want, size = ref.attend(*two, "HND", causal, d ** -0.5, 16, 64)
    off, bound = (got[:, 3:5].double() - want).abs(), ref.attend_bound(want, size)
    assert bool((off <= bound).all()), float((off / bound.clamp_min(1e-30)).max())
