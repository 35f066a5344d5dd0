"""GPU: calls of the block-sparse attention and the adapters that their
documentation allows and no ordinary program makes: overlapping and one-row
strides, lists longer than a compacted segment, scales that ask for a gradient,
tensors without data, and both routes of a facade."""
from __future__ import annotations

import pytest
import torch

import comfyui_turing_utils_kernel as kernel
from comfyui_turing_utils_kernel import turing_sage
from tests import operator_reference as ref
from tests import test_gpu_adapters as adapters
from tests import test_gpu_block_attn as attn

pytestmark = pytest.mark.gpu


def _both(args, index, **kw):
    """The facade's result, which the op has to repeat bit for bit."""
    got = attn._check(args, index, **kw)
    again = torch.ops.turing_utils.sage_block_attention(*args, index, "HND", kw.get("causal", False), -1.0, 128, 128)
    assert torch.equal(got, again)


@pytest.mark.parametrize("d", [64, 128])
def test_keys_that_share_memory(gpu_device, d):
    """A view whose keys are one row over and over, or overlap."""
    q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 1, 2, 2, 200, 500, d)
    index = attn._random_lists(1, 2, 200, 500, 5, g, gpu_device)
    one = k8[:, :, :1].expand(1, 2, 500, d)
    assert one.stride(2) == 0
    _both((q8, qs, one, ks, vt), index)
    flat = torch.randint(-127, 128, (2, 500 * 16 + d), generator=g, dtype=torch.int8).to(gpu_device)
    slide = flat.as_strided((1, 2, 500, d), (2 * flat.size(1), flat.size(1), 16, 1)) if flat.size(1) % 16 == 0 else None
    assert slide is not None
    _both((q8, qs, slide, ks, vt), index)
    for k in (one, slide):
        got = turing_sage.select_key_blocks(q8, qs, k, ks, keep=3)
        assert torch.equal(got.cpu(), ref.select(q8, qs, k, ks, 3, "HND", False, 0, 0, 128, 128))


@pytest.mark.parametrize("stride", [0, 16, 1 << 20])
def test_one_key_of_any_stride(gpu_device, stride):
    q8, qs, k8, ks, vt, _ = attn._inputs(gpu_device, 1, 2, 2, 130, 1, 64)
    key = k8.as_strided((1, 2, 1, 64), (128, 64, stride, 1))
    index = torch.zeros(1, 2, 2, 1, dtype=torch.int32, device=gpu_device)
    _both((q8, qs, key, ks, vt), index)


def test_lists_longer_than_a_segment(gpu_device):
    """800 query blocks, so that no list is split, of up to 300 and 600 entries, some out of order."""
    for lk, width in ((19199, 300), (64 * 600, 600)):
        q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 1, 20, 20, 128 * 40 - 3, lk, 64, seed=lk)
        index = attn._random_lists(1, 20, 128 * 40 - 3, lk, width, g, gpu_device)
        index[:, 3, 5] = index[:, 3, 5].flip(-1)
        index[:, 4, :, 255:257] = index[:, 4, :, 254:255]
        attn._check((q8[:, :5], qs[:, :5], k8[:, :5], ks[:, :5], vt[:, :5]), index[:, :5].contiguous())
        full = turing_sage.key_block_attention(q8, qs, k8, ks, vt, index)
        part = ref.attend(q8[:, 3:5], qs[:, 3:5], k8[:, 3:5], ks[:, 3:5], vt[:, 3:5], index[:, 3:5], "HND", False, 0.125,
                          128, 128)
        assert bool(((full[:, 3:5].double() - part[0]).abs() <= ref.attend_bound(*part)).all())


def test_a_gradient_is_refused_not_dropped(gpu_device):
    a = adapters._inputs(gpu_device, 5, 64, 32, 8, 2)
    a["scaling"].requires_grad_()
    out = kernel.turing_int8_linear_adapters(**a)
    assert out.requires_grad
    with pytest.raises(RuntimeError):
        out.sum().backward()
    with torch.no_grad():
        assert torch.equal(out.detach(), kernel.turing_int8_linear_adapters(**a))
    q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 1, 1, 1, 64, 64, 64)
    index = torch.zeros(1, 1, 1, 1, dtype=torch.int32, device=gpu_device)
    out = turing_sage.key_block_attention(q8, qs, k8, ks, vt.requires_grad_(), index)
    assert out.requires_grad
    with pytest.raises(RuntimeError):
        out.sum().backward()


def test_tensors_without_data(gpu_device):
    from torch._subclasses.fake_tensor import FakeTensorMode

    a = adapters._inputs(gpu_device, 5, 64, 32, 8, 2)
    q8, qs, k8, ks, vt, g = attn._inputs(gpu_device, 1, 2, 1, 200, 300, 64)
    with FakeTensorMode() as mode:
        fake = {x: mode.from_tensor(v) if isinstance(v, torch.Tensor) else v for x, v in a.items()}
        assert kernel.turing_int8_linear_adapters(**fake).shape == (5, 32)
        q8, qs, k8, ks, vt = (mode.from_tensor(t) for t in (q8, qs, k8, ks, vt))
        index = turing_sage.select_key_blocks(q8, qs, k8, ks, keep=2)
        assert index.shape == (1, 2, 2, 2) and index.dtype == torch.int32
        assert turing_sage.key_block_attention(q8, qs, k8, ks, vt, index).shape == q8.shape


def test_both_routes_of_the_adapters(gpu_device):
    """Tensors the native route does not take (rows not contiguous) give the same bits."""
    for m, rank in ((3, 8), (61, 40), (700, 64)):
        a = adapters._inputs(gpu_device, m, 384, 200, rank, 4, residual=True, gate=True, seed=m)
        want = kernel.turing_int8_linear_adapters(**a)
        wide = torch.zeros(m, 384 + 16, dtype=torch.int8, device=gpu_device)
        wide[:, :384] = a["activation"]
        assert torch.equal(want, kernel.turing_int8_linear_adapters(**dict(a, activation=wide[:, :384])))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("blkq,blkk", [(16, 64), (32, 128), (128, 64)])
def test_scales_behind_the_end_are_not_seen(gpu_device, d, blkq, blkk):
    """Scale groups that begin at or behind a sample's end hold NaN and infinity."""
    dev = gpu_device
    g = torch.Generator().manual_seed(d + blkq)
    q8, qs = ref.codes(3, 2, 300, d, blkq, g, dev)
    k8, ks = ref.codes(3, 2, 700, d, blkk, g, dev)
    ql, kl = (torch.tensor(x, dtype=torch.int32, device=dev) for x in ([300, 131, 17], [700, 130, 65]))
    want = ref.select(q8, qs, k8, ks, 2, "HND", False, 0, 0, blkq, blkk, ql, kl)
    vt = torch.randn(3, 2, d, 704, generator=g).to(torch.bfloat16).to(dev)
    kw = dict(blkq=blkq, blkk=blkk, query_lengths=ql, key_lengths=kl)
    clean = turing_sage.key_block_attention(q8, qs, k8, ks, vt, want.to(dev), **kw)
    for scales, lengths, blk in ((qs, ql, blkq), (ks, kl, blkk)):
        first = torch.arange(scales.size(2), device=dev) * blk
        behind = (first >= lengths[:, None, None]).expand_as(scales)
        scales[behind] = torch.tensor([float("nan"), float("inf")], device=dev)[torch.arange(int(behind.sum()), device=dev) % 2]
    got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep=2, **kw)
    assert torch.equal(got.cpu(), want)
    out = turing_sage.key_block_attention(q8, qs, k8, ks, vt, got, **kw)
    assert torch.equal(out, clean) and torch.isfinite(out).all()
