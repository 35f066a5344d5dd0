"""GPU: ``key_block_attention`` against the 64-bit reference of
tests/operator_reference.py, within the bound derived there: lengths, lists
that are empty, repeated, out of order or out of range, causal masks that
leave rows empty, padded batches with NaN behind the last key, split lists,
captured graphs, other streams."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import turing_sage
from tests import operator_reference as ref

pytestmark = pytest.mark.gpu


def _inputs(dev, b, hq, hkv, lq, lk, d, layout="HND", blkq=128, blkk=128, seed=0, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    q8, qs = ref.codes(b, hq, lq, d, blkq, g, dev, layout, spread)
    k8, ks = ref.codes(b, hkv, lk, d, blkk, g, dev, layout, spread)
    lpad = (lk + 63) // 64 * 64
    vt = torch.randn(b, hkv, d, lpad, generator=g) + torch.randn(b, hkv, d, 1, generator=g)
    vt[..., lk:] = 0
    return q8, qs, k8, ks, vt.to(torch.bfloat16).to(dev), g


def _random_lists(b, hq, lq, lk, width, g, dev):
    """Ascending lists of random length in [0, width]."""
    nqb, nkb = (lq + 127) // 128, (lk + 63) // 64
    rank = torch.rand(b, hq, nqb, nkb, generator=g).argsort(-1)[..., :width]
    count = torch.randint(0, width + 1, (b, hq, nqb, 1), generator=g)
    rank = torch.where(torch.arange(rank.size(-1)) < count, rank, nkb).sort(-1).values
    return torch.where(rank < nkb, rank, -1).to(torch.int32).to(dev)


def _check(args, index, layout="HND", causal=False, sm_scale=None, blkq=128, blkk=128, ql=None, kl=None):
    q8, qs, k8, ks, vt = args
    print(f"[block attn] Q{tuple(q8.shape)} K{tuple(k8.shape)} list {index.size(-1)} {layout} causal {causal}", flush=True)
    got = turing_sage.key_block_attention(q8, qs, k8, ks, vt, index, tensor_layout=layout, is_causal=causal,
                                          sm_scale=sm_scale, blkq=blkq, blkk=blkk, query_lengths=ql, key_lengths=kl)
    assert got.shape == q8.shape and got.dtype == torch.bfloat16
    clean = vt if kl is None else vt.masked_fill(
        torch.arange(vt.size(-1), device=vt.device) >= kl[:, None, None, None], 0)
    want, size = ref.attend(q8, qs, k8, ks, clean, index, layout, causal, sm_scale or q8.size(-1) ** -0.5, blkq, blkk,
                            ql, kl)
    off = (got.double() - want).abs()
    bound = ref.attend_bound(want, size)
    assert torch.isfinite(got).all() and bool((off <= bound).all()), float((off / bound.clamp_min(1e-30)).max())
    return got


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk,width", [(1, 1, 1), (1, 64, 1), (1, 700, 9), (33, 65, 2), (128, 128, 2), (129, 1000, 7),
                                         (513, 640, 10), (300, 4000, 40), (64, 20000, 300)])
def test_lengths(gpu_device, d, lq, lk, width):
    *args, g = _inputs(gpu_device, 1, 2, 1, lq, lk, d, seed=lq + lk + d)
    _check(args, _random_lists(1, 2, lq, lk, width, g, gpu_device))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("blkq,blkk", [(16, 64), (128, 128), (24, 256)])
def test_layouts_and_scales(gpu_device, d, layout, blkq, blkk):
    *args, g = _inputs(gpu_device, 2, 6, 2, 390, 520, d, layout, blkq, blkk, seed=d + blkq)
    _check(args, _random_lists(2, 6, 390, 520, 5, g, gpu_device), layout, blkq=blkq, blkk=blkk, sm_scale=0.3)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk", [(700, 700), (700, 300), (130, 900)])
def test_causal_with_rows_that_see_nothing(gpu_device, d, lq, lk):
    *args, g = _inputs(gpu_device, 1, 3, 3, lq, lk, d, seed=lk + d)
    index = _random_lists(1, 3, lq, lk, 4, g, gpu_device)
    index[:, 0] = -1
    index[:, 0, :, 0] = torch.arange(index.size(2)) * 2 + 1  # rows 128 i .. + 63 see no key of it
    got = _check(args, index, causal=True)
    assert (got[:, 0, :64] == 0).all()


def test_lists_that_repeat_fall_or_leave_the_range(gpu_device):
    *args, _ = _inputs(gpu_device, 1, 1, 1, 128, 640, 128, seed=9)
    for row in ([3, 3, 3], [5, 2, 7], [-1, -5, 4, -1, 4, 6, -1], [0, 10, 1], [2147483647, 1, 2], [-2147483648, 0, 9],
                [-1], [9, 10, 11], [1, -1, -1, -1, -1, -1, -1, -1, 2]):
        index = torch.tensor(row, dtype=torch.int32, device=gpu_device).view(1, 1, 1, -1)
        _check(args, index)


def test_empty_lists(gpu_device):
    *args, _ = _inputs(gpu_device, 2, 2, 2, 200, 300, 64, seed=10)
    for width in (0, 1, 300):
        index = torch.full((2, 2, 2, width), -1, dtype=torch.int32, device=gpu_device)
        assert (turing_sage.key_block_attention(*args, index) == 0).all()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_padded_batch_with_nan_behind_the_last_key(gpu_device, d, causal):
    b, lq, lk = 6, 400, 400
    q8, qs, k8, ks, vt, g = _inputs(gpu_device, b, 2, 1, lq, lk, d, seed=d)
    ql = torch.tensor([400, 131, 1, 0, 400, 257], dtype=torch.int32, device=gpu_device)
    kl = torch.tensor([400, 129, 1, 200, 0, 321], dtype=torch.int32, device=gpu_device)
    for i, n in enumerate(kl.tolist()):
        vt[i, ..., n:] = float("nan") if i % 2 else float("inf")
    index = _random_lists(b, 2, lq, lk, 7, g, gpu_device)
    index[2:] = torch.arange(7, device=gpu_device)
    _check((q8, qs, k8, ks, vt), index, causal=causal, ql=ql, kl=kl)


@pytest.mark.parametrize("lq,lk,width,causal", [(1, 20000, 312, False), (40, 9000, 141, False), (300, 9000, 64, True)])
def test_long_lists_of_few_rows_are_split(gpu_device, lq, lk, width, causal):
    from comfyui_turing_utils_kernel import _lib

    *args, g = _inputs(gpu_device, 1, 2, 1, lq, lk, 128, seed=width)
    assert _lib.load().tu_sage_block_attn_workspace(1, 2, lq, 128, width, 256) > 0
    index = _random_lists(1, 2, lq, lk, width, g, gpu_device)
    index[0, 0] = -1
    index[0, 0, :, width - 1] = 3  # every range but the last is empty
    _check(args, index, causal=causal)


def test_large_scores_and_zero_scales(gpu_device):
    q8, qs, k8, ks, vt, g = _inputs(gpu_device, 1, 2, 2, 256, 512, 128, blkk=64, seed=12, spread=6.0)
    index = _random_lists(1, 2, 256, 512, 6, g, gpu_device)
    _check((q8, qs, k8, ks, vt), index, blkk=64)
    ks[:, :, ::2] = 0.0
    qs[:, 1] = 0.0
    kl = torch.tensor([500], dtype=torch.int32, device=gpu_device)
    _check((q8, qs, k8, ks, vt), index, blkk=64, kl=kl)


def test_full_lists_equal_dense_attention(gpu_device):
    from comfyui_turing_utils_kernel.turing_sage import core

    *args, _ = _inputs(gpu_device, 1, 2, 2, 300, 500, 128, seed=13)
    index = torch.arange(8, dtype=torch.int32, device=gpu_device).expand(1, 2, 3, 8)
    for causal in (False, True):
        got = _check(args, index, causal=causal)
        dense = core.attention_from_vt(*args, is_causal=causal, kv_splits=1)
        want, size = ref.attend(*args, index, "HND", causal, 128 ** -0.5, 128, 128)
        assert ((dense.double() - got.double()).abs() <= 2 * ref.attend_bound(want, size)).all()


def test_run_twice_gives_the_same_bits_and_streams_do_not_mix(gpu_device):
    *args, g = _inputs(gpu_device, 1, 4, 2, 64, 9000, 128, seed=14)
    index = _random_lists(1, 4, 64, 9000, 100, g, gpu_device)
    first = turing_sage.key_block_attention(*args, index)
    other = torch.roll(index, 1, 1)
    second = turing_sage.key_block_attention(*args, other)
    streams = [torch.cuda.Stream(gpu_device) for _ in range(2)]
    torch.cuda.synchronize(gpu_device)
    outs = []
    for _ in range(4):
        for s, idx in zip(streams, (index, other)):
            with torch.cuda.stream(s):
                outs.append(turing_sage.key_block_attention(*args, idx))
    torch.cuda.synchronize(gpu_device)
    for i, o in enumerate(outs):
        assert torch.equal(o, (first, second)[i % 2]), i


def test_captured_selection_and_attention(gpu_device):
    """Selection and (split) attention in one graph, replayed on changing
    inputs with eager work between the replays."""
    dev = gpu_device
    q8, qs, k8, ks, vt, g = _inputs(dev, 1, 4, 2, 130, 5000, 128, seed=15)

    def step():
        index = turing_sage.select_key_blocks(q8, qs, k8, ks, keep=40, local_blocks=1)
        return turing_sage.key_block_attention(q8, qs, k8, ks, vt, index), index

    step()
    torch.cuda.synchronize(dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, index = step()
    for _ in range(3):
        k8.copy_(torch.randint(-127, 128, k8.shape, generator=g, dtype=torch.int8))
        graph.replay()
        want, want_index = step()
        torch.cuda.synchronize(dev)
        assert torch.equal(index, want_index) and torch.equal(out, want)


@pytest.mark.parametrize("head_dim,dtype", [(64, torch.bfloat16), (80, torch.float16), (128, torch.bfloat16)])
@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_one_call_form(gpu_device, head_dim, dtype, layout):
    """sparse_sageattn is its three parts, and keeping every block is sageattn
    within both kernels' bounds."""
    from comfyui_turing_utils_kernel.turing_sage import core

    g = torch.Generator().manual_seed(16)
    shape = (2, 4, 300, head_dim)
    q, k, v = (torch.randn(shape, generator=g).to(dtype).to(gpu_device) for _ in range(3))
    if layout == "NHD":
        q, k, v = (t.transpose(1, 2).contiguous() for t in (q, k, v))
    state = core.prequantize_sageattn(q, k, v, layout)
    qk = (state.query_int8, state.query_scale, state.key_int8, state.key_scale)
    got = turing_sage.sparse_sageattn(q, k, v, layout, keep=2, local_blocks=1)
    assert got.shape == q.shape and got.dtype == dtype
    index = turing_sage.select_key_blocks(*qk, keep=2, local_blocks=1, tensor_layout=layout)
    parts = turing_sage.key_block_attention(*qk, state.value_t, index, tensor_layout=layout, sm_scale=state.sm_scale)
    assert torch.equal(got, parts[..., :head_dim].to(dtype))
    full = turing_sage.sparse_sageattn(q, k, v, layout, keep=5)
    dense = turing_sage.sageattn(q, k, v, layout)
    everything = torch.arange(5, dtype=torch.int32, device=gpu_device).expand(2, 4, 3, 5)
    want, size = ref.attend(*qk, state.value_t, everything, layout, False, state.sm_scale, 128, 128)
    bound = 2 * ref.attend_bound(want, size)[..., :head_dim]
    # both were rounded to bf16, and to fp16 from there
    assert ((full.double() - dense.double()).abs() <= bound + 2.0 ** -10 * dense.double().abs()).all()
