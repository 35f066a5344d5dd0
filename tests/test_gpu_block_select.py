"""GPU: ``select_key_blocks`` picks exactly the blocks of the 64-bit reference
(tests/operator_reference.py): scale granularities, odd lengths, causal,
forced blocks, padded batches, ties, and more key blocks than LDS holds."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import turing_sage
from tests import operator_reference as ref

pytestmark = pytest.mark.gpu


def _check(dev, b, hq, hkv, lq, lk, d, keep, layout="HND", causal=False, sink=0, local=0, blkq=128, blkk=128,
           ql=None, kl=None, seed=0):
    print(f"[block select] B{b} H{hq}/{hkv} L{lq}/{lk} D{d} keep {keep} {layout} causal {causal}", flush=True)
    g = torch.Generator().manual_seed(seed)
    q8, qs = ref.codes(b, hq, lq, d, blkq, g, dev, layout)
    k8, ks = ref.codes(b, hkv, lk, d, blkk, g, dev, layout)
    ql, kl = (None if x is None else torch.tensor(x, dtype=torch.int32, device=dev) for x in (ql, kl))
    got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep=keep, tensor_layout=layout, is_causal=causal,
                                        sink_blocks=sink, local_blocks=local, blkq=blkq, blkk=blkk, query_lengths=ql,
                                        key_lengths=kl)
    want = ref.select(q8, qs, k8, ks, keep, layout, causal, sink, local, blkq, blkk, ql, kl)
    assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)
    return got


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("lq,lk,keep", [(1, 1, 1), (1, 65, 1), (129, 64, 3), (300, 1000, 5), (2100, 700, 4),
                                        (257, 4100, 64), (700, 700, 1000)])
def test_lengths(gpu_device, d, lq, lk, keep):
    _check(gpu_device, 1, 2, 2, lq, lk, d, keep, seed=lq + d)


@pytest.mark.parametrize("blkq,blkk", [(16, 64), (32, 128), (64, 64), (128, 128), (24, 64), (256, 128), (7, 64), (8, 64)])
@pytest.mark.parametrize("d", [64, 128])
def test_scale_granularities(gpu_device, blkq, blkk, d):
    _check(gpu_device, 2, 4, 2, 333, 517, d, 3, layout="NHD", blkq=blkq, blkk=blkk, seed=blkq)


@pytest.mark.parametrize("sink,local", [(0, 0), (1, 0), (0, 1), (2, 2), (5, 9), (1000, 0), (0, 1000)])
@pytest.mark.parametrize("causal", [False, True])
def test_forced_blocks(gpu_device, sink, local, causal):
    _check(gpu_device, 1, 4, 1, 1300, 1300, 128, 6, causal=causal, sink=sink, local=local, blkq=16, blkk=64, seed=3)


@pytest.mark.parametrize("causal", [False, True])
def test_padded_batch(gpu_device, causal):
    _check(gpu_device, 5, 2, 1, 500, 500, 64, 3, causal=causal, local=1, ql=[500, 129, 1, 0, 300],
           kl=[500, 129, 64, 300, 0], seed=5)


def test_lengths_outside_the_tensor_are_its_ends(gpu_device):
    _check(gpu_device, 2, 2, 2, 300, 300, 64, 3, ql=[-4, 9000], kl=[9000, 9000], seed=6)


def test_more_key_blocks_than_lds_holds(gpu_device):
    _check(gpu_device, 1, 1, 1, 140, 70000, 64, 300, seed=7)
    _check(gpu_device, 1, 1, 1, 140, 70000, 128, 3, causal=True, seed=8)
    _check(gpu_device, 1, 1, 1, 140, 65536, 64, 40, seed=9)
    _check(gpu_device, 1, 1, 1, 140, 131200, 64, 40, seed=10)


def test_near_scores(gpu_device):
    """Key blocks that differ by one code in 64 x 64: scores closer than 16 or 24 bits tell apart."""
    dev = gpu_device
    g = torch.Generator().manual_seed(11)
    for d, blocks, keep in ((64, 40, 13), (128, 300, 150), (64, 600, 5)):
        q8, qs = ref.codes(1, 1, 300, d, 128, g, dev)
        row = torch.randint(-120, 120, (1, 1, 64, d), generator=g, dtype=torch.int8)
        k8 = row.repeat(1, 1, blocks, 1)
        for j in range(blocks):
            k8[0, 0, 64 * j + j % 64, j % d] += int(torch.randint(-3, 4, (1,), generator=g))
        ks = torch.full((1, 1, blocks), 0.02, device=dev)
        got = turing_sage.select_key_blocks(q8, qs, k8.to(dev), ks, keep=keep, blkk=64)
        assert torch.equal(got.cpu(), ref.select(q8, qs, k8.to(dev), ks, keep, "HND", False, 0, 0, 128, 64))


@pytest.mark.parametrize("q_factor,k_factor", [(1e-25, 1.0), (1.0, 1e-30), (1e30, 1e25), (1e-36, 1e36), (1e25, 1e-25)])
def test_scales_at_the_ends_of_fp32(gpu_device, q_factor, k_factor):
    dev = gpu_device
    g = torch.Generator().manual_seed(12)
    q8, qs = ref.codes(1, 2, 260, 64, 128, g, dev)
    k8, ks = ref.codes(1, 2, 1000, 64, 64, g, dev)
    qs, ks = qs * q_factor, ks * k_factor
    got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep=6, blkk=64, local_blocks=1)
    assert torch.equal(got.cpu(), ref.select(q8, qs, k8, ks, 6, "HND", False, 0, 1, 128, 64))


def test_a_few_keys_far_larger_than_the_others(gpu_device):
    """The margin follows the longest mean: most blocks are then undecided."""
    dev = gpu_device
    g = torch.Generator().manual_seed(13)
    q8, qs = ref.codes(2, 2, 500, 128, 128, g, dev)
    k8, ks = ref.codes(2, 2, 6400, 128, 64, g, dev)
    ks[:, :, 7] *= 3e4
    for keep in (1, 40, 99):
        got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep=keep, blkk=64)
        assert torch.equal(got.cpu(), ref.select(q8, qs, k8, ks, keep, "HND", False, 0, 0, 128, 64))


def test_equal_scores_go_to_the_lower_block(gpu_device):
    dev = gpu_device
    q8 = torch.ones(1, 1, 128, 64, dtype=torch.int8, device=dev)
    k8 = torch.zeros(1, 1, 640, 64, dtype=torch.int8, device=dev)
    k8[:, :, 128:192] = 3
    k8[:, :, 384:448] = 3
    k8[:, :, 576:] = -1
    s = torch.full((1, 1, 10), 0.01, device=dev)
    for keep, want in ((1, [2]), (2, [2, 6]), (4, [0, 1, 2, 6]), (9, [0, 1, 2, 3, 4, 5, 6, 7, 8])):
        got = turing_sage.select_key_blocks(q8, s[..., :1].contiguous(), k8, s, keep=keep, blkk=64)
        assert got.flatten().tolist() == want


def test_scores_that_are_no_numbers_come_last(gpu_device):
    dev = gpu_device
    g = torch.Generator().manual_seed(1)
    q8, qs = ref.codes(1, 1, 128, 64, 128, g, dev)
    k8, ks = ref.codes(1, 1, 640, 64, 64, g, dev)
    ks[0, 0, 3] = float("nan")
    ks[0, 0, 0] = 0.0
    for keep in (1, 5, 9, 10):
        got = turing_sage.select_key_blocks(q8, qs, k8, ks, keep=keep, blkk=64)
        assert torch.equal(got.cpu(), ref.select(q8, qs, k8, ks, keep, "HND", False, 0, 0, 128, 64))


def test_strided_codes_and_another_stream(gpu_device):
    """Codes as views of wider rows (16-byte aligned and not), on a side stream."""
    dev = gpu_device
    g = torch.Generator().manual_seed(2)
    q8, qs = ref.codes(1, 2, 400, 64, 128, g, dev)
    k8, ks = ref.codes(1, 2, 400, 64, 128, g, dev)
    want = ref.select(q8, qs, k8, ks, 3, "HND", False, 0, 0, 128, 128)
    stream = torch.cuda.Stream(dev)
    for pad, first in ((16, 16), (9, 5)):
        wide = [torch.zeros(1, 2, 400, 64 + pad, dtype=torch.int8, device=dev) for _ in range(2)]
        views = [w[..., first:first + 64] for w in wide]
        for v, c in zip(views, (q8, k8)):
            v.copy_(c)
        torch.cuda.synchronize(dev)
        with torch.cuda.stream(stream):
            got = turing_sage.select_key_blocks(views[0], qs, views[1], ks, keep=3)
        stream.synchronize()
        assert torch.equal(got.cpu(), want)


def test_compiled_op(gpu_device):
    g = torch.Generator().manual_seed(3)
    q8, qs = ref.codes(1, 2, 300, 64, 128, g, gpu_device)
    k8, ks = ref.codes(1, 2, 300, 64, 128, g, gpu_device)
    got = torch.ops.turing_utils.sage_block_select(q8, qs, k8, ks, "HND", 2, False, 0, 1, 128, 128)
    assert torch.equal(got, turing_sage.select_key_blocks(q8, qs, k8, ks, keep=2, local_blocks=1))
