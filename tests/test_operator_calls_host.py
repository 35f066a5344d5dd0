"""Calls of the adapters and of the Wan block that their documentation allows
and no ordinary program makes, on the host: strided arguments on the general
route, batches and contexts without rows.  CPU only."""
from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch

import comfyui_turing_utils_kernel as kernel
from comfyui_turing_utils_kernel import _lib, adapters, ops

COUNT, RANK, M, N, K = 5, 8, 5, 16, 16


def _adapter_args():
    g = torch.Generator().manual_seed(0)
    return dict(activation=torch.randint(-127, 128, (M, K), generator=g, dtype=torch.int8),
                weight=torch.randint(-127, 128, (N, K), generator=g, dtype=torch.int8),
                activation_scale=torch.rand(M, generator=g), weight_scale=torch.rand(N, generator=g), bias=None,
                down=torch.randn(COUNT, RANK, K, generator=g).to(torch.bfloat16),
                up=torch.randn(COUNT, N, RANK, generator=g).to(torch.bfloat16),
                scaling=torch.rand(COUNT, generator=g), adapter_ids=torch.arange(M, dtype=torch.int32).flip(0))


@pytest.fixture
def entry_point(monkeypatch):
    """The general route on CPU tensors; what stands behind `scaling` and `ids`
    when the entry point is called."""
    seen = {}

    def call(name, *args):
        assert name == "tu_int8_gemm_adapters"
        seen["scaling"] = list((ctypes.c_float * COUNT).from_address(args[7]))
        seen["ids"] = list((ctypes.c_int32 * M).from_address(args[8]))

    monkeypatch.setattr(ops, "_require_device", lambda *a: None)
    monkeypatch.setattr(adapters, "_compute_units", lambda device: 256)
    monkeypatch.setattr(_lib, "call", call)
    monkeypatch.setattr(_lib, "stream_of", lambda device: None)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    return seen


@pytest.mark.parametrize("strided", [("scaling",), ("adapter_ids",), ("scaling", "adapter_ids")])
def test_strided_scaling_and_ids_live_until_the_launch(entry_point, strided):
    """Columns of a table: the copies that the kernel reads are not freed, and
    their memory is not taken again, before the entry point has been called."""
    a = _adapter_args()
    want = a["scaling"].tolist(), a["adapter_ids"].tolist()
    for x in strided:
        table = torch.zeros(a[x].numel(), 3, dtype=a[x].dtype)
        table[:, 1] = a[x]
        a[x] = table[:, 1]
        assert not a[x].is_contiguous()
    for _ in range(20):  # (whether freed memory is taken again at once is the allocator's choice)
        kernel.turing_int8_linear_adapters(**a)
        assert (entry_point["scaling"], entry_point["ids"]) == want


def _block(adapted):
    """A Wan block without data; with adapters of every linear."""
    from comfyui_turing_utils_kernel.wan_block import W8A8Linear, WanBlockConfig, WanBlockW8A8

    def lin(n, k):
        return W8A8Linear(torch.zeros(n, k, dtype=torch.int8, device="meta"), torch.ones(n, device="meta"), None)

    ones = torch.ones(256, device="meta")
    block = WanBlockW8A8(WanBlockConfig(dim=256, heads=2, ffn_dim=512, text_dim=256),
                         modulation=torch.zeros(1, 6, 256, device="meta"), self_qkv=lin(768, 256),
                         self_o=lin(256, 256), self_norm_q=ones, self_norm_k=ones, norm3_weight=ones,
                         norm3_bias=ones * 0, cross_q=lin(256, 256), cross_kv=lin(512, 256), cross_o=lin(256, 256),
                         cross_norm_q=ones, cross_norm_k=ones, ffn_up=lin(512, 256), ffn_down=lin(256, 512))
    block.set_adapters({name: kernel.LinearAdapters(
        torch.zeros(2, 8, getattr(block, name).in_features, dtype=torch.bfloat16, device="meta"),
        torch.zeros(2, getattr(block, name).out_features, 8, dtype=torch.bfloat16, device="meta"),
        torch.ones(2, device="meta")) for name in (block.LINEARS if adapted else ())})
    return block


@pytest.mark.parametrize("b,l", [(0, 5), (2, 0), (0, 0), (2, 5)])
@pytest.mark.parametrize("with_ids", [False, True])
def test_sublayers_without_rows(b, l, with_ids):
    """An empty batch, or samples without rows, with or without adapters."""
    block = _block(with_ids)
    h = torch.empty(b, l, 256, dtype=torch.bfloat16, device="meta")
    ids = torch.zeros(b, dtype=torch.int32, device="meta") if with_ids else None
    gate = torch.empty(b, 1, 256, dtype=torch.bfloat16, device="meta")
    assert block.ffn(h, adapter_ids=ids).shape == (b, l, 256)
    if l:  # (a gate has a row for each of the output's)
        assert block.ffn(h, residual=h, gate=gate, adapter_ids=ids).shape == (b, l, 256)
    assert block._project("self_o", h.reshape(b * l, 256), b, h, None, ids).shape == (b * l, 256)
