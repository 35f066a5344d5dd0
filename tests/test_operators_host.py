"""Host side of the block-sparse attention and the adapters: fake-tensor
contracts, refusals before any launch, workspace sizes, the adapters' rotation
and layout, and the 64-bit reference the GPU tests use.  CPU only."""
from __future__ import annotations

import numpy as np
import pytest
import torch

import comfyui_turing_utils_kernel as kernel
from comfyui_turing_utils_kernel import _lib, turing_sage
from comfyui_turing_utils_kernel.adapters import _rotation
from oracle import oracle
from tests import operator_reference as ref

META = "meta"


def _qk(device=META, b=2, hq=4, hkv=2, lq=300, lk=500, d=64, blkq=128, blkk=128):
    return (torch.empty((b, hq, lq, d), dtype=torch.int8, device=device),
            torch.empty((b, hq, (lq + blkq - 1) // blkq), device=device),
            torch.empty((b, hkv, lk, d), dtype=torch.int8, device=device),
            torch.empty((b, hkv, (lk + blkk - 1) // blkk), device=device))


def _adapter_args(device=META, m=7, k=128, n=64, rank=16, count=3, rows=1):
    def e(*shape, dtype=torch.float32):
        return torch.zeros(shape, dtype=dtype, device=device)

    return dict(activation=e(m, k, dtype=torch.int8), weight=e(n, k, dtype=torch.int8), activation_scale=e(m),
                weight_scale=e(n), bias=None, down=e(count, rank, k, dtype=torch.bfloat16),
                up=e(count, n, rank, dtype=torch.bfloat16), scaling=e(count),
                adapter_ids=e((m + rows - 1) // rows, dtype=torch.int32), adapter_rows=rows)


def test_fake_contracts_and_fullgraph_leaves():
    qk = _qk()
    index = turing_sage.select_key_blocks(*qk, keep=3)
    assert index.shape == (2, 4, 3, 3) and index.dtype == torch.int32 and index.device.type == META
    assert turing_sage.select_key_blocks(*qk, keep=99).shape == (2, 4, 3, 8)
    vt = torch.empty((2, 2, 64, 512), dtype=torch.bfloat16, device=META)
    out = turing_sage.key_block_attention(*qk, vt, index)
    assert out.shape == (2, 4, 300, 64) and out.dtype == torch.bfloat16
    y = kernel.turing_int8_linear_adapters(**_adapter_args())
    assert y.shape == (7, 64) and y.dtype == torch.bfloat16

    def chain(q, qs, k, ks, v, a):
        idx = turing_sage.select_key_blocks(q, qs, k, ks, keep=2, local_blocks=1)
        return turing_sage.key_block_attention(q, qs, k, ks, v, idx), kernel.turing_int8_linear_adapters(**a)

    o, y = torch.compile(chain, backend="eager", fullgraph=True)(*qk, vt, _adapter_args())
    assert o.shape == (2, 4, 300, 64) and y.shape == (7, 64)


def test_cpu_tensors_are_refused():
    qk = tuple(torch.zeros_like(t, device="cpu") for t in _qk())
    index = torch.zeros((2, 4, 3, 1), dtype=torch.int32)
    vt = torch.zeros((2, 2, 64, 512), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="CUDA|HIP"):
        turing_sage.select_key_blocks(*qk, keep=1)
    with pytest.raises(RuntimeError, match="CUDA|HIP"):
        turing_sage.key_block_attention(*qk, vt, index)
    with pytest.raises(RuntimeError, match="CUDA|HIP"):
        kernel.turing_int8_linear_adapters(**_adapter_args("cpu"))
    with pytest.raises(ValueError, match="CUDA"):
        q = torch.zeros((1, 2, 64, 64), dtype=torch.bfloat16)
        turing_sage.sparse_sageattn(q, q, q, keep=1)


@pytest.mark.parametrize("change,match", [
    (dict(keep=0), "keep"), (dict(keep=1, sink_blocks=-1), "sink"), (dict(keep=1, local_blocks=-1), "local"),
    (dict(keep=1, blkk=96), "blkk"), (dict(keep=1, blkq=64), "scale shape"), (dict(keep=1, tensor_layout="BLHD"), "layout"),
])
def test_selection_refusals(change, match):
    with pytest.raises(Exception, match=match):
        turing_sage.select_key_blocks(*_qk(), **change)


def test_attention_refusals():
    qk = _qk()
    vt = torch.empty((2, 2, 64, 512), dtype=torch.bfloat16, device=META)
    index = torch.empty((2, 4, 3, 2), dtype=torch.int32, device=META)
    for bad in (vt[..., :500], vt.float(), vt[:, :1]):
        with pytest.raises(Exception, match="V\\^T"):
            turing_sage.key_block_attention(*qk, bad, index)
    for bad in (index.long(), index[:, :, :2], index[:, :2], index[0]):
        with pytest.raises(Exception, match="block_index"):
            turing_sage.key_block_attention(*qk, vt, bad)
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="sm_scale"):
            turing_sage.key_block_attention(*qk, vt, index, sm_scale=scale)
    scales = torch.empty((2, 2, 3), device=META)
    with pytest.raises(Exception, match="blkk"):
        turing_sage.key_block_attention(*qk[:3], scales, vt, index, blkk=192)


@pytest.mark.parametrize("change,match", [
    (lambda a: a.update(down=a["down"].float()), "bfloat16"),
    (lambda a: a.update(down=a["down"][:, :12], up=a["up"][..., :12]), "multiple of 8"),
    (lambda a: a.update(down=a["down"][..., :64]), "adapters must be"),
    (lambda a: a.update(up=a["up"][:2]), "adapters must be"),
    (lambda a: a.update(scaling=a["scaling"][:1]), "scaling"),
    (lambda a: a.update(adapter_ids=a["adapter_ids"].long()), "int32"),
    (lambda a: a.update(adapter_ids=a["adapter_ids"][:3]), "adapter_ids"),
    (lambda a: a.update(adapter_rows=0), "adapter_ids"),
    (lambda a: a.update(parts=0), "parts"),
    (lambda a: a.update(parts=3), "parts"),
    (lambda a: a.update(parts=2), "adapters must be"),
    (lambda a: a.update(residual=torch.zeros(3, 64, dtype=torch.bfloat16, device=META)), "residual"),
])
def test_adapter_refusals(change, match):
    args = _adapter_args()
    change(args)
    with pytest.raises(Exception, match=match):
        kernel.turing_int8_linear_adapters(**args)


def test_entry_points_refuse_before_any_launch():
    lib = _lib.load()

    def error(name, *args):
        assert getattr(lib, name)(*args) != 0
        return lib.tu_last_error().decode()

    p = 1 << 20  # never read: every call below is refused on the host
    select = [p, p, 128, p, p, 128, 1, 2, 1, 300, 300, 64, 64, 64, 64, 64, 64, 64, None, None, 2, 0, 0, 0, p, 1 << 30, p, None]
    for at, value, word in ((11, 96, "head_dim"), (8, 3, "multiple"), (9, 0, "lengths"), (20, 0, "keep"), (0, p + 8, "aligned"),
                            (25, 16, "workspace"), (24, p + 8, "workspace"), (0, None, "non-null"), (7, 70000, "grid")):
        assert word in error("tu_sage_block_select", *(value if i == at else x for i, x in enumerate(select))), at
    attn = [p, p, 128, p, p, 128, p, 320, p, 4, p, 1, 2, 1, 300, 300, 64] + [64] * 9 + [None, None, 0.1, 0, 256, None, 0, None]
    for at, value, word in ((16, 32, "head_dim"), (13, 3, "multiple"), (7, 300, "padded"), (5, 192, "blkk"), (28, 0.0, "sm_scale"),
                            (9, 0, "sizes"), (8, None, "non-null"), (30, 0, "sizes"), (31, p + 4, "workspace"), (12, 70000, "grid")):
        assert word in error("tu_sage_block_attn", *(value if i == at else x for i, x in enumerate(attn))), at
    lora = [p, p, p, p, None, p, p, p, p, 1, 16, 2, 1, None, None, 1, p, 64, 128, 256, 256, p, 1 << 30, None]
    for at, value, word in ((10, 12, "rank"), (10, 0, "rank"), (11, 0, "count"), (9, 0, "rows"), (5, p + 8, "aligned"),
                            (19, 24, "K%16"), (6, None, "non-null"), (14, p, "gate"), (22, 8, "workspace"), (21, None, "workspace"),
                            (12, 0, "parts"), (12, 4, "parts"), (12, 3, "parts")):
        assert word in error("tu_int8_gemm_adapters", *(value if i == at else x for i, x in enumerate(lora))), at


def test_workspaces():
    lib = _lib.load()
    # 3 query and 8 key blocks a head: mean rows in fp64, as two bf16 terms of 16 blocks each, their lengths
    assert lib.tu_sage_block_select_workspace(2, 4, 2, 300, 500, 64) == 2 * 28 * (64 * 8 + 4) + 2 * 6 * 16 * 64 * 4
    # past 2048 key blocks the scores too
    assert (lib.tu_sage_block_select_workspace(1, 1, 1, 128, 131200, 64)
            == 2051 * 64 * 8 + 2052 * 4 + (16 + 2064) * 64 * 4 + 2050 * 8)
    # many query blocks: no list is split; one row: lists in ranges of at least four
    assert lib.tu_sage_block_attn_workspace(1, 40, 32760, 128, 128, 256) == 0
    assert lib.tu_sage_block_attn_workspace(1, 1, 1, 128, 3, 256) == 0
    assert lib.tu_sage_block_attn_workspace(4, 16, 1, 128, 32, 256) > 0
    # two bf16 terms a row and rank
    assert lib.tu_int8_gemm_adapters_workspace(61, 24) == 64 * 32 * 4  # whole fragments of 16 rows and 32 ranks


@pytest.mark.parametrize("group", [128, 256])
def test_rotation_is_the_quantizers(group):
    m = _rotation(group, "cpu").numpy()
    np.testing.assert_allclose(m, m.T, atol=0)
    np.testing.assert_allclose(m @ m, np.eye(group), atol=1e-12)
    rows = np.random.default_rng(0).standard_normal((3, group)).astype(np.float32)
    want = np.stack([oracle.rotate_group(r, group) for r in rows])
    np.testing.assert_allclose(rows.astype(np.float64) @ m, want, rtol=0, atol=2e-5)


def test_adapter_layout():
    g = torch.Generator().manual_seed(0)
    pairs = [(torch.randn(r, 256, generator=g), torch.randn(40, r, generator=g), s) for r, s in ((3, 0.5), (9, 2.0))]
    bank = kernel.LinearAdapters.from_float(pairs, 128)
    assert bank.down.shape == (2, 16, 256) and bank.up.shape == (2, 40, 16) and bank.scaling.tolist() == [0.5, 2.0]
    assert (bank.down[0, 3:] == 0).all() and (bank.up[0, :, 3:] == 0).all() and bank.down[1, 8].any()
    back = bank.down[1, :9].double().view(9, 2, 128) @ _rotation(128, "cpu")
    # a row's bf16 rounding, rotated back, keeps its length
    assert ((back.view(9, 256) - pairs[1][0].double()).norm(dim=1) <= ref.BF16 * pairs[1][0].double().norm(dim=1)).all()
    other = kernel.LinearAdapters.from_float([(a[:2], torch.randn(8, 2, generator=g), s) for a, _, s in pairs], 128)
    both = kernel.LinearAdapters.concat([bank, other])
    assert both.down.shape == (2, 24, 256) and both.up.shape == (2, 48, 24)
    assert torch.equal(both.up[:, :40, :16], bank.up) and torch.equal(both.up[:, 40:, 16:], other.up)
    assert (both.up[:, :40, 16:] == 0).all() and (both.up[:, 40:, :16] == 0).all()
    same = kernel.LinearAdapters.from_float([(a[:2], torch.randn(48, 2, generator=g), s) for a, _, s in pairs], 128)
    wide = kernel.LinearAdapters.from_float([(a, torch.randn(48, a.shape[0], generator=g), s) for a, _, s in pairs], 128)
    three = kernel.LinearAdapters.concat([same, wide, same])
    assert three.parts == 3 and three.rank == 48 and three.up.shape == (2, 144, 16)
    assert torch.equal(three.down[:, 16:32], wide.down) and torch.equal(three.up[:, 48:96], wide.up)
    for at in (0, 1):
        assert torch.equal(three.down[:, 32 * at:32 * at + 8], same.down) and (three.down[:, 32 * at + 8:32 * at + 16] == 0).all()
        assert torch.equal(three.up[:, 96 * at:96 * at + 48, :8], same.up) and (three.up[:, 96 * at:96 * at + 48, 8:] == 0).all()
    with pytest.raises(ValueError, match="again"):
        kernel.LinearAdapters.concat([three, three])
    for bad, match in (([], "at least one"), ([(torch.zeros(2, 200), torch.zeros(8, 2), 1.0)], "divide"),
                       ([(torch.zeros(2, 128), torch.zeros(8, 3), 1.0)], "each adapter")):
        with pytest.raises(ValueError, match=match):
            kernel.LinearAdapters.from_float(bad, 128)
    with pytest.raises(ValueError, match="scalings"):
        kernel.LinearAdapters.concat([bank, kernel.LinearAdapters(bank.down, bank.up, bank.scaling * 2)])
    with pytest.raises(ValueError, match="group"):
        kernel.LinearAdapters(bank.down, bank.up, bank.scaling, 64)


def test_reference_attention_is_masked_softmax():
    """The reference's block lists against a dense masked softmax."""
    g = torch.Generator().manual_seed(4)
    q8, qs = ref.codes(1, 2, 200, 64, 128, g, "cpu")
    k8, ks = ref.codes(1, 1, 300, 64, 128, g, "cpu")
    vt = torch.randn(1, 1, 64, 320, generator=g).to(torch.bfloat16)
    index = torch.tensor([[[[0, 2, -1], [4, 4, 1]], [[3, -1, 4], [-1, -1, -1]]]], dtype=torch.int32)
    kl = torch.tensor([290], dtype=torch.int32)
    out, size = ref.attend(q8, qs, k8, ks, vt, index, "HND", True, 0.125, 128, 128, None, kl)
    s = (q8.double() * qs.double().repeat_interleave(128, 2)[..., :200, None]) @ (
        k8.double() * ks.double().repeat_interleave(128, 2)[..., :300, None]).transpose(-1, -2) * 0.125
    mask = torch.zeros(1, 2, 200, 300, dtype=torch.bool)
    for h, n, blocks in ((0, 0, (0, 2)), (0, 1, (4,)), (1, 0, (3, 4))):
        for e in blocks:
            mask[0, h, n * 128:(n + 1) * 128, e * 64:(e + 1) * 64] = True
    mask &= torch.arange(300) <= torch.arange(200)[:, None]
    mask &= torch.arange(300) < 290
    p = torch.nan_to_num(s.masked_fill(~mask, -float("inf")).softmax(-1))
    want = p @ vt[0, 0, :, :300].double().t()
    assert torch.allclose(out, want, rtol=1e-12, atol=1e-12) and (size >= out.abs() - 1e-12).all()


def _block():
    from comfyui_turing_utils_kernel.wan_block import W8A8Linear, WanBlockConfig, WanBlockW8A8

    def lin(n, k):
        return W8A8Linear(torch.zeros(n, k, dtype=torch.int8), torch.ones(n), None)

    ones = torch.ones(256)
    return WanBlockW8A8(WanBlockConfig(dim=256, heads=2, ffn_dim=512, text_dim=256), modulation=torch.zeros(1, 6, 256),
                        self_qkv=lin(768, 256), self_o=lin(256, 256), self_norm_q=ones, self_norm_k=ones,
                        norm3_weight=ones, norm3_bias=ones * 0, cross_q=lin(256, 256), cross_kv=lin(512, 256),
                        cross_o=lin(256, 256), cross_norm_q=ones, cross_norm_k=ones, ffn_up=lin(512, 256),
                        ffn_down=lin(256, 512))


def test_block_adapters_are_checked():
    from comfyui_turing_utils_kernel import LinearAdapters

    def adapters(n, k, count=2, group=128):
        return LinearAdapters.from_float([(torch.ones(4, k), torch.ones(n, 4), 1.0)] * count, group)

    block = _block()
    block.set_adapters({"self_qkv": adapters(768, 256), "ffn_down": adapters(256, 512)})
    assert set(block.adapters) == {"self_qkv", "ffn_down"}
    for bad, match in (({"qkv": adapters(768, 256)}, "no linear"), ({"self_o": adapters(512, 256)}, "do not fit"),
                       ({"self_o": adapters(256, 256, group=256)}, "do not fit"),
                       ({"self_o": adapters(256, 256), "ffn_up": adapters(512, 256, 3)}, "one count")):
        with pytest.raises(ValueError, match=match):
            block.set_adapters(bad)
    assert set(block.adapters) == {"self_qkv", "ffn_down"}  # a refused mapping changes nothing

    x = torch.zeros(2, 8, 256, dtype=torch.bfloat16)
    args = (x, torch.zeros(2, 6, 256), x, None)
    for ids in (torch.zeros(3, dtype=torch.int32), torch.zeros(2, dtype=torch.int64), torch.zeros(1, 2, dtype=torch.int32)):
        with pytest.raises(ValueError, match="adapter_ids must be"):
            block(*args, adapter_ids=ids)
    block.set_adapters({})
    with pytest.raises(ValueError, match="need adapters"):
        block(*args, adapter_ids=torch.zeros(2, dtype=torch.int32))


def test_linear_adapters_are_checked():
    from comfyui_turing_utils_kernel import LinearAdapters
    from comfyui_turing_utils_kernel.wan_block import QuantizedActivation, W8A8Linear

    lin = W8A8Linear(torch.zeros(64, 256, dtype=torch.int8), torch.ones(64), None)
    x = QuantizedActivation(torch.zeros(8, 256, dtype=torch.int8), torch.ones(8, 1), 1, 8, 128)
    one = [(torch.ones(4, 256), torch.ones(64, 4), 1.0)]
    ids = torch.zeros(8, dtype=torch.int32)
    with pytest.raises(ValueError, match="need adapter_ids"):
        lin(x, adapters=LinearAdapters.from_float(one))
    with pytest.raises(ValueError, match="need adapters"):
        lin(x, adapter_ids=ids)
    with pytest.raises(ValueError, match="group 256"):
        lin(x, adapters=LinearAdapters.from_float(one, 256), adapter_ids=ids)
