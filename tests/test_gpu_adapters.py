"""GPU: ``turing_int8_linear_adapters`` against the 64-bit reference of
tests/operator_reference.py within the bound derived there, and rows without
an adapter bit for bit against int8_linear / int8_linear_residual."""
from __future__ import annotations

import pytest
import torch

import comfyui_turing_utils_kernel as kernel
from tests import operator_reference as ref

pytestmark = pytest.mark.gpu


def _inputs(dev, m, k, n, rank, count, rows=1, bias=True, residual=False, gate=False, seed=0, ids=None):
    g = torch.Generator().manual_seed(seed)
    groups = (m + rows - 1) // rows
    a = {
        "activation": torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8),
        "weight": torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8),
        "activation_scale": 0.01 + 0.02 * torch.rand(m, 1, generator=g),
        "weight_scale": (0.5 + torch.rand(n, generator=g)) * 1e-3,
        "bias": torch.randn(n, generator=g) if bias else None,
        "down": (torch.randn(count, rank, k, generator=g) * k ** -0.5).to(torch.bfloat16),
        "up": (torch.randn(count, n, rank, generator=g) * 0.3).to(torch.bfloat16),
        "scaling": 0.5 + torch.rand(count, generator=g),
        "adapter_ids": torch.randint(-1, count, (groups,), generator=g, dtype=torch.int32) if ids is None
        else torch.tensor(ids, dtype=torch.int32),
        "adapter_rows": rows,
    }
    if residual:
        a["residual"] = torch.randn(m, n, generator=g).to(torch.bfloat16)
        if gate:
            a["gate"] = torch.randn(groups, n, generator=g).to(torch.bfloat16)
            a["gate_rows"] = rows
    return {x: v.to(dev) if isinstance(v, torch.Tensor) else v for x, v in a.items()}


def _plain(a):
    """The projection without adapters."""
    args = [a[x] for x in ("activation", "weight", "activation_scale", "weight_scale", "bias")]
    if a.get("residual") is None:
        return torch.ops.turing_utils.int8_linear(*args)
    return torch.ops.turing_utils.int8_linear_residual(*args, a["residual"], a.get("gate"), a.get("gate_rows", 1))


def _dense(up, parts):
    """``up`` with zeros where a part's columns do not see a rank."""
    count, n, rank = up.shape
    out = torch.zeros(count, parts, n // parts, parts, rank, dtype=up.dtype, device=up.device)
    for p in range(parts):
        out[:, p, :, p] = up.view(count, parts, n // parts, rank)[:, p]
    return out.view(count, n, parts * rank)


def _check(a):
    m, k = a["activation"].shape
    print(f"[adapters] M{m} K{k} N{a['weight'].shape[0]} rank {a['down'].shape[1]} count {a['down'].shape[0]} "
          f"rows {a['adapter_rows']}", flush=True)
    got = kernel.turing_int8_linear_adapters(**a)
    want, bound = ref.linear(a["activation"], a["weight"], a["activation_scale"], a["weight_scale"], a["bias"], a["down"],
                             _dense(a["up"], a.get("parts", 1)), a["scaling"], a["adapter_ids"], a["adapter_rows"], a.get("residual"),
                             a.get("gate"), a.get("gate_rows", 1))
    off = (got.double() - want).abs()
    assert got.dtype == torch.bfloat16 and bool((off <= bound).all()), float((off / bound).max())
    ids = a["adapter_ids"].repeat_interleave(a["adapter_rows"])[:m]
    none = (ids < 0) | (ids >= a["down"].shape[0])
    assert torch.equal(got[none].view(torch.int16), _plain(a)[none].view(torch.int16))
    return got


@pytest.mark.parametrize("m,k,n,rank,count", [
    (1, 16, 8, 8, 1), (1, 1536, 9216, 16, 1), (4, 1536, 256, 16, 4), (17, 48, 72, 24, 3), (61, 640, 520, 40, 7),
    (33, 5120, 264, 8, 33), (130, 2064, 128, 136, 2), (300, 208, 136, 64, 5), (64, 1024, 64, 32, 200)])
def test_shapes(gpu_device, m, k, n, rank, count):
    _check(_inputs(gpu_device, m, k, n, rank, count, seed=m + k))


@pytest.mark.parametrize("m,n", [(1, 9216), (4096, 256), (512, 5120), (1024, 1536), (1024, 8960), (2050, 2048),
                                 (4100, 5120), (512, 10240)])
@pytest.mark.parametrize("residual", [False, True])
def test_every_tile(gpu_device, m, n, residual):
    """Sizes at which the GEMM takes each of its tiles."""
    rows = max(1, m // 3 + 5)
    _check(_inputs(gpu_device, m, 256, n, 32, 3, rows, residual=residual, gate=residual, seed=n))


@pytest.mark.parametrize("rank", [8, 16, 32])
def test_many_rows(gpu_device, rank):
    """The tall tile of the down-projection, borders inside it."""
    _check(_inputs(gpu_device, 33001, 160, 64, rank, 5, 37, seed=rank))


@pytest.mark.parametrize("m,count,rank,rows,k", [
    (256, 8, 8, 1, 160), (255, 8, 8, 1, 160), (300, 5, 40, 1, 160), (257, 40, 16, 2, 160), (1000, 300, 24, 1, 160),
    (1000, 1024, 8, 1, 160), (1000, 1025, 8, 1, 160), (5001, 33, 72, 1, 160), (9000, 4, 64, 1, 2560), (9000, 4, 64, 1, 160)])
def test_many_rows_of_many_requests(gpu_device, m, count, rank, rows, k):
    """Rows that are sorted by their adapter first, and sizes just past that."""
    a = _inputs(gpu_device, m, k, 72, rank, count, rows, seed=m + count)
    got = _check(a)
    assert torch.equal(got, kernel.turing_int8_linear_adapters(**a))
    # one adapter has nearly all rows, most have none
    a["adapter_ids"][: 9 * a["adapter_ids"].numel() // 10] = count - 1
    _check(a)
    a["adapter_ids"].fill_(-1)
    assert torch.equal(_check(a), _plain(a))


@pytest.mark.parametrize("m,n,rank,parts", [
    (1, 32, 16, 2), (5, 144, 24, 3), (61, 240, 120, 3), (130, 96, 24, 3), (4096, 256, 64, 2), (512, 4800, 96, 3),
    (1024, 1584, 192, 3), (1024, 8976, 96, 3), (2050, 2064, 120, 3), (4100, 4800, 192, 3), (4100, 4800, 96, 3),
    (512, 10176, 240, 3), (4100, 5120, 128, 2)])
@pytest.mark.parametrize("rows", [1, 1000])
def test_parts(gpu_device, m, n, rank, parts, rows):
    """Columns that see their own ranks, with borders of parts inside a wave's columns; every tile."""
    a = _inputs(gpu_device, m, 256, n, rank, 3, rows, seed=n + rank, residual=rows > 1)
    a["up"], a["parts"] = a["up"][..., :rank // parts].contiguous(), parts
    got = _check(a)
    assert torch.equal(got, torch.ops.turing_utils.int8_linear_adapters(**a))


def test_sizes_reach_every_tile(gpu_device):
    from comfyui_turing_utils_kernel import _lib

    cus = torch.cuda.get_device_properties(gpu_device).multi_processor_count
    sizes = [(1, 9216), (4096, 256), (512, 5120), (1024, 1536), (1024, 8960), (2050, 2048), (4100, 5120), (512, 10240)]
    tiles = {_lib.load().tu_int8_gemm_tile(m, n, 256, cus) for m, n in sizes}
    print([(t >> 16, t & 0xffff) for t in sorted(tiles)])
    assert len(tiles) >= 4


@pytest.mark.parametrize("residual,gate,bias", [(True, False, True), (True, True, False), (False, False, False)])
@pytest.mark.parametrize("rows", [1, 7, 100])
def test_residual_gate_and_bias(gpu_device, residual, gate, bias, rows):
    _check(_inputs(gpu_device, 203, 384, 200, 16, 3, rows, bias, residual, gate, seed=rows))


def test_requests_of_unequal_rows(gpu_device):
    ids = [0] * 1 + [3] * 40 + [-1] * 5 + [1] * 200 + [3] * 3 + [2] * 60 + [7] * 9 + [-9] * 2
    _check(_inputs(gpu_device, len(ids), 640, 384, 48, 4, ids=ids, seed=1))


def test_alternating_rows(gpu_device):
    _check(_inputs(gpu_device, 300, 512, 256, 32, 2, ids=[i % 2 for i in range(300)], seed=2))


def test_all_without_an_adapter(gpu_device):
    a = _inputs(gpu_device, 70, 512, 256, 32, 2, ids=[-1, 2] * 35, seed=3)
    assert torch.equal(_check(a), _plain(a))


def test_weights_of_another_request_do_not_leak(gpu_device):
    """Infinite and NaN weights of one adapter stay with its own rows."""
    a = _inputs(gpu_device, 90, 512, 256, 32, 3, ids=[0, 1, 2] * 30, seed=4)
    clean = kernel.turing_int8_linear_adapters(**a)
    a["down"][1] = float("nan")
    a["up"][2, 5] = float("inf")
    got = kernel.turing_int8_linear_adapters(**a)
    assert torch.equal(got[0::3], clean[0::3])
    assert torch.isnan(got[1::3]).all()
    keep = [c for c in range(256) if c != 5]
    assert torch.equal(got[2::3, keep], clean[2::3, keep]) and not torch.isfinite(got[2::3, 5]).any()


def test_residual_in_place_of_nothing_and_strided_inputs(gpu_device):
    a = _inputs(gpu_device, 50, 256, 128, 16, 2, seed=5, residual=True)
    want = kernel.turing_int8_linear_adapters(**a)
    b = dict(a)
    for x in ("activation", "weight", "down", "up", "residual"):
        t = a[x]
        wide = torch.zeros(*t.shape[:-1], t.shape[-1] + 3, dtype=t.dtype, device=gpu_device)
        wide[..., 1:-2] = t
        b[x] = wide[..., 1:-2]
    flat = torch.empty(a["down"].numel() + 1, dtype=torch.bfloat16, device=gpu_device)
    b["down"] = flat[1:].view_as(a["down"]).copy_(a["down"])  # not on 16 bytes
    assert torch.equal(kernel.turing_int8_linear_adapters(**b), want)


def test_no_rows(gpu_device):
    a = _inputs(gpu_device, 0, 256, 128, 16, 2)
    assert kernel.turing_int8_linear_adapters(**a).shape == (0, 128)


def test_captured_and_on_two_streams(gpu_device):
    dev = gpu_device
    a = _inputs(dev, 40, 2048, 512, 24, 5, seed=6)
    b = _inputs(dev, 40, 2048, 512, 24, 5, seed=7)
    want = [kernel.turing_int8_linear_adapters(**x) for x in (a, b)]
    torch.cuda.synchronize(dev)
    graphs, outs = [], []
    for x in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(kernel.turing_int8_linear_adapters(**x))
        graphs.append(graph)
    for _ in range(3):
        for graph in graphs:
            graph.replay()
        eager = kernel.turing_int8_linear_adapters(**a)
        torch.cuda.synchronize(dev)
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[0])
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    got = []
    for _ in range(4):
        for s, x in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                got.append(kernel.turing_int8_linear_adapters(**x))
    torch.cuda.synchronize(dev)
    assert all(torch.equal(o, want[i % 2]) for i, o in enumerate(got))


def test_op_and_function_agree(gpu_device):
    a = _inputs(gpu_device, 20, 256, 64, 8, 2, seed=8)
    assert torch.equal(torch.ops.turing_utils.int8_linear_adapters(**a), kernel.turing_int8_linear_adapters(**a))


@pytest.mark.parametrize("group", [128, 256])
def test_loaded_adapters_act_on_the_unrotated_activation(gpu_device, group):
    """LinearAdapters.from_float on a W8A8 linear: the adapter's part of the
    output is scaling (x A^T) B^T of the activation that the codes stand for."""
    from comfyui_turing_utils_kernel.adapters import _rotation

    g = torch.Generator().manual_seed(9)
    k, n, m = 768, 256, 37
    x = torch.randn(m, k, generator=g).to(torch.bfloat16).to(gpu_device)
    pairs = [(torch.randn(r, k, generator=g) * k ** -0.5, torch.randn(n, r, generator=g) * 0.3, s)
             for r, s in ((4, 1.0), (11, 0.25))]
    bank = kernel.LinearAdapters.from_float(pairs, group, device=gpu_device)
    assert bank.rank == 16 and bank.count == 2
    codes, scale = torch.ops.turing_utils.bf16_int8_convrot_quantize(x, group)
    weight = torch.zeros(n, k, dtype=torch.int8, device=gpu_device)
    ids = torch.tensor([i % 3 - 1 for i in range(m)], dtype=torch.int32, device=gpu_device)
    got = kernel.turing_int8_linear_adapters(codes, weight, scale, torch.ones(n, device=gpu_device), None, bank.down,
                                             bank.up, bank.scaling, ids)
    held = (codes.double() * scale.double()).view(m, -1, group) @ _rotation(group, gpu_device)  # its own inverse
    held = held.view(m, k)
    assert (held - x.double()).norm() <= 0.02 * x.double().norm()
    for i, (a, b, s) in enumerate(pairs):
        rows = (ids == i).nonzero().view(-1)
        a, b = a.to(gpu_device).double(), b.to(gpu_device).double()
        want = (held[rows] @ a.t()) @ b.t() * s
        # A rotated and B rounded to bf16 (half a step each), then the kernel's own
        slack = (held[rows].norm(dim=1, keepdim=True) * a.norm(dim=1)) @ b.abs().t() * s
        assert ((got[rows].double() - want).abs() <= 3 * ref.BF16 * slack + ref.BF16 * want.abs()).all()
    assert (got[ids == -1] == 0).all()
