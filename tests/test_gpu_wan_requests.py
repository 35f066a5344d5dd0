"""GPU: a Wan block whose samples carry the adapters of their own requests and
whose self-attention keeps chosen key blocks, against the fp32 reference block
(tests/wan_reference.py) with each sample's adapters merged into its dense
weights and the keys that were not chosen masked out.

The bar.  A sublayer of test_gpu_wan_block.py is within 0.025 of its reference
(INT8 activations, bf16), and the adapters add a rounding of A, 2^-8 of a third
of y at most, which 0.025 absorbs (sqrt(0.025^2 + 0.0013^2) = 0.02503).  The
update u is the sum of three sublayers' terms, whose errors are independent:
sqrt(sum (0.025 |s_i|)^2) = 0.025 |u| for terms as good as orthogonal.  The
residual stream is rounded to bf16 three times, each by 2^-8 |x| / sqrt(3) rms
at most: 2^-8 |x| together, with |x| about 1.15 and |u| at least 0.54 here
0.0083 |u|.  sqrt(0.025^2 + 0.0083^2) = 0.0264.  (The block bar of that file,
0.018, was set by a measurement at ten times the channels; the block without
adapters, whose path is that file's, is off by 0.0193 to 0.0204 here.)  A
sample with another's adapters, or none, is off by 0.5.  The linears here have
a tenth of that file's inputs, so their weights are sqrt(10) times larger, for
sublayers of the same size."""
from __future__ import annotations

import copy

import pytest
import torch

from tests import wan_reference as ref

pytestmark = pytest.mark.gpu

BLOCK_REL_MAX = 0.0264
GRID, TEXT, BATCH, COUNT = (3, 8, 29), 45, 3, 2  # 696 tokens: 6 query and 11 key blocks, both ragged
IDS = (1, -1, 0)
NAMES = {"self_qkv": 3, "self_o": 1, "cross_q": 1, "cross_kv": 2, "cross_o": 1, "ffn_up": 1, "ffn_down": 1}


def _matrices(block, dev):
    """{linear: [adapter: [(A, B, scaling) of each of its parts]]}, a third of the weights' size."""
    g = torch.Generator(device=dev).manual_seed(21)
    out = {}
    for name, parts in NAMES.items():
        lin = getattr(block, name)
        n, std = lin.out_features // parts, float(ref.dense_weight(lin).std())
        out[name] = [[(torch.randn(r, lin.in_features, generator=g, device=dev) * std / 3 * r ** -0.5 / s,
                       torch.randn(n, r, generator=g, device=dev).to(torch.bfloat16).float(), s)
                      for _ in range(parts)] for r, s in ((8, 0.5), (20, 2.0))]
    return out


def _merged(block, matrices, which):
    """The block with adapter ``which`` in its reference weights."""
    block = copy.copy(block)
    for name, adapters in matrices.items():
        lin = copy.copy(getattr(block, name))
        lin._ref_dense = ref.dense_weight(lin) + torch.cat([s * b @ a for a, b, s in adapters[which]])
        setattr(block, name, lin)
    return block


@pytest.fixture(scope="module")
def setup(gpu_device):
    from comfyui_turing_utils_kernel import LinearAdapters
    from comfyui_turing_utils_kernel.wan_block import WanBlockConfig, random_block, rope_freqs

    block, _ = random_block(WanBlockConfig(dim=512, heads=4, ffn_dim=1408, text_dim=256), seed=3, device=gpu_device)
    for name in NAMES:
        getattr(block, name).weight_scale *= 10 ** 0.5
    matrices = _matrices(block, gpu_device)
    block.set_adapters({
        name: LinearAdapters.concat([LinearAdapters.from_float([a[p] for a in adapters]) for p in range(NAMES[name])])
        for name, adapters in matrices.items()})
    g = torch.Generator(device=gpu_device).manual_seed(22)
    tokens = GRID[0] * GRID[1] * GRID[2]
    x = torch.randn(BATCH, tokens, 512, generator=g, device=gpu_device).to(torch.bfloat16)
    e = 0.1 * torch.randn(BATCH, 6, 512, generator=g, device=gpu_device)
    context = torch.randn(BATCH, TEXT, 512, generator=g, device=gpu_device).to(torch.bfloat16)
    freqs = rope_freqs(GRID, 128, device=gpu_device).to(torch.bfloat16).float()
    ids = torch.tensor(IDS, dtype=torch.int32, device=gpu_device)
    return block, matrices, (x, e, context, freqs), ids


def _reference(block, matrices, inputs):
    x, e, context, freqs = inputs
    return torch.cat([ref.block_rows(block if a < 0 else _merged(block, matrices, a), x[i:i + 1], e[i:i + 1],
                                     context[i:i + 1], freqs) for i, a in enumerate(IDS)])


def _check(got, want, x):
    for i in range(BATCH):
        m = ref.metrics(got[i].float() - x[i].float(), want[i] - x[i].float())
        print(f"sample {i}: {m}", flush=True)
        assert m["rel_l2"] <= BLOCK_REL_MAX, m


def test_adapters_of_each_sample(setup):
    block, matrices, inputs, ids = setup
    got = block(*inputs, adapter_ids=ids)
    _check(got, _reference(block, matrices, inputs), inputs[0])
    # a sample without an adapter keeps its bits, the others do not
    plain = block(*inputs)
    assert torch.equal(got[1], plain[1]) and not torch.equal(got[0], plain[0])


def test_adapters_and_key_blocks(setup, monkeypatch):
    from comfyui_turing_utils_kernel import turing_sage, wan_block

    block, matrices, inputs, ids = setup
    sparsity = wan_block.BlockSparsity(keep=4, sink_blocks=1, local_blocks=1)
    chosen = []

    def attend(state, **kw):
        chosen.append(turing_sage.select_key_blocks(
            state.query_int8, state.query_scale, state.key_int8, state.key_scale, tensor_layout=state.tensor_layout,
            blkq=state.blkq, blkk=state.blkk, **kw))
        return turing_sage.sparse_sageattn_from_prequantized(state, **kw)

    monkeypatch.setattr(wan_block, "sparse_sageattn_from_prequantized", attend)
    got = block(*inputs, adapter_ids=ids, sparsity=sparsity)
    index, = chosen
    assert index.shape == (BATCH, 4, 6, 4) and bool((index >= 0).all())
    tokens = inputs[0].shape[1]
    near = torch.arange(tokens, device=index.device) // 128 * 2
    sample = iter(range(BATCH))

    def attention(q, k, v):
        if k.shape[1] != tokens:
            return dense(q, k, v)
        keep = torch.zeros(4, 6, 11, dtype=torch.bool, device=q.device).scatter_(2, index[next(sample)].long(), True)
        assert bool(keep[:, :, 0].all()) and bool(keep.gather(2, near[::128].expand(4, 6).unsqueeze(-1)).all())
        seen = keep.repeat_interleave(128, 1)[:, :tokens].repeat_interleave(64, 2)[:, :, :tokens]
        qh, kh, vh = (t.permute(0, 2, 1, 3).contiguous() for t in (q, k, v))
        s = (qh @ kh.transpose(2, 3).contiguous()) * q.shape[-1] ** -0.5
        return (torch.softmax(s.masked_fill(~seen, -torch.inf), -1) @ vh).permute(0, 2, 1, 3)

    dense = ref.attention
    monkeypatch.setattr(ref, "attention", attention)
    want = _reference(block, matrices, inputs)
    _check(got, want, inputs[0])
    # Every key block kept: the dense block's result but for the order of its
    # sums.  A sum that rounds to the next bf16 moves a code of the projection
    # after it by a whole step in a few per cent of the places, so the two are
    # as far apart as two roundings: each within the bar of the same reference,
    # so within twice the bar of each other.
    every = block(*inputs, adapter_ids=ids, sparsity=wan_block.BlockSparsity(keep=11))
    full = block(*inputs, adapter_ids=ids)
    x = inputs[0].float()
    assert ref.metrics(every.float() - x, full.float() - x)["rel_l2"] <= 2 * BLOCK_REL_MAX


def test_replayed_graph(setup, gpu_device):
    """A captured forward, replayed with eager forwards of the same block and new inputs in between."""
    from comfyui_turing_utils_kernel.wan_block import BlockSparsity

    block, _, inputs, ids = setup
    sparsity = BlockSparsity(keep=3, local_blocks=1)
    x, e, context, freqs = (t.clone() for t in inputs)
    which = ids.clone()
    block(x, e, context, freqs, adapter_ids=which, sparsity=sparsity)
    torch.cuda.synchronize(gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x, e, context, freqs, adapter_ids=which, sparsity=sparsity)
    for n in range(4):
        x.copy_(inputs[0] * (1 + 0.25 * n))
        which.copy_(torch.tensor([n % 2, 1, -1], dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize(gpu_device)
        got = out.clone()
        assert torch.equal(got, block(x, e, context, freqs, adapter_ids=which, sparsity=sparsity)), n
