"""GPU: a Wan block that reads a key/value cache of the chunks before, against the fp32
reference block (tests/wan_reference.py) over all tokens up to the chunk's end."""
from __future__ import annotations

import pytest
import torch

from tests import wan_reference as ref
from tests.test_gpu_wan_requests import BATCH, IDS, _merged, setup  # noqa: F401  (the fixture)

pytestmark = pytest.mark.gpu

# The bar: as BLOCK_REL_MAX of test_gpu_wan_requests.py, with two more errors in the self-attention's term.  Values are
# codes of a page's largest, about 4 of their deviations over 8192 of them, so off by 4 / 127 / sqrt(12) = 0.0091 of
# them rms; keys whose pages do not begin where the chunk's blocks of 64 do are made into codes a second time, by 0.0091
# likewise.  sqrt(0.025^2 + 2 * 0.0091^2) = 0.0281 of that term and so of the update at most, and with the residual's
# roundings sqrt(0.0281^2 + 0.0083^2) = 0.0293.
CACHED_REL_MAX = 0.0293
CHUNKS = ((0, 232), (232, 464), (464, 696))  # a frame of the grid each: no multiple of 64


def _cached(block, inputs, cache, ids=None, chunks=CHUNKS):
    x, e, context, freqs = inputs
    return [block(x[:, lo:hi], e, context, freqs[:, lo:hi], adapter_ids=ids, cache=cache) for lo, hi in chunks]


def _sequences(device):
    from comfyui_turing_utils_kernel.turing_sage import SequenceKVCache

    return SequenceKVCache.allocate(BATCH, 696, 4, 128, device)


def test_chunk_by_chunk(setup, gpu_device):
    """Each chunk sees the chunks before it and itself, with the adapters of its sample."""
    block, matrices, inputs, ids = setup
    x, e, context, freqs = inputs
    cache = _sequences(gpu_device)
    for (lo, hi), got in zip(CHUNKS, _cached(block, inputs, cache, ids)):
        want = torch.cat([ref.block_rows(block if a < 0 else _merged(block, matrices, a), x[i:i + 1, :hi], e[i:i + 1],
                                         context[i:i + 1], freqs[:, :hi], rows=slice(lo, hi)) for i, a in enumerate(IDS)])
        for i in range(BATCH):
            m = ref.metrics(got[i].float() - x[i, lo:hi].float(), want[i] - x[i, lo:hi].float())
            print(f"chunk {lo} sample {i}: {m}", flush=True)
            assert m["rel_l2"] <= CACHED_REL_MAX, m
    assert cache.lengths.tolist() == [696] * BATCH


def test_a_chunk_again(setup, gpu_device):
    """The next denoising step of a chunk: lengths set back, other tokens there first.  The keys and values of the
    chunks before keep their bits but in the page that both share, whose scale may have grown."""
    block, _, inputs, _ = setup
    x, e, context, freqs = inputs
    cache, plain = _sequences(gpu_device), _sequences(gpu_device)
    _cached(block, inputs, plain, chunks=CHUNKS[:1])
    _cached(block, inputs, cache, chunks=CHUNKS[:1])
    held = cache.lengths.clone()
    noisy = (torch.roll(x, 1, 1), e, context, freqs)
    _cached(block, noisy, cache, chunks=CHUNKS[1:2])
    cache.lengths.copy_(held)
    got, = _cached(block, inputs, cache, chunks=CHUNKS[1:2])
    want, = _cached(block, inputs, plain, chunks=CHUNKS[1:2])
    assert torch.equal(cache.lengths, plain.lengths)
    # pages 0 .. 2 hold the first chunk alone, page 3 both, 4 .. 6 the second alone, begun anew
    for a, b in zip(cache.cache.tensors, plain.cache.tensors):
        a, b = (t.view(BATCH, 11, *t.shape[1:]) for t in (a, b))
        assert torch.equal(a[:, :3], b[:, :3]) and torch.equal(a[:, 4:7], b[:, 4:7])
    xs = x[:, 232:464].float()
    assert ref.metrics(got.float() - xs, want.float() - xs)["rel_l2"] <= 2 * CACHED_REL_MAX


def test_replayed_chunks(setup, gpu_device):
    """A captured forward over a cache, replayed for one chunk after the other."""
    block, _, inputs, ids = setup
    x, e, context, freqs = inputs
    cache, eager = _sequences(gpu_device), _sequences(gpu_device)
    part, places = x[:, :232].clone(), freqs[:, :232].clone()
    block(part, e, context, places, adapter_ids=ids, cache=_sequences(gpu_device))
    torch.cuda.synchronize(gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(part, e, context, places, adapter_ids=ids, cache=cache)
    for n, (lo, hi) in enumerate(CHUNKS):
        part.copy_(x[:, lo:hi])
        places.copy_(freqs[:, lo:hi])
        graph.replay()
        torch.cuda.synchronize(gpu_device)
        assert torch.equal(out, block(x[:, lo:hi], e, context, freqs[:, lo:hi], adapter_ids=ids, cache=eager)), n
    assert cache.lengths.tolist() == [696] * BATCH
