"""GPU: the calls of the key/value cache in 8 bits as programs make them: the native
route's bits against the general one's, captured and replayed, on other streams,
without gradients, with little workspace, and one after the other as a model that
writes token by token or chunk by chunk has them."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import _lib, turing_sage
from comfyui_turing_utils_kernel.turing_sage import QuantizedKVCache, SequenceKVCache
from tests import cache_reference as ref
from tests.test_gpu_cache_attn import _ints, _pool, _query

pytestmark = pytest.mark.gpu

REAL = _lib.host_calls


class _General:
    """Every native call refused: the general route alone."""

    def __getattr__(self, name):
        return lambda *args: None


@pytest.fixture
def routes(monkeypatch):
    """Runs a call on the native route and on the general one: (results, results, which native calls served)."""
    def run(f):
        served = []

        class Spy:
            def __getattr__(self, name):
                def call(*args):
                    served.append(getattr(REAL(), name)(*args))
                    return served[-1]
                return call

        monkeypatch.setattr(_lib, "host_calls", Spy)
        native = f()
        monkeypatch.setattr(_lib, "host_calls", _General)
        general = f()
        monkeypatch.setattr(_lib, "host_calls", REAL)
        return native, general, [s is not None for s in served]
    return run


def _tokens(gen, device, *shape, dtype=torch.bfloat16):
    return torch.randn(*shape, generator=gen).to(dtype).to(device)


def _copy(pool):
    return QuantizedKVCache(*(t.clone() for t in pool))


@pytest.mark.parametrize("layout", ["HND", "NHD"])
@pytest.mark.parametrize("kind", ["bf16", "f16", "int8"])
@pytest.mark.parametrize("lq", [1, 90])
def test_routes_give_the_same_bits(gpu_device, routes, layout, kind, lq):
    pool, table, g = _pool(gpu_device, 2, 3, 64, 5, lq)
    dtype = torch.float16 if kind == "f16" else torch.bfloat16
    shape = (2, 3, lq, 64) if layout == "HND" else (2, lq, 3, 64)
    key, value = (_tokens(g, gpu_device, *shape, dtype=dtype) for _ in range(2))
    mean = _tokens(g, gpu_device, 2, 3, 64)
    q, kw = _query(gpu_device, 2, 6, lq, 64, kind, layout, g)
    lengths, new = _ints([70, 200], gpu_device), _ints([lq, 0], gpu_device)

    def run():
        cache = _copy(pool)
        after = turing_sage.kv_cache_append(key, value, cache, table, lengths, tensor_layout=layout, new_lengths=new, key_mean=mean)
        return (after, *cache.tensors, turing_sage.kv_cache_attention(q, cache, table, after, tensor_layout=layout,
                                                                      is_causal=True, query_lengths=new, sm_scale=0.2, **kw),
                *turing_sage.kv_cache_read(cache, table, after, max_length=300, starts=_ints([3, 0], gpu_device),
                                           tensor_layout=layout, dtype=dtype, key_mean=mean))

    native, general, served = routes(run)
    assert served == [True] * 3
    for a, b in zip(native, general):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b)


def test_int8_keys_on_both_routes(gpu_device, routes):
    pool, table, g = _pool(gpu_device, 2, 3, 128, 5, 4)
    key = torch.randint(-127, 128, (2, 100, 3, 128), generator=g, dtype=torch.int8).to(gpu_device)
    scale = (torch.rand(2, 3, 2, generator=g) + 0.1).to(gpu_device)
    value = _tokens(g, gpu_device, 2, 100, 3, 128)

    def run():
        cache = _copy(pool)
        return (turing_sage.kv_cache_append(key, value, cache, table, _ints([0, 65], gpu_device), tensor_layout="NHD",
                                            key_scale=scale), *cache.tensors)

    native, general, served = routes(run)
    assert served == [True] and all(torch.equal(a, b) for a, b in zip(native, general))


def test_forms_that_are_not_plain(gpu_device, routes):
    """Strided tables, lengths and queries, narrow heads: the general route, and the plain call's bits."""
    pool, table, g = _pool(gpu_device, 2, 3, 64, 5, 6)
    cache = QuantizedKVCache(*pool)
    lengths = _ints([70, 300], gpu_device)
    wide = torch.stack((table, table), -1)[..., 0]
    spread = torch.stack((lengths, lengths), -1)[:, 0]
    assert not wide.is_contiguous() and not spread.is_contiguous()
    q, _ = _query(gpu_device, 2, 6, 40, 64, "bf16", "HND", g)
    plain = turing_sage.kv_cache_attention(q, cache, table, lengths)
    off = torch.empty(q.numel() + 1, dtype=q.dtype, device=gpu_device)[1:].view(q.shape).copy_(q)
    for args in ((q, cache, wide, lengths), (q, cache, table, spread), (off, cache, table, lengths),
                 (q.transpose(2, 3).contiguous().transpose(2, 3), cache, table, lengths)):
        native, general, _ = routes(lambda: turing_sage.kv_cache_attention(*args))
        assert torch.equal(native, plain) and torch.equal(general, plain)
    assert torch.equal(turing_sage.kv_cache_attention(q, cache, table, lengths, query_lengths=_ints([40, 40], gpu_device)), plain)
    k, v = turing_sage.kv_cache_read(cache, table, lengths, max_length=90)
    again = turing_sage.kv_cache_read(cache, wide, spread, max_length=90)
    assert torch.equal(k, again[0]) and torch.equal(v, again[1])


def test_errors_on_the_native_route(gpu_device):
    """What the general route refuses on the host is refused with the native calls too."""
    pool, table, g = _pool(gpu_device, 2, 3, 64, 5, 8)
    cache, lengths = QuantizedKVCache(*pool), _ints([5, 6], gpu_device)
    q, _ = _query(gpu_device, 2, 6, 4, 64, "bf16", "HND", g)
    key = q[:, :3].contiguous()
    for error, call in (
            (ValueError, lambda: turing_sage.kv_cache_attention(q[:, :5].contiguous(), cache, table, lengths)),
            (ValueError, lambda: turing_sage.kv_cache_attention(q, cache, table[:1], lengths)),
            (TypeError, lambda: turing_sage.kv_cache_attention(q, cache, table.long(), lengths)),
            (TypeError, lambda: turing_sage.kv_cache_attention(q.float(), cache, table, lengths)),
            (ValueError, lambda: turing_sage.kv_cache_attention(q, cache, table, lengths.cpu())),
            (ValueError, lambda: turing_sage.kv_cache_append(q, q, cache, table, lengths)),
            (TypeError, lambda: turing_sage.kv_cache_append(key, key.half(), cache, table, lengths)),
            (ValueError, lambda: turing_sage.kv_cache_append(key, key[:, :, :3], cache, table, lengths)),
            (ValueError, lambda: turing_sage.kv_cache_read(cache, table, lengths, max_length=-1)),
            (ValueError, lambda: turing_sage.kv_cache_read(cache, table, lengths[:1], max_length=4))):
        with pytest.raises(error):
            call()


def test_no_backward(gpu_device):
    """The calls have no gradients, as the framework's other attention: results of leaves carry none, and a
    backward pass says so."""
    pool, table, g = _pool(gpu_device, 1, 2, 64, 3, 9)
    cache, lengths = QuantizedKVCache(*pool), _ints([100], gpu_device)
    q = _query(gpu_device, 1, 2, 3, 64, "bf16", "HND", g)[0].requires_grad_()
    out = turing_sage.kv_cache_attention(q, cache, table, lengths)
    if out.requires_grad:
        with pytest.raises(Exception):
            out.float().sum().backward()
    after = turing_sage.kv_cache_append(q, q, _copy(pool), table, lengths)
    assert not after.requires_grad
    with torch.inference_mode():
        again = turing_sage.kv_cache_attention(q, cache, table, lengths)
        inference = _copy(pool)
        turing_sage.kv_cache_append(q, q, inference, table, lengths)
    assert torch.equal(again, out.detach())
    outside = _copy(pool)
    turing_sage.kv_cache_append(q.detach(), q.detach(), outside, table, lengths)
    assert all(torch.equal(a, b) for a, b in zip(inference.tensors, outside.tensors))


def test_a_write_is_noticed(gpu_device):
    """The cache's tensors count as changed, so that autograd refuses what it saved of them."""
    pool, table, g = _pool(gpu_device, 1, 2, 64, 3, 10)
    before = [t._version for t in pool]
    x = _tokens(g, gpu_device, 1, 2, 4, 64)
    turing_sage.kv_cache_append(x, x, QuantizedKVCache(*pool), table, _ints([0], gpu_device))
    assert all(t._version > n for t, n in zip(pool, before))


@pytest.mark.parametrize("lq", [1, 40, 200])
def test_replayed_graph(gpu_device, lq):
    """A captured step of append and attention, replayed with eager work in between; two graphs of one cache."""
    g = torch.Generator().manual_seed(lq)
    seq = SequenceKVCache.allocate(2, 900, 2, 128, gpu_device)
    x, y = (_tokens(g, gpu_device, 2, 700, 2, 128) for _ in range(2))
    seq.append(x, y, tensor_layout="NHD")
    new, q = _tokens(g, gpu_device, 2, lq, 2, 128), _tokens(g, gpu_device, 2, lq, 8, 128)

    def step(s):
        s.append(new, new, tensor_layout="NHD")
        return s.attend(q, tensor_layout="NHD", is_causal=True)

    def clone():
        return SequenceKVCache(_copy(seq.cache.tensors), seq.block_table, seq.lengths.clone())

    start = clone()
    step(clone())
    torch.cuda.synchronize(gpu_device)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(seq)
        graphs.append((graph, out))
    for n in range(5):
        new.copy_(torch.randn(new.shape, generator=g).to(torch.bfloat16) * (n + 1))
        q.copy_(torch.randn(q.shape, generator=g).to(torch.bfloat16))
        for t, s in zip((*seq.cache.tensors, seq.lengths), (*start.cache.tensors, start.lengths)):
            t.copy_(s)
        eager = clone()
        want = step(eager)
        torch.cuda.synchronize(gpu_device)
        graph, out = graphs[n % 2]
        graph.replay()
        torch.cuda.synchronize(gpu_device)
        assert torch.equal(out, want) and torch.equal(seq.lengths, eager.lengths)
        assert all(torch.equal(a, b) for a, b in zip(seq.cache.tensors, eager.cache.tensors))


def test_another_stream(gpu_device):
    """Calls run on the current stream: made behind a long kernel on a side stream, they see its results."""
    pool, table, g = _pool(gpu_device, 2, 2, 128, 20, 12)
    q, _ = _query(gpu_device, 2, 8, 150, 128, "bf16", "HND", g)
    cache, lengths = QuantizedKVCache(*pool), _ints([1200, 700], gpu_device)
    want = turing_sage.kv_cache_attention(2 * q, cache, table, lengths)
    k, v = turing_sage.kv_cache_read(cache, table, lengths, max_length=1200)
    torch.cuda.synchronize(gpu_device)
    side = torch.cuda.Stream(gpu_device)
    big = torch.zeros(1 << 28, device=gpu_device)
    late = q.clone()
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream(gpu_device))
        for _ in range(20):
            big.add_(1.0)
        late.mul_(2.0)
        got = turing_sage.kv_cache_attention(late, cache, table, lengths)
        back = turing_sage.kv_cache_read(cache, table, lengths, max_length=1200)
    side.synchronize()
    assert torch.equal(got, want) and torch.equal(back[0], k) and torch.equal(back[1], v)


@pytest.mark.parametrize("lq", [1, 10, 60, 300])
def test_little_workspace(gpu_device, lq):
    """Fewer ranges where the workspace is small, down to none: the same result within the bound."""
    pool, table, g = _pool(gpu_device, 1, 2, 128, 90, 13)
    q, _ = _query(gpu_device, 1, 4, lq, 128, "bf16", "HND", g)
    lengths = _ints([5700], gpu_device)
    want, bound = ref.attend(q, pool, table, lengths, "HND", True)
    lib, stream = _lib.load(), torch.cuda.current_stream(gpu_device).cuda_stream
    full = lib.tu_kv_cache_attn_workspace(1, 4, 2, lq, 128, 5700, 0, 1, 256)
    assert full > 0
    for nbytes in (full, full // 2 + 16, 4 * lq * 132 * 4 * 2, 4 * lq * 132 * 4 - 16, 0):
        work = torch.full((nbytes + 256,), 0xa5, dtype=torch.uint8, device=gpu_device)
        out = torch.empty_like(q)
        status = lib.tu_kv_cache_attn(q.data_ptr(), None, 0, 1, *(t.data_ptr() for t in pool), pool[0].size(0), table.data_ptr(),
                                      90, lengths.data_ptr(), None, out.data_ptr(), 1, 4, 2, lq, 128, *q.stride()[:3],
                                      *out.stride()[:3], 128 ** -0.5, 1, 5700, 256, work.data_ptr() if nbytes else None,
                                      nbytes, stream)
        torch.cuda.synchronize(gpu_device)
        assert status == 0 and bool(((out.double() - want).abs() <= bound).all()), nbytes
        assert bool((work[nbytes:] == 0xa5).all())


def test_outputs_of_strided_memory(gpu_device):
    """The entry point writes its rows and nothing between or behind them."""
    pool, table, g = _pool(gpu_device, 2, 2, 64, 5, 14)
    cache, lengths = QuantizedKVCache(*pool), _ints([300, 90], gpu_device)
    lib, stream = _lib.load(), torch.cuda.current_stream(gpu_device).cuda_stream
    for lq in (1, 21, 130):
        q, _ = _query(gpu_device, 2, 4, lq, 64, "bf16", "HND", g)
        want = turing_sage.kv_cache_attention(q, cache, table, lengths)
        room = torch.full((2, 4, lq + 3, 72), 7.0, dtype=torch.bfloat16, device=gpu_device)
        out = room[:, :, :lq, :64]
        work = torch.empty(1 << 24, dtype=torch.uint8, device=gpu_device)
        status = lib.tu_kv_cache_attn(q.data_ptr(), None, 0, 1, *(t.data_ptr() for t in pool), pool[0].size(0), table.data_ptr(),
                                      5, lengths.data_ptr(), None, out.data_ptr(), 2, 4, 2, lq, 64, *q.stride()[:3],
                                      *out.stride()[:3], 0.125, 0, 320, 256, work.data_ptr(), work.numel(), stream)
        torch.cuda.synchronize(gpu_device)
        assert status == 0 and torch.equal(out, want)
        out.fill_(7.0)
        assert bool((room == 7.0).all())


@pytest.mark.parametrize("d,hq,hkv", [(64, 6, 2), (128, 4, 4)])
def test_token_by_token_and_in_chunks(gpu_device, d, hq, hkv):
    """A prompt, tokens one at a time, and a chunk again at the place of the last: each step's attention against
    the definition over what the cache holds then, and the whole against attention without a cache.

    The bars.  A page's scale is at most s = max |x| / 127, here about 0.04.  A code is off by half a step for its
    first rounding and by half for each time its page's scale grows after that, three times here at most (22 tokens,
    1, 1, 40): keys and values by 2 s.  A score's error is a sum of d such roundings with a query's elements of size 1:
    rms at most sqrt(4) * s / sqrt(12) = 0.023, six times which is 0.14.  The output moves by sum p_j delta_j (v_j -
    out), at most 0.14 of the weighted mean of |v_j - out|, which is below 1 for these values; the values' own errors
    add 2 s = 0.08 and the rounding of the output 4.8 * 2^-8 = 0.02: 0.24."""
    g = torch.Generator().manual_seed(d)
    seq = SequenceKVCache.allocate(2, 400, hkv, d, gpu_device)
    total = 330
    k, v = (_tokens(g, gpu_device, 2, hkv, total, d) for _ in range(2))
    q = _tokens(g, gpu_device, 2, hq, total, d)
    at = 0
    for n in (150, 1, 1, 63, 1, 64, 50):
        if at == 216:  # a chunk that is written twice: other tokens first
            held = seq.lengths.clone()
            seq.append(-k[:, :, at:at + n] * 0.5, v[:, :, at:at + n] * 0.5)
            seq.lengths.copy_(held)
        seq.append(k[:, :, at:at + n], v[:, :, at:at + n])
        at += n
        got = seq.attend(q[:, :, at - n:at].contiguous(), is_causal=True)
        want, bound = ref.attend(q[:, :, at - n:at], list(seq.cache.tensors), seq.block_table, seq.lengths, "HND", True)
        assert seq.lengths.tolist() == [at, at] and bool(((got.double() - want).abs() <= bound).all())
        kd, vd = (t[:, :, :at].double().repeat_interleave(hq // hkv, 1) for t in (k, v))
        s = (q[:, :, at - n:at].double() @ kd.transpose(2, 3).contiguous()) * d ** -0.5
        hidden = torch.arange(at, device=gpu_device)[None] > torch.arange(at - n, at, device=gpu_device)[:, None]
        whole = torch.softmax(s.masked_fill(hidden, -torch.inf), -1) @ vd
        assert float((got.double() - whole).abs().max()) <= 0.24
    back = seq.read(max_length=at)
    for got, want in zip(back, (k, v)):
        top = float(want.float().abs().max())
        assert float((got.float() - want.float()).abs().max()) <= 2.01 * top / 127 + top * 2 ** -8


def test_two_pools_at_once(gpu_device):
    """Calls on two caches from two streams do not meet."""
    pools = [_pool(gpu_device, 1, 2, 128, 60, s) for s in (20, 21)]
    lengths = _ints([3800], gpu_device)
    q, _ = _query(gpu_device, 1, 4, 33, 128, "bf16", "HND", pools[0][2])
    want = [turing_sage.kv_cache_attention(q, QuantizedKVCache(*p), t, lengths) for p, t, _ in pools]
    torch.cuda.synchronize(gpu_device)
    streams = [torch.cuda.Stream(gpu_device) for _ in pools]
    got = [[], []]
    for _ in range(10):
        for i, (p, t, _) in enumerate(pools):
            with torch.cuda.stream(streams[i]):
                got[i].append(turing_sage.kv_cache_attention(q, QuantizedKVCache(*p), t, lengths))
    torch.cuda.synchronize(gpu_device)
    for i in range(2):
        assert all(torch.equal(x, want[i]) for x in got[i])


def test_a_backward_pass_is_refused(gpu_device, routes):
    """Of a leaf the result is one that autograd knows, and its backward pass an error, on whichever route; the values
    are those of a call without gradients."""
    pool, table, g = _pool(gpu_device, 1, 2, 64, 3, 9)
    cache, lengths = QuantizedKVCache(*pool), _ints([100], gpu_device)
    q = _query(gpu_device, 1, 2, 3, 64, "bf16", "HND", g)[0].requires_grad_()
    native, general, served = routes(lambda: turing_sage.kv_cache_attention(q, cache, table, lengths))
    assert served == [False]
    for out in (native, general):
        assert out.requires_grad
        with pytest.raises(RuntimeError, match="backward"):
            out.float().sum().backward()
    assert q.grad is None
    with torch.no_grad():
        again = turing_sage.kv_cache_attention(q, cache, table, lengths)
    assert not again.requires_grad and torch.equal(again, native.detach())
