"""The key/value cache in 8 bits on the host: what its calls refuse, their fake
forms, the C entry points' checks before any launch, the batch's sequences, the
Wan block's checks of a cache.  CPU only."""
from __future__ import annotations

import contextlib
import ctypes

import pytest
import torch

from comfyui_turing_utils_kernel import _lib, turing_sage
from comfyui_turing_utils_kernel.turing_sage import QuantizedKVCache, SequenceKVCache, kv_cache
from comfyui_turing_utils_kernel.wan_block import BlockSparsity
from tests import cache_reference as ref
from tests.test_wan_block_host import CFG, _kwargs

META = "meta"


def _i(*shape, device=META):
    return torch.zeros(shape, dtype=torch.int32, device=device)


def _cache(pages=7, heads=2, width=64, device=META):
    return QuantizedKVCache.allocate(pages, heads, width, device)


def _x(*shape, dtype=torch.bfloat16, device=META):
    return torch.zeros(shape, dtype=dtype, device=device)


def _append(key=None, value=None, cache=None, table=None, lengths=None, **kw):
    key = _x(3, 2, 70, 64) if key is None else key
    return turing_sage.kv_cache_append(key, torch.zeros_like(key) if value is None else value, cache or _cache(),
                                       _i(3, 2) if table is None else table, _i(3) if lengths is None else lengths, **kw)


def _read(cache=None, table=None, lengths=None, max_length=100, **kw):
    return turing_sage.kv_cache_read(cache or _cache(), _i(3, 2) if table is None else table,
                                     _i(3) if lengths is None else lengths, max_length=max_length, **kw)


def _attend(query=None, cache=None, table=None, lengths=None, **kw):
    return turing_sage.kv_cache_attention(_x(3, 4, 5, 64) if query is None else query, cache or _cache(),
                                          _i(3, 2) if table is None else table, _i(3) if lengths is None else lengths, **kw)


def test_fake_contracts_and_fullgraph_leaves():
    after = _append()
    assert after.shape == (3,) and after.dtype == torch.int32 and after.device.type == META
    for layout, shape in (("HND", (3, 2, 100, 64)), ("NHD", (3, 100, 2, 64))):
        for x in _read(tensor_layout=layout, dtype=torch.float16):
            assert x.shape == shape and x.dtype == torch.float16
    assert _attend().shape == (3, 4, 5, 64) and _attend().dtype == torch.bfloat16
    out = _attend(_x(3, 5, 4, 40, dtype=torch.float16), tensor_layout="NHD", is_causal=True)
    assert out.shape == (3, 5, 4, 40) and out.dtype == torch.float16
    out = _attend(_x(3, 4, 5, 64, dtype=torch.int8), query_scale=_x(3, 4, 1, dtype=torch.float32))
    assert out.dtype == torch.bfloat16

    def step(x, q, cache, table, lengths):
        after = turing_sage.kv_cache_append(x, x, cache, table, lengths)
        return turing_sage.kv_cache_attention(q, cache, table, after, is_causal=True), \
            turing_sage.kv_cache_read(cache, table, after, max_length=9), after

    out, (k, v), after = torch.compile(step, backend="eager", fullgraph=True)(
        _x(3, 2, 5, 64), _x(3, 4, 5, 64), _cache(), _i(3, 2), _i(3))
    assert out.shape == (3, 4, 5, 64) and k.shape == v.shape == (3, 2, 9, 64) and after.shape == (3,)


def test_cpu_tensors_are_refused():
    cache, table, lengths = _cache(device="cpu"), _i(3, 2, device="cpu"), _i(3, device="cpu")
    with pytest.raises(RuntimeError, match="CUDA|HIP"):
        _append(_x(3, 2, 4, 64, device="cpu"), cache=cache, table=table, lengths=lengths)
    with pytest.raises(RuntimeError, match="CUDA|HIP"):
        _read(cache, table, lengths)
    with pytest.raises(RuntimeError, match="CUDA|HIP"):
        _attend(_x(3, 4, 5, 64, device="cpu"), cache, table, lengths)


def _bad_caches():
    good = _cache()
    yield ValueError, QuantizedKVCache(good.key_codes[:, :, :32], *good.tensors[1:])
    yield ValueError, QuantizedKVCache(good.key_codes, good.value_codes.transpose(2, 3)[..., :32], *good.tensors[2:])
    yield ValueError, QuantizedKVCache(good.key_codes[..., ::2], good.value_codes[:, :, ::2], *good.tensors[2:])
    yield ValueError, QuantizedKVCache(*good.tensors[:2], good.key_scale[:, :1], good.value_scale)
    yield ValueError, QuantizedKVCache(*good.tensors[:3], good.value_scale[:1])
    yield ValueError, QuantizedKVCache(good.key_codes.transpose(2, 3).contiguous().transpose(2, 3), *good.tensors[1:])
    yield ValueError, QuantizedKVCache(*good.tensors[:3], torch.zeros(7, 2))
    yield TypeError, QuantizedKVCache(good.key_codes.to(torch.uint8), *good.tensors[1:])
    yield TypeError, QuantizedKVCache(*good.tensors[:3], good.value_scale.half())


@pytest.mark.parametrize("call", [_append, _read, _attend])
def test_bad_caches_tables_and_lengths(call):
    for error, cache in _bad_caches():
        with pytest.raises(error):
            call(cache=cache)
    for error, kw in ((TypeError, dict(table=_i(3, 2).long())), (TypeError, dict(lengths=_i(3).long())),
                      (ValueError, dict(table=_i(6))), (ValueError, dict(table=_i())), (ValueError, dict(table=_i(3, 0))), (ValueError, dict(lengths=_i(2))),
                      (ValueError, dict(lengths=_i(3, 1))), (ValueError, dict(table=_i(3, 2, device="cpu"))),
                      (ValueError, dict(tensor_layout="BLHD"))):
        with pytest.raises(error):
            call(**kw)


def test_bad_tokens():
    f32 = torch.float32
    codes = _x(3, 2, 70, 64, dtype=torch.int8)
    value = _x(3, 2, 70, 64)
    for error, kw in (
            (ValueError, dict(key=_x(2, 70, 64))), (ValueError, dict(key=_x(3, 3, 70, 64))),
            (ValueError, dict(key=_x(2, 2, 70, 64))), (ValueError, dict(key=_x(3, 2, 70, 65))),
            (ValueError, dict(value=_x(3, 2, 71, 64))), (TypeError, dict(key=_x(3, 2, 70, 64, dtype=f32))),
            (TypeError, dict(value=_x(3, 2, 70, 64, dtype=torch.float16))), (TypeError, dict(key=codes, value=value)),
            (ValueError, dict(key=_x(3, 2, 70, 64, device="cpu"), value=value)),
            (ValueError, dict(key=codes, value=value, key_scale=_x(3, 2, 1, dtype=f32))),
            (TypeError, dict(key=codes, value=value, key_scale=_x(3, 2, 2))),
            (TypeError, dict(key_scale=_x(3, 2, 2, dtype=f32))),
            (ValueError, dict(key=codes, value=value, key_scale=_x(3, 2, 2, dtype=f32, device="cpu"))),
            (TypeError, dict(key_mean=_x(3, 2, 64, dtype=f32))), (ValueError, dict(key_mean=_x(3, 64))),
            (ValueError, dict(key_mean=_x(3, 2, 65))), (ValueError, dict(key_mean=_x(3, 2, 64, device="cpu"))),
            (ValueError, dict(new_lengths=_i(3).long())), (ValueError, dict(new_lengths=_i(2))),
            (ValueError, dict(new_lengths=_i(3, device="cpu")))):
        with pytest.raises(error):
            _append(**kw)


def test_bad_reads():
    for error, kw in ((ValueError, dict(max_length=-1)), (ValueError, dict(max_length=2 ** 31)),
                      (TypeError, dict(dtype=torch.float32)), (ValueError, dict(starts=_i(2))),
                      (ValueError, dict(starts=_i(3).float())), (TypeError, dict(key_mean=_x(3, 2, 64, dtype=torch.float16))),
                      (ValueError, dict(key_mean=_x(3, 3, 64)))):
        with pytest.raises(error):
            _read(**kw)


def test_bad_queries():
    codes, scale = _x(3, 4, 5, 64, dtype=torch.int8), _x(3, 4, 1, dtype=torch.float32)
    for error, kw in (
            (ValueError, dict(query=_x(3, 3, 5, 64))), (ValueError, dict(query=_x(2, 4, 5, 64))),
            (ValueError, dict(query=_x(3, 4, 5, 128))), (ValueError, dict(query=_x(3, 4, 64))),
            (TypeError, dict(query=_x(3, 4, 5, 64, dtype=torch.float32))), (TypeError, dict(query=codes)),
            (TypeError, dict(query_scale=scale)), (TypeError, dict(query=codes, query_scale=scale.half())),
            (ValueError, dict(query=codes, query_scale=scale, blkq=0)), (ValueError, dict(query=codes, query_scale=scale, blkq=4)),
            (ValueError, dict(query=codes, query_scale=torch.zeros(3, 4, 1))), (ValueError, dict(query=_x(3, 4, 5, 64, device="cpu"))),
            (ValueError, dict(max_length=0)), (ValueError, dict(sm_scale=0.0)), (ValueError, dict(sm_scale=float("inf"))),
            (ValueError, dict(sm_scale=float("nan"))), (ValueError, dict(query_lengths=_i(4))),
            (ValueError, dict(query_lengths=_i(3).long()))):
        with pytest.raises(error):
            _attend(**kw)


def test_sequences():
    seq = SequenceKVCache.allocate(3, 130, 2, 40, "cpu")
    assert seq.max_length == 192 and seq.cache.key_codes.shape == (9, 2, 64, 64)
    assert seq.cache.value_codes.shape == (9, 2, 64, 64) and seq.cache.key_scale.shape == (9, 2)
    assert seq.block_table.tolist() == [[0, 1, 2], [3, 4, 5], [6, 7, 8]] and not seq.lengths.any()
    assert QuantizedKVCache.allocate(1, 1, 65, META).key_codes.shape == (1, 1, 64, 128)
    for args in ((0, 1, 1, 64), (1, 0, 1, 64), (1, 1, 0, 64), (1, 1, 1, 129), (1, 1, 1, 0)):
        with pytest.raises(ValueError):
            SequenceKVCache.allocate(*args)
        if args[0]:
            with pytest.raises(ValueError):
                QuantizedKVCache.allocate(*args[1:] if args[1] == 0 else (0, 1, 64))


def test_sequences_move_their_lengths_in_place(monkeypatch):
    seq = SequenceKVCache.allocate(2, 64, 2, 64, META)
    lengths = seq.lengths
    seq.append(_x(2, 2, 3, 64), _x(2, 2, 3, 64))
    assert seq.lengths is lengths
    assert seq.attend(_x(2, 4, 3, 64)).shape == (2, 4, 3, 64)
    assert seq.read(max_length=5, tensor_layout="NHD")[0].shape == (2, 5, 2, 64)


@pytest.fixture
def entry_point(monkeypatch):
    """The general route on CPU tensors, and the arguments that reach the entry points."""
    seen = []
    monkeypatch.setattr(kv_cache, "_require_gpu", lambda *a: None)
    monkeypatch.setattr(kv_cache, "_compute_units", lambda device: 256)
    monkeypatch.setattr(_lib, "call", lambda name, *args: seen.append((name, args)))
    monkeypatch.setattr(_lib, "stream_of", lambda device: None)
    monkeypatch.setattr(torch.cuda, "device", lambda device: contextlib.nullcontext())
    return seen


def _ints_at(address, n):
    return list((ctypes.c_int32 * n).from_address(address))


def test_strided_arguments_reach_the_entry_points_whole(entry_point):
    """Columns of tables, tensors that start off 16 bytes and narrow heads: copies, alive at the call."""
    cache = _cache(device="cpu")
    rows = torch.arange(12, dtype=torch.int32).view(6, 2)
    table, lengths = rows[::2], rows[:, 1][:3]
    x = torch.randn(3, 70, 2, 41).to(torch.bfloat16)[..., 1:]
    turing_sage.kv_cache_append(x, x, cache, table, lengths, tensor_layout="NHD", new_lengths=rows[:, 0][:3])
    turing_sage.kv_cache_read(cache, table, lengths, max_length=5, starts=rows[:, 0][1:4])
    turing_sage.kv_cache_attention(x[:, :9], cache, table, lengths, tensor_layout="NHD", query_lengths=rows[:, 0][2:5])
    (a, append), (r, read), (t, attend) = entry_point
    assert (a, r, t) == ("tu_kv_cache_append", "tu_kv_cache_read", "tu_kv_cache_attn")
    assert append[4:8] == (3, 2, 70, 64) and append[8:14] == (70 * 2 * 64, 64, 2 * 64) * 2
    assert append[0] % 16 == 0 and append[16] == 2
    assert read[4] == 7 and read[6] == 2
    assert attend[14:19] == (3, 2, 2, 9, 64) and attend[27] == 128


@pytest.mark.parametrize("layout", ["HND", "NHD"])
def test_odd_strides_of_axes_of_one(entry_point, layout):
    """One sequence, head and token of rows of 67 channels: torch calls it contiguous, with strides of no 16 bytes."""
    cache = _cache(heads=1, device="cpu")
    table, lengths = _i(1, 2, device="cpu"), _i(1, device="cpu")
    x = torch.randn(1, 9, 2, 67).to(torch.bfloat16)[:, :1, :1, :64]
    assert x.is_contiguous() and 67 in x.stride()
    codes, scale = torch.zeros(1, 9, 2, 67, dtype=torch.int8)[:, :1, :1, :64], torch.ones(1, 1, 1)
    mean = torch.randn(1, 3, 67).to(torch.bfloat16)[:, :1, :64]
    kw = dict(tensor_layout=layout)
    turing_sage.kv_cache_append(x, x, cache, table, lengths, key_mean=mean, **kw)
    turing_sage.kv_cache_append(codes, x, cache, table, lengths, key_scale=scale, **kw)
    turing_sage.kv_cache_attention(x, cache, table, lengths, **kw)
    turing_sage.kv_cache_attention(codes, cache, table, lengths, query_scale=scale, **kw)
    (_, bf16), (_, int8), (_, q), (_, q8) = entry_point
    assert bf16[8:14] == int8[8:14] == (64, 64, 64) * 2
    assert q[19:22] == q8[19:22] == (64, 64, 64)
    assert all(args[i] % 16 == 0 for args, i in ((bf16, 0), (bf16, 2), (int8, 0), (int8, 2), (q, 0), (q8, 0)))


def test_no_tokens(entry_point):
    cache, table = _cache(device="cpu"), _i(2, 2, device="cpu")
    lengths = torch.tensor([-3, 1000], dtype=torch.int32)
    x = _x(2, 2, 0, 64, device="cpu")
    assert turing_sage.kv_cache_append(x, x, cache, table, lengths).tolist() == [0, 128]
    assert turing_sage.kv_cache_attention(x, cache, table, lengths).shape == (2, 2, 0, 64)
    assert turing_sage.kv_cache_read(cache, table, lengths, max_length=0)[0].shape == (2, 2, 0, 64)
    none = _x(0, 2, 5, 64, device="cpu")
    assert turing_sage.kv_cache_append(none, none, cache, table[:0], lengths[:0]).shape == (0,)
    assert turing_sage.kv_cache_attention(none, cache, table[:0], lengths[:0]).shape == (0, 2, 5, 64)
    assert turing_sage.kv_cache_read(cache, table[:0], lengths[:0], max_length=4)[1].shape == (0, 2, 4, 64)
    assert entry_point == []


def test_codes_off_16_bytes_are_refused(entry_point):
    raw = torch.zeros(2 * 64 * 64 + 1, dtype=torch.int8)[1:].view(1, 2, 64, 64)
    scale = torch.zeros(1, 2)
    cache = QuantizedKVCache(raw, torch.zeros_like(raw), scale, scale)
    for call in (lambda: _read(cache, _i(1, 1, device="cpu"), _i(1, device="cpu")),
                 lambda: _attend(_x(1, 2, 3, 64, device="cpu"), cache, _i(1, 1, device="cpu"), _i(1, device="cpu")),
                 lambda: _append(_x(1, 2, 3, 64, device="cpu"), cache=cache, table=_i(1, 1, device="cpu"),
                                 lengths=_i(1, device="cpu"))):
        with pytest.raises(ValueError, match="16 bytes"):
            call()


# The C entry points' own checks: each call but for the one argument named is a good one, and none launches.

P = 1 << 20  # an address that nothing reads


def _entry(name, **kw):
    forms = dict(
        tu_kv_cache_append=dict(
            k=P, k_in_scale=None, v=P, dtype=0, batch=2, hkv=3, len=5, dim=64, k_sb=960, k_sh=320, k_sl=64, v_sb=960, v_sh=320,
            v_sl=64, mean=None, table=P, width=4, lengths=P, new=None, kc=P, vc=P, ks=P, vs=P, pages=9, out=2 * P, stream=None),
        tu_kv_cache_read=dict(
            kc=P, vc=P, ks=P, vs=P, pages=9, table=P, width=4, lengths=P, starts=None, mean=None, k=P, v=P, dtype=0, batch=2,
            hkv=3, len=5, dim=64, k_sb=960, k_sh=320, k_sl=64, v_sb=960, v_sh=320, v_sl=64, stream=None),
        tu_kv_cache_attn=dict(
            q=P, q_scale=None, q_type=0, blkq=16, kc=P, vc=P, ks=P, vs=P, pages=9, table=P, width=4, lengths=P, q_lengths=None,
            o=P, batch=2, hq=6, hkv=3, lq=5, dim=64, q_sb=1920, q_sh=320, q_sl=64, o_sb=1920, o_sh=320, o_sl=64, sm_scale=0.125,
            causal=0, max_length=256, cus=256, workspace=None, workspace_bytes=0, stream=None))
    args = dict(forms[name], **kw)
    assert set(args) == set(forms[name])
    lib = _lib.load()
    status = getattr(lib, name)(*args.values())
    return status, lib.tu_last_error().decode()


SIZES = [dict(dim=96), dict(batch=0), dict(hkv=0), dict(len=0), dict(len=2 ** 31), dict(width=0), dict(width=2 ** 31),
         dict(pages=0), dict(pages=2 ** 31), dict(batch=40000), dict(hkv=70000)]
TOKENS = [dict(dtype=2), dict(k=None), dict(v=None), dict(k=P + 8), dict(v=P + 2), dict(k_sl=68), dict(v_sh=4), dict(k_sb=1),
          dict(mean=P + 4), dict(kc=None), dict(vc=P + 1), dict(ks=None), dict(vs=None), dict(table=None), dict(lengths=None)]


@pytest.mark.parametrize("change", SIZES + TOKENS + [dict(out=None), dict(out=P), dict(k_in_scale=P, k_sl=72)])
def test_append_entry_refuses(change):
    status, message = _entry("tu_kv_cache_append", **change)
    assert status == -1 and "cache append" in message


@pytest.mark.parametrize("change", SIZES + TOKENS)
def test_read_entry_refuses(change):
    status, message = _entry("tu_kv_cache_read", **change)
    assert status == -1 and "cache read" in message


@pytest.mark.parametrize("change", [
    dict(dim=96), dict(q_type=3), dict(q_type=-1), dict(batch=0), dict(hq=0), dict(hkv=0), dict(hq=7), dict(lq=0),
    dict(lq=2 ** 31), dict(batch=70000), dict(hq=70002), dict(batch=65535, hq=65535, hkv=65535, lq=2 ** 30), dict(lq=2 ** 62), dict(cus=0), dict(max_length=0), dict(width=0), dict(width=2 ** 31),
    dict(pages=0), dict(pages=2 ** 31), dict(pages=2 ** 30), dict(q=None), dict(kc=None), dict(vc=None), dict(ks=None),
    dict(vs=None), dict(table=None), dict(lengths=None), dict(o=None), dict(q_type=2), dict(q_type=2, q_scale=P, blkq=0),
    dict(sm_scale=0.0), dict(sm_scale=float("nan")), dict(q=P + 8), dict(q_sl=68), dict(q_type=2, q_scale=P, q_sl=72),
    dict(kc=P + 8), dict(vc=P + 4), dict(o=P + 4), dict(o_sl=66), dict(workspace=P + 8, workspace_bytes=64)])
def test_attention_entry_refuses(change):
    status, message = _entry("tu_kv_cache_attn", **change)
    assert status == -1 and "cache attention" in message


@pytest.mark.parametrize("scale", [1e39, float("inf"), 3e38])
def test_scales_past_32_bits_are_refused(scale):
    """In 32 bits, log2 e of it included, an infinite scale would make a NaN of every row."""
    status, message = _entry("tu_kv_cache_attn", sm_scale=scale)
    assert status == -1 and "positive and finite" in message


@pytest.mark.parametrize("name,kw", [
    ("tu_kv_cache_append", dict(hkv=65535, len=64 * 257, width=1000)),
    ("tu_kv_cache_read", dict(hkv=65535, len=64 * 257, width=1000)),
    ("tu_kv_cache_attn", dict(batch=65535, hq=257, hkv=257, lq=1, max_length=64)),
    ("tu_kv_cache_attn", dict(batch=1, hq=65535, hkv=65535, lq=128 * 257, max_length=64))])
def test_more_workgroups_than_a_launch_has(name, kw):
    """More than 2^32 threads, in workgroups of 256."""
    status, message = _entry(name, **kw)
    assert status == -1 and "grid too large" in message


def test_workspace():
    """Bytes for whole ranges of rows; none where a call has no ranges or no sizes."""
    size = _lib.load().tu_kv_cache_attn_workspace
    row = 132 * 4
    assert size(4, 16, 4, 1, 128, 8190, 0, 0, 256) % (64 * row) == 0 < size(4, 16, 4, 1, 128, 8190, 0, 0, 256)
    assert size(1, 8, 8, 1, 64, 64, 0, 0, 256) == 0  # one page
    for bad in (0, 1, 2, 3, 4, 5, 8):
        args = [4, 16, 4, 1, 128, 8190, 0, 0, 256]
        args[bad] = 0
        assert size(*args) == 0
    huge = 2 ** 31 - 1
    for args in ((65535, 65535, 65535, huge // 2, 128, huge, 0, 0, 256), (65535, 65535, 1, 2 ** 40, 128, 64, 0, 0, 256),
                 (2 ** 40, 16, 4, 1, 128, 64, 0, 0, 256), (4, 2 ** 40, 4, 1, 128, 64, 0, 0, 256), (4, 16, 4, 1, 96, 64, 0, 0, 256)):
        assert size(*args) == 0
    assert size(1, 1, 1, 1, 128, 2 ** 62, 0, 0, 256) > 0
    for causal in (0, 1):  # ranges stay in number, and so does the memory
        for lq in (1, 3, 9, 40, 300, 5000, 32760):
            for pages in (1, 5, 63, 512, 2048):
                got = size(1, 40, 40, lq, 128, 64 * pages, 2 * causal, causal, 256)
                assert got % (40 * lq * row) == 0 and got <= 256 * 40 * lq * row, (lq, pages)


def test_plain_form_of_the_cache():
    """The tests' own plain forms agree with one another: what is appended in pieces and read back is what the
    codes' steps allow, and attention over it is the softmax of its definition."""
    g = torch.Generator().manual_seed(3)
    pool, (table, pages) = None, ref.tables(2, 3, g, "cpu")
    pool = ref.rubbish_pool(pages, 2, 64, g, "cpu")
    x, y = (torch.randn(2, 2, 150, 64, generator=g).to(torch.bfloat16) for _ in range(2))
    lengths = torch.zeros(2, dtype=torch.int32)
    for lo, hi in ((0, 1), (1, 70), (70, 150)):
        pool, lengths = ref.append(x[:, :, lo:hi], y[:, :, lo:hi], pool, table, lengths, "HND")
    assert lengths.tolist() == [150, 150]
    k, v = ref.read(pool, table, lengths, 150, "HND", torch.float16)
    for got, want in ((k, x), (v, y)):
        # one step is at most max / 127, a code made again is off by half a step twice
        assert bool(((got.float() - want.float()).abs() <= want.abs().max() / 127 * 1.01).all())
    q = torch.randn(2, 4, 3, 64, generator=g).to(torch.bfloat16)
    out, bound = ref.attend(q, pool, table, lengths, "HND", True)
    k, v = (t.double().repeat_interleave(2, 1) for t in (k, v))
    seen = torch.arange(150)[None] <= 147 + torch.arange(3)[:, None]
    want = torch.softmax((q.double() @ k.transpose(2, 3) / 8).masked_fill(~seen, -torch.inf), -1) @ v
    # (k and v are rounded to fp16 here: 2^-11 of scores up to 4 or so, and of values)
    assert bool(((out - want).abs() <= 0.01).all()) and bool((bound > 0).all())


def test_wan_block_checks_its_cache():
    from comfyui_turing_utils_kernel.wan_block import WanBlockW8A8, rope_freqs

    block = WanBlockW8A8(CFG, norm3_weight=torch.ones(256), **_kwargs())
    x = torch.zeros(1, 8, 256, dtype=torch.bfloat16)

    def call(cache, sparsity=None, x=x):
        block(x, torch.zeros(1, 6, 256), x, rope_freqs((1, 2, 4), 128), cache=cache, sparsity=sparsity)

    with pytest.raises(ValueError, match="exclude"):
        call(SequenceKVCache.allocate(1, 64, 2, 128, "cpu"), BlockSparsity(keep=1))
    for cache in (SequenceKVCache.allocate(2, 64, 2, 128, "cpu"), SequenceKVCache.allocate(1, 64, 4, 128, "cpu"),
                  SequenceKVCache.allocate(1, 64, 2, 64, "cpu")):
        with pytest.raises(ValueError, match="the cache has"):
            call(cache)
    with pytest.raises(ValueError, match="do not fit"):
        call(SequenceKVCache.allocate(1, 64, 2, 128, "cpu"), x=torch.zeros(1, 65, 256, dtype=torch.bfloat16))
