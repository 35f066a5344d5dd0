"""GPU: attention over the key/value cache in 8 bits in each form that a launch takes,
asserted by the launch's own choice: 16, 128 and 256 rows a workgroup, a sequence's keys
as one range and as several.  Two sequences of 75 and 33 pages, more than a wave knows at
once where one range has them all (the bound that the split is made for is less than the
lengths then), with ends inside pages, pages that are none and rows behind the queries."""
from __future__ import annotations

import pytest
import torch

from comfyui_turing_utils_kernel import _lib, turing_sage
from tests import cache_reference as ref
from tests.test_gpu_cache_attn import _check, _ints, _pool, _query

# form: (rows a workgroup, split or not): (K/V heads, query heads of each, query tokens, bound of the lengths)
FORMS = {(16, False): (2, 2, 41, 64), (16, True): (2, 2, 41, 1536), (128, False): (66, 1, 260, 64),
         (128, True): (2, 2, 130, 4800), (256, False): (48, 2, 150, 1536), (256, True): (24, 1, 150, 1536)}
PAGES, LENGTHS = 75, (4790, 2100)
KINDS = dict(bf16=0, f16=1, int8=2)

gpu = pytest.mark.gpu
each_form = pytest.mark.parametrize("form", FORMS, ids=lambda f: f"{f[0]}{'-split' if f[1] else ''}")


@each_form
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("causal", [0, 1])
def test_the_sizes_take_the_forms(form, d, kind, causal):
    heads, group, lq, most = FORMS[form]
    plan = _lib.load().tu_kv_cache_attn_plan(2, heads * group, heads, lq, d, most, KINDS[kind], causal, 256)
    assert (plan >> 16, (plan & 0xffff) > 1) == form


def test_the_plan_and_its_workspace():
    lib = _lib.load()
    for args in ((4, 16, 4, 1, 128, 8190, 0, 0, 256), (1, 12, 12, 1560, 128, 9360, 2, 0, 256), (2, 16, 4, 4001, 128, 4001, 0, 1, 256)):
        plan, rows = lib.tu_kv_cache_attn_plan(*args), args[0] * args[1] * args[3]
        assert plan >> 16 in (16, 128, 256) and plan & 0xffff >= 1
        assert lib.tu_kv_cache_attn_workspace(*args) == ((plan & 0xffff) * rows * 132 * 4 if plan & 0xffff > 1 else 0)
        for i in (0, 1, 2, 3, 4, 5, 8):
            assert lib.tu_kv_cache_attn_plan(*args[:i], 0, *args[i + 1:]) == 0


class _Call:
    """A form's inputs; the same call again with what a test changed of them."""

    def __init__(self, device, form, d, kind="bf16", layout="HND", blkq=16, seed=0):
        if torch.cuda.get_device_properties(device).multi_processor_count != 256:
            pytest.skip("the sizes take these forms on 256 compute units")
        heads, group, self.lq, self.most = FORMS[form]
        print(f"[cache attention] {form} D {d} {kind}", flush=True)
        self.device, self.layout, self.heads = device, layout, heads
        self.pool, self.table, g = _pool(device, 2, heads, d, PAGES, 100 * form[0] + d + seed)
        self.q, self.kw = _query(device, 2, heads * group, self.lq, d, kind, layout, g, blkq)
        self.lengths, self.counts = _ints(LENGTHS, device), _ints([self.lq, self.lq - 7], device)

    def __call__(self, causal=True):
        return turing_sage.kv_cache_attention(
            self.q, turing_sage.QuantizedKVCache(*self.pool), self.table, self.lengths, tensor_layout=self.layout,
            is_causal=causal, max_length=self.most, query_lengths=self.counts, **self.kw)

    def check(self, causal=True):
        return _check(self.q, self.pool, self.table, self.lengths, self.layout, causal, max_length=self.most,
                      query_lengths=self.counts, **self.kw)


@gpu
@each_form
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("kind,layout,blkq", [("bf16", "NHD", 16), ("int8", "HND", 16), ("f16", "HND", 16)])
def test_values(gpu_device, form, d, kind, layout, blkq):
    call = _Call(gpu_device, form, d, kind, layout, blkq)
    for causal in (False, True):
        got = call.check(causal)
        assert not ref.hnd(got, layout)[1, :, call.lq - 7:].any()
        assert torch.equal(got, call(causal))


@gpu
@each_form
@pytest.mark.parametrize("blkq", [1, 48, 128])
def test_query_blocks(gpu_device, form, blkq):
    _Call(gpu_device, form, 64, "int8", "NHD", blkq, seed=1).check()


@gpu
@each_form
@pytest.mark.parametrize("kind", ["bf16", "int8"])
def test_pages_that_are_none(gpu_device, form, kind):
    call = _Call(gpu_device, form, 64, kind, seed=2)
    for at, page in (((0, 0), -1), ((0, 1), 10 ** 6), ((0, 40), -(10 ** 9)), ((0, 70), -1), ((0, 74), -2), ((1, 31), 10 ** 9)):
        call.table[at] = page
    for causal in (False, True):
        call.check(causal)


@gpu
@each_form
@pytest.mark.parametrize("d", [64, 128])
def test_what_is_not_seen_changes_nothing(gpu_device, form, d):
    """Codes behind the ends, pages of no table, rows behind a sequence's queries: any bytes, the same bits."""
    call = _Call(gpu_device, form, d, seed=3)
    want = call()
    for b, length in enumerate(LENGTHS):
        page, rest = int(call.table[b, length // 64]), length % 64
        call.pool[0][page, :, rest:] = -128
        call.pool[1][page, :, :, rest:] = -128
        behind = call.table[b, length // 64 + 1:].long()
        call.pool[2][behind], call.pool[3][behind] = float("nan"), float("inf")
    call.q[1, :, call.lq - 7:] = float("nan")
    got = call()
    assert torch.equal(got, want) and torch.isfinite(got).all()


@gpu
@each_form
@pytest.mark.parametrize("which,value", [(2, float("nan")), (2, float("inf")), (3, float("nan")), (3, float("inf"))])
def test_scales_that_are_no_numbers(gpu_device, form, which, value):
    """NaN of the rows that see the page, and of no others: those keep their bits."""
    call = _Call(gpu_device, form, 64, seed=4)
    call.counts[1] = call.lq
    want = call()
    page = 4750 // 64  # keys 4736 .. 4799: of the first sequence's rows from 4736 - (4790 - lq) on
    call.pool[which][int(call.table[0, page]), 1] = value
    if which == 2 and value == float("inf"):
        call.pool[0][int(call.table[0, page]), 1] = 0
    got = call()
    sees = torch.arange(4790 - call.lq, 4790, device=gpu_device) >= 4736
    group = call.q.size(1) // call.heads
    bad = torch.zeros(got.shape, dtype=torch.bool, device=gpu_device)
    bad[0, group:2 * group, sees] = True
    assert got[bad].isnan().all() and torch.equal(got[~bad], want[~bad]) and torch.isfinite(want).all()


@gpu
@each_form
@pytest.mark.parametrize("sign", [1, -1])
def test_infinite_scales_of_codes_that_are_not_zero(gpu_device, form, sign):
    """Of keys and of queries: NaN wherever they are seen, scores of minus infinity among them."""
    call = _Call(gpu_device, form, 64, "int8", seed=9)
    call.q.fill_(1)
    call.pool[0].abs_().clamp_(min=1).mul_(sign)
    want = call(False)
    first = int(call.table[0, 3])
    call.pool[2][first, 1] = float("inf")
    call.kw["query_scale"][1, 0, 1] = float("inf")
    got = call(False)
    group = call.q.size(1) // call.heads
    bad = torch.zeros(got.shape, dtype=torch.bool, device=gpu_device)
    bad[0, group:2 * group] = bad[1, 0, 16:32] = True
    assert got[bad].isnan().all() and torch.isfinite(want).all() and torch.isfinite(got[~bad]).all()


@gpu
@each_form
def test_queries_that_are_no_numbers(gpu_device, form):
    """NaN of those rows, and no other's."""
    call = _Call(gpu_device, form, 64, seed=5)
    want = call(False)
    call.q[0, 1, call.lq // 2, 5] = float("nan")
    call.q[0, 0, call.lq - 1, 60] = float("inf")
    got = call(False)
    bad = torch.zeros(got.shape[:3], dtype=torch.bool, device=gpu_device)
    bad[0, 1, call.lq // 2] = bad[0, 0, call.lq - 1] = True
    assert got[bad].isnan().all()
    # A wave's rows share one form of the exponent, so that the others' last bits may change.  Each result is a mean of
    # values below 127 * 0.045 = 5.8 with weights off by 2^-11 (fp16) and 2 ln 2 * 2^-13 (the exponent's constant), rounded
    # once: twice that is 2^-7 of the result and 2 * (2^-11 + 2 ln 2 * 2^-13) * 5.8 = 0.0077 < 2^-7.
    off = (got[~bad].double() - want[~bad].double()).abs()
    assert bool((off <= 2.0 ** -7 * want[~bad].double().abs() + 2.0 ** -7).all())


@gpu
@each_form
@pytest.mark.parametrize("ratio", [0.5, 1 / 200, 1e-9, 0.0])
def test_pages_of_unlike_value_scales(gpu_device, form, ratio):
    """Next pages whose scales differ by less and by more than what one sum of 16-bit weights takes."""
    call = _Call(gpu_device, form, 64, "int8", seed=6)
    call.pool[3][call.table[0, ::2].long()] *= ratio
    call.pool[3][call.table[1, 1:20].long()] *= ratio
    for causal in (False, True):
        call.check(causal)


@gpu
@each_form
def test_past_32_bits(gpu_device, form):
    """Pages whose bytes lie past 2^31 and 2^32 in the pool."""
    call = _Call(gpu_device, form, 128, "int8", seed=7)
    heads, before = call.heads, call.pool
    pages = 2 * 2 ** 32 // (heads * 64 * 128) // 2 + 200  # (4.3 GB of codes each)
    call.pool = [torch.zeros(pages, *t.shape[1:], dtype=t.dtype, device=gpu_device) for t in before]
    at = torch.linspace(0, pages - 1, before[0].size(0)).long().to(gpu_device)
    for t, s in zip(call.pool, before):
        t[at] = s
    call.table = at[call.table.long()].to(torch.int32)
    assert int(call.table.max()) * heads * 64 * 128 > 2 ** 32
    call.check()


@gpu
@each_form
def test_replayed(gpu_device, form):
    """A captured call with new inputs, with eager work between the replays."""
    call = _Call(gpu_device, form, 128, seed=8)
    eager = call().clone()
    torch.cuda.synchronize(gpu_device)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for n in range(3):
        graph.replay()
        torch.cuda.synchronize(gpu_device)
        assert torch.equal(out, eager), n
        call.q.copy_(call.q.flip(2 if n else 1))
        call.lengths.copy_(call.lengths - 70 * n)
        eager = call().clone()
        torch.cuda.synchronize(gpu_device)
