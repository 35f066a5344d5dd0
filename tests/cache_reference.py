"""Plain forms of the key/value cache in 8 bits, and the inputs and bounds that its
tests share (test infrastructure): codes by the formula in 32 bits, attention in
64."""
from __future__ import annotations

import math

import torch

PAGE = 64
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def blocks(n):
    return (n + PAGE - 1) // PAGE


def hnd(x, layout):
    return x if layout == "HND" else x.transpose(1, 2)


def rubbish_pool(pages, heads, d, gen, device):
    """A pool whose pages hold anything: codes of the whole byte, scales among them NaN and infinity."""
    scale = torch.rand(pages, heads, generator=gen)
    scale[::3] = float("nan")
    scale[1::3] = float("inf")
    return [torch.randint(-128, 128, (pages, heads, PAGE, d), generator=gen, dtype=torch.int8).to(device),
            torch.randint(-128, 128, (pages, heads, d, PAGE), generator=gen, dtype=torch.int8).to(device),
            scale.to(device), scale.clone().to(device)]


def tables(batch, row, gen, device, spare=3):
    """(block tables with pages in no order, pages of the pool): `spare` pages are in no table."""
    pages = batch * row + spare
    return torch.randperm(pages, generator=gen)[:batch * row].view(batch, row).to(torch.int32).to(device), pages


def append(key, value, pool, table, lengths, layout, new_lengths=None, key_scale=None, key_mean=None):
    """kv_cache_append on a copy of the pool, on the CPU, page by page in 32 bits: (pool, lengths afterwards)."""
    kc, vc, ks, vs = (t.cpu().clone() for t in pool)
    table, held = table.cpu(), lengths.cpu().tolist()
    k, v = hnd(key, layout).cpu().float(), hnd(value, layout).cpu().float()
    if key_scale is not None:
        k = k * key_scale.cpu().repeat_interleave(PAGE, 2)[:, :, :k.size(2), None]
    if key_mean is not None:
        mean = torch.zeros(k.size(0), k.size(1), k.size(3))
        mean[..., :key_mean.size(2)] = key_mean.cpu().float()
        k = k - mean[:, :, None]
    d = kc.size(3)
    k, v = (torch.nn.functional.pad(x, (0, d - x.size(3))) for x in (k, v))
    after = []
    for b, had in enumerate(held):
        had = min(max(had, 0), table.size(1) * PAGE)
        n = k.size(2) if new_lengths is None else min(max(int(new_lengths[b]), 0), k.size(2))
        n = min(n, table.size(1) * PAGE - had)
        after.append(had + n)
        for j in range(had // PAGE, blocks(had + n) if n else 0):
            page = int(table[b, j])
            if not 0 <= page < kc.size(0):
                continue
            lo, hi = max(had - j * PAGE, 0), min(had + n - j * PAGE, PAGE)
            first = j * PAGE - had
            for x, codes, scales in ((k[b], kc[page], ks[page]), (v[b], vc[page].transpose(1, 2), vs[page])):
                for h in range(x.size(0)):
                    new = x[h, first + lo:first + hi]
                    before = scales[h].abs()
                    # (amax and maximum keep a NaN)
                    s = torch.maximum(new.abs().amax(), torch.tensor(1e-7)) / torch.tensor(127.0)
                    s = torch.maximum(s, before) if lo > 0 else s
                    inverse = 1.0 / s if torch.isfinite(s) else torch.tensor(0.0)

                    def made(y):
                        return torch.nan_to_num(torch.round(y * inverse).clamp(-127, 127), nan=0.0).to(torch.int8)

                    if lo > 0 and not torch.equal(s, before) and not (s.isnan() and before.isnan()):
                        codes[h, :lo] = made(codes[h, :lo].float() * before)
                    codes[h, lo:hi] = made(new)
                    scales[h] = s
    return [kc, vc, ks, vs], torch.tensor(after, dtype=torch.int32)


def sequence(pool, table, length, b):
    """fp64 (codes of keys and values [heads, length, d], their scales [heads, length], valid [length]) of a sequence."""
    kc, vc, ks, vs = pool
    length = min(max(length, 0), table.size(1) * PAGE)
    pages = table[b, :blocks(length)].long()
    valid = ((pages >= 0) & (pages < kc.size(0)))
    pages = torch.where(valid, pages, 0)
    k = kc[pages].permute(1, 0, 2, 3).reshape(kc.size(1), -1, kc.size(3))[:, :length].double()
    v = vc[pages].permute(1, 0, 3, 2).reshape(kc.size(1), -1, kc.size(3))[:, :length].double()
    each = [s[pages].t().repeat_interleave(PAGE, 1)[:, :length].double() for s in (ks, vs)]
    return k, v, *each, valid.repeat_interleave(PAGE)[:length]


def read(pool, table, lengths, max_length, layout, dtype, starts=None, key_mean=None):
    """kv_cache_read on the CPU."""
    pool, table = [t.cpu() for t in pool], table.cpu()
    heads, d = pool[0].size(1), pool[0].size(3)
    out = torch.zeros(2, len(lengths), heads, max_length, d, dtype=dtype)
    for b, length in enumerate(lengths.cpu().tolist()):
        k, v, ks, vs, valid = sequence(pool, table, length, b)
        start = 0 if starts is None else max(int(starts[b]), 0)
        k, v = ((x.float() * s.float()[..., None]) for x, s in ((k, ks), (v, vs)))
        if key_mean is not None:
            k[..., :key_mean.size(2)] += key_mean[b].cpu().float()[:, None]
        for i, x in enumerate((k, v)):
            x = torch.where(valid[:, None], x, 0.0)[:, start:start + max_length]
            out[i, b, :, :x.size(1)] = x.to(dtype)
    return hnd(out[0], layout), hnd(out[1], layout)


def attend(query, pool, table, lengths, layout, causal, sm_scale=None, query_scale=None, blkq=128, query_lengths=None):
    """kv_cache_attention in fp64: (out, bound of |kernel - out| by element), in the query's layout.

    The bound, from the arithmetic that the kernel's head describes: a float query's
    elements are off by half a unit of 16 bits; the exponent's factors by a few
    roundings of 32 bits, its constant by 2^-13; weights are rounded to fp16, 2^-11
    of them or, where they are small, 2^-25 of the largest; sums run in 32 bits; the
    result is rounded once."""
    q = hnd(query, layout)
    batch, hq, lq, d = q.shape
    heads = pool[0].size(1)
    width = pool[0].size(3)
    scale = d ** -0.5 if sm_scale is None else sm_scale
    out = torch.zeros(batch, hq, lq, d, dtype=torch.float64, device=q.device)
    bound = torch.zeros_like(out)
    half = HALF[torch.bfloat16 if query_scale is not None else query.dtype]
    for b, length in enumerate(lengths.tolist()):
        k, v, ks, vs, valid = sequence(pool, table, length, b)
        k, v = k[..., :d], v[..., :d]
        length = k.size(1)
        n = lq if query_lengths is None else min(max(int(query_lengths[b]), 0), lq)
        if n == 0 or length == 0:
            continue
        for h in range(hq):
            hk = h // (hq // heads)
            x = q[b, h, :n].double()
            if query_scale is not None:
                x = x * query_scale[b, h].double().repeat_interleave(blkq)[:n, None]
                off = torch.zeros(n, 1, dtype=torch.float64, device=q.device)
            else:
                off = x.abs().amax(1, keepdim=True) / 65024 * 1.0001
            s = (x @ k[hk].t()) * scale * ks[hk]
            seen = valid.expand(n, length)
            if causal:
                last = length - n + torch.arange(n, device=q.device)
                seen = seen & (torch.arange(length, device=q.device) <= last[:, None])
            some = seen.any(1)
            if not some.any():
                continue
            s, seen, off = s[some], seen[some], off[some]
            reach = s.abs().masked_fill(~seen, 0).amax(1, keepdim=True)
            # (natural units; the factors of the product, its rounding and the base's)
            e = off * k[hk].abs().sum(1) * scale * ks[hk] + 10 * 2.0 ** -24 * (reach + 1)
            e = e.masked_fill(~seen, 0).amax(1, keepdim=True) + 2 * math.log(2) * 2.0 ** -13
            p = s.masked_fill(~seen, -math.inf).softmax(1)
            values = v[hk] * vs[hk][:, None]
            out[b, h, :n][some] = p @ values
            size = p @ values.abs()
            w = p * vs[hk]
            top = w.amax(1, keepdim=True)
            step = torch.maximum(w * 2.0 ** -11, top * 2.0 ** -25).masked_fill(~seen, 0)
            bound[b, h, :n][some] = ((torch.expm1(2 * e) + 4 * (length + width) * 2.0 ** -24) * size + step @ v[hk].abs()) \
                * (1 + half) + half * (p @ values).abs()
    return hnd(out, layout), hnd(bound, layout)
