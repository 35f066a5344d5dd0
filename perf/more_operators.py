"""The measured operators of the key/value cache in 8 bits: what a DiT that makes a video chunk by chunk, or a served
prompt, keeps of its earlier tokens and attends to.

* ``write``: ``turing_sage.kv_cache_append``, which quantizes new keys and values into their pages (64 tokens with one
  scale a page and head), and ``turing_sage.kv_cache_read`` of what was written;
* ``read``: ``turing_sage.kv_cache_read``, the cached keys and values of whole sequences in 16 bits;
* ``attend``: ``turing_sage.kv_cache_attention``, attention over the cache, for single tokens and for chunks.

The package is an inference path, so there is no backward direction.  Where ``own`` is false, ``run`` computes the
same formulas with elementary torch operations.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
PAGE = 64  # tokens of a page
FLOOR = 1e-7  # least |x| a scale is made for
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def _package():
    """The framework, imported on the first call that needs it."""
    global _kernel
    if _kernel is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        "comfyui-turing-utils_amd"))
        import comfyui_turing_utils_kernel

        _kernel = comfyui_turing_utils_kernel
    return _kernel


_kernel = None


# ---------------------------------------------------------------------------
# The cases
# ---------------------------------------------------------------------------

def _write(b, hkv, d, new, held, dtype="bf16", layout="NHD", ragged=False, mean=False, codes=False):
    return {"kind": "write", "b": b, "hkv": hkv, "d": d, "new": new, "held": held, "dtype": dtype, "layout": layout,
            "ragged": ragged, "mean": mean, "codes": codes}


def _read(b, hkv, d, held, dtype="bf16", layout="NHD", ragged=False, mean=False):
    return {"kind": "read", "b": b, "hkv": hkv, "d": d, "held": held, "dtype": dtype, "layout": layout,
            "ragged": ragged, "mean": mean}


def _attend(b, hq, hkv, d, lq, held, dtype="bf16", layout="NHD", causal=False, ragged=False):
    return {"kind": "attend", "b": b, "hq": hq, "hkv": hkv, "d": d, "lq": lq, "held": held, "dtype": dtype,
            "layout": layout, "causal": causal, "ragged": ragged}


def listed():
    return [
        # A step of 32 served sequences of different lengths, grouped queries: one token each.
        dict(_write(32, 8, 128, 1, 8190, ragged=True), name="write_token"),
        # A latent frame of 30 x 52 tokens (Wan 1.3B) behind two others, two samples; the keys come as the codes of the
        # fused norm + rotation.
        dict(_write(2, 12, 128, 1560, 3121, ragged=True, codes=True), name="write_frame"),
        # The largest: all keys and values of a 480p video (Wan 14B).
        dict(_write(1, 40, 128, 32760, 0), name="write_32760"),
        # The text tokens of four prompts, head_dim 64, keys held without their mean, fp16.
        dict(_read(4, 12, 64, 513, dtype="f16", layout="HND", ragged=True, mean=True), name="read_text"),
        # A whole 480p video's keys and values (Wan 14B).
        dict(_read(1, 40, 128, 32760), name="read_32760"),
        # One query token a sequence, four sequences, grouped queries: latency.
        dict(_attend(4, 16, 4, 128, 1, 8190, ragged=True), name="attend_token"),
        # A step of 32 served sequences of different lengths.
        dict(_attend(32, 40, 8, 128, 1, 8190, ragged=True), name="attend_tokens_32"),
        # One token over the longest cache: four videos' tokens, no grouping.
        dict(_attend(1, 40, 40, 128, 1, 131040), name="attend_token_131040"),
        # A latent frame (Wan 1.3B) over the frames before it, queries as the codes of the fused norm + rotation.
        dict(_attend(1, 12, 12, 128, 1560, 9360, dtype="int8"), name="attend_frame"),
        # A prompt's tokens over themselves: causal, grouped, odd length.
        dict(_attend(2, 16, 4, 128, 4001, 4001, causal=True), name="attend_causal_4001"),
        # A padded batch of prompts behind cached ones, head_dim 64.
        dict(_attend(2, 9, 9, 64, 2050, 6000, layout="HND", causal=True, ragged=True), name="attend_padded_d64"),
        # The largest: three latent frames of a 480p video (Wan 14B) over all the video's tokens.
        dict(_attend(1, 40, 40, 128, 4680, 32760, dtype="int8"), name="attend_chunk_32760"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["write", "write", "read", "attend", "attend", "attend"])
    d, b, hkv, ragged = rng.choice([64, 128]), _log(rng, 1, 32), _log(rng, 1, 40), rng.random() < 0.5
    layout, mean, dtype = rng.choice(["HND", "NHD"]), rng.random() < 0.4, rng.choice(["bf16", "bf16", "f16"])
    if kind != "attend":
        tokens = max(1, 40 * 32760 * 128 // (b * hkv * d))
        if kind == "read":
            return _read(b, hkv, d, _log(rng, 1, min(32760, tokens)), dtype, layout, ragged, mean)
        codes = rng.random() < 0.3
        new = 1 if rng.random() < 0.3 else _log(rng, 2, 32760)
        new = min(new, tokens)
        held = 0 if rng.random() < 0.2 else _log(rng, 1, min(8190, tokens))
        return _write(b, hkv, d, new, held, dtype, layout, ragged, mean and not codes, codes)
    group = rng.choice([1, 1, 2, 4, 8])
    held = _log(rng, 2, 131040)
    short = rng.random()
    lq = 1 if short < 0.35 else rng.randint(2, 8) if short < 0.5 else _log(rng, 9, 4680)
    causal = rng.random() < 0.5
    lq = min(lq, held)
    while b * hkv * held * d > 40 * 131040 * 128:
        b, hkv = max(1, b // 2), hkv if b > 1 else max(1, hkv // 2)
    while b * hkv * group * lq * held * d > 40 * 4680 * 32760 * 128:
        lq = max(1, lq // 2)
    if dtype == "bf16" and rng.random() < 0.4:
        dtype = "int8"
    return _attend(b, hkv * group, hkv, d, lq, held, dtype, layout, causal, ragged)


def _lengths(case, length):
    """The sequences' lengths: equal, or from a third of the longest on."""
    b = case["b"]
    return [max(min(1, length), length * (b + 2 * i + 1) // (3 * b)) if case["ragged"] and i + 1 < b else length
            for i in range(b)]


def _queries(case):
    """The sequences' query tokens: not more than they hold."""
    return [min(n, held) for n, held in zip(_lengths(case, case["lq"]), _lengths(case, case["held"]))]


def _spans(case):
    """Of a write: (tokens held, new ones, tokens in front of them in their page) of each sequence."""
    return [(held, new, held % PAGE) for held, new in zip(_lengths(case, case["held"]), _lengths(case, case["new"]))]


def work(case):
    b, hkv, d = case["b"], case["hkv"], case["d"]
    row = hkv * d
    if case["kind"] == "write":
        moved = back = 0
        for _, new, front in _spans(case):
            back += front + new
            moved += new * row * (3 if case["codes"] else 4) + 2 * new * row
        pages = back // PAGE + b
        if case["codes"]:
            moved += 4 * hkv * pages
        if case["mean"]:
            moved += 2 * b * row
        # written, and read back with the tokens in front of the new ones
        return {"bytes": moved + 8 * hkv * pages + back * row * 6, "flops": row * (12 * back)}
    held = sum(_lengths(case, case["held"]))
    if case["kind"] == "read":
        return {"bytes": held * row * 6 + 8 * hkv * (held // PAGE + b) + (2 * b * row if case["mean"] else 0),
                "flops": 4 * held * row}
    pairs = 0
    for n, length in zip(_queries(case), _lengths(case, case["held"])):
        pairs += n * length - (n * (n - 1) // 2 if case["causal"] else 0)
    rows = case["hq"] * sum(_queries(case))
    size = 1 if case["dtype"] == "int8" else 2
    return {"bytes": 2 * held * row + 8 * hkv * (held // PAGE + b) + rows * d * (size + 2) + 4 * b * (held // PAGE // b),
            "flops": 4 * case["hq"] * d * pairs}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _rows(g, b, heads, length, d, offset, spread):
    """fp32 rows [b, heads, length, d] that resemble their neighbours', as a video's tokens do: noise on slow waves,
    around an offset of each channel."""
    t = torch.arange(length, device=DEVICE, dtype=torch.float32)[:, None] / 640.0
    f = torch.arange(1, 5, device=DEVICE, dtype=torch.float32)[None, :]
    slow = torch.matmul(torch.sin(t * f + f * f), 0.4 * torch.randn(b, heads, 4, d, generator=g, device=DEVICE))
    x = torch.randn(b, heads, length, d, generator=g, device=DEVICE).add_(slow)
    return x.add_(offset * torch.randn(b, heads, 1, d, generator=g, device=DEVICE)).mul_(spread)


def _block_codes(x, block):
    """(codes, scales) of x [b, h, l, d] with one scale for `block` tokens."""
    b, h, l, d = x.shape
    n = (l + block - 1) // block
    blocks = torch.nn.functional.pad(x, (0, 0, 0, n * block - l)).view(b, h, n, block, d)
    scale = blocks.abs().amax((3, 4)).clamp_min(FLOOR) / 127.0
    codes = torch.round(blocks * (1.0 / scale)[..., None, None]).clamp_(-127, 127).to(torch.int8)
    return codes, scale


def _cache(g, case, held, capacity):
    """A pool whose pages are handed out in no order, with `held` tokens of each sequence."""
    b, hkv, d = case["b"], case["hkv"], case["d"]
    n = max(1, (capacity + PAGE - 1) // PAGE)
    table = torch.randperm(b * n, generator=g, device=DEVICE).view(b, n)
    pages = b * n + 1  # (the last one is in no table)
    state = {"key_codes": torch.zeros(pages, hkv, PAGE, d, dtype=torch.int8, device=DEVICE),
             "value_codes": torch.zeros(pages, hkv, d, PAGE, dtype=torch.int8, device=DEVICE),
             "key_scale": torch.ones(pages, hkv, device=DEVICE), "value_scale": torch.ones(pages, hkv, device=DEVICE)}
    blocks = (max(held) + PAGE - 1) // PAGE
    if blocks:
        at = table[:, :blocks].reshape(-1)
        for name, offset in (("key", 1.0), ("value", 0.3)):
            codes, scale = _block_codes(_rows(g, b, hkv, max(held), d, offset, 1.0), PAGE)
            codes = codes.transpose(1, 2).reshape(b * blocks, hkv, PAGE, d)
            state[name + "_codes"][at] = codes if name == "key" else codes.transpose(2, 3)
            state[name + "_scale"][at] = scale.transpose(1, 2).reshape(b * blocks, hkv)
    return state, table.to(torch.int32)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    kind, b, hkv, d, nhd = case["kind"], case["b"], case["hkv"], case["d"], case["layout"] == "NHD"
    held = _lengths(case, case["held"])
    new = _lengths(case, case["new"]) if kind == "write" else [0] * b
    pool, table = _cache(g, case, held, max(x + y for x, y in zip(held, new)))
    laid = (lambda x: x.transpose(1, 2).contiguous()) if nhd else (lambda x: x)
    state = {"case": case, "pool": pool, "table": table, "lengths": _ints(held)}
    if case.get("mean"):
        state["mean"] = torch.randn(b, hkv, d, generator=g, device=DEVICE).to(torch.bfloat16)
    if kind == "write":
        key, value = (_rows(g, b, hkv, case["new"], d, offset, 1.1) for offset in (1.0, 0.3))
        state["value"] = laid(value.to(TYPES[case["dtype"]]))
        if case["codes"]:
            codes, state["key_scale"] = _block_codes(key, PAGE)
            state["key"] = laid(codes.flatten(2, 3)[:, :, :case["new"]].contiguous())
        else:
            state["key"] = laid(key.to(TYPES[case["dtype"]]))
        state["new"] = _ints(new) if case["ragged"] else None
        spans = _spans(case)
        state["starts"] = _ints([x - front for x, _, front in spans])
        state["back"] = max(front + n for _, n, front in spans)
    elif kind == "attend":
        query = _rows(g, b, case["hq"], case["lq"], d, 0.3, 1.0)
        if case["dtype"] == "int8":
            codes, state["query_scale"] = _block_codes(query, 16)
            state["query"] = laid(codes.flatten(2, 3)[:, :, :case["lq"]].contiguous())
        else:
            state["query"] = laid(query.to(TYPES[case["dtype"]]))
        state["queries"] = _ints(_queries(case)) if case["ragged"] else None
    return state


# ---------------------------------------------------------------------------
# The passes
# ---------------------------------------------------------------------------

def run(state):
    case = state["case"]
    kind, layout, mean = case["kind"], case["layout"], state.get("mean")
    if own:
        sage = _package().turing_sage
        cache = sage.QuantizedKVCache(**state["pool"])
        at = (cache, state["table"], state["lengths"])
        if kind == "attend":
            return sage.kv_cache_attention(state["query"], *at, tensor_layout=layout, is_causal=case["causal"],
                                           query_scale=state.get("query_scale"), blkq=16,
                                           query_lengths=state["queries"])
        if kind == "read":
            return sage.kv_cache_read(*at, max_length=case["held"], tensor_layout=layout, dtype=TYPES[case["dtype"]],
                                      key_mean=mean)
        after = sage.kv_cache_append(state["key"], state["value"], *at, tensor_layout=layout,
                                     new_lengths=state["new"], key_scale=state.get("key_scale"), key_mean=mean)
        return (after, *sage.kv_cache_read(cache, state["table"], after, starts=state["starts"],
                                           max_length=state["back"], tensor_layout=layout,
                                           dtype=state["value"].dtype, key_mean=mean))
    if kind == "attend":
        return _plain_attend(state)
    if kind == "read":
        return _plain_read(state, state["lengths"], None, case["held"], TYPES[case["dtype"]])
    after = _plain_write(state)
    return (after, *_plain_read(state, after, state["starts"], state["back"], state["value"].dtype))


def _hnd(x, layout):
    return x if layout == "HND" else x.transpose(1, 2)


def _paged(pool, name, pages):
    """fp32 values [b, h, tokens, d] of the pages [b, n] of a pool."""
    codes, scale = pool[name + "_codes"][pages], pool[name + "_scale"][pages]
    codes = codes if name == "key" else codes.transpose(3, 4)
    x = codes.float() * scale[..., None, None]
    return x.permute(0, 2, 1, 3, 4).flatten(2, 3)


def _plain_write(state):
    case, pool = state["case"], state["pool"]
    b, new = case["b"], case["new"]
    device = state["table"].device
    held = state["lengths"].long()
    count = torch.full_like(held, new) if state["new"] is None else state["new"].long()
    n = (new + 2 * PAGE - 2) // PAGE  # pages that so many tokens can touch
    front = held % PAGE
    slot = torch.arange(n * PAGE, device=device)
    token = slot - front[:, None]  # [b, n * PAGE]
    fresh = (token >= 0) & (token < count[:, None])
    block = held[:, None] // PAGE + torch.arange(n, device=device)
    spare = pool["key_codes"].size(0) - 1
    used = fresh.view(b, n, PAGE).any(-1)
    pages = torch.where(used, state["table"].long().gather(1, block.clamp_max(state["table"].size(1) - 1)), spare)
    earlier = (slot < front[:, None]).view(b, n, 1, PAGE, 1)
    fresh = fresh.view(b, n, 1, PAGE, 1)
    for name in ("key", "value"):
        x = _hnd(state[name], case["layout"]).float()
        if name == "key" and "key_scale" in state:
            x = x * state["key_scale"].repeat_interleave(PAGE, 2)[:, :, :new, None]
        if name == "key" and "mean" in state:
            x = x - state["mean"].float()[:, :, None]
        at = token.clamp(0, new - 1)[:, None, :, None].expand(b, x.size(1), n * PAGE, x.size(3))
        x = x.gather(2, at).unflatten(2, (n, PAGE)).transpose(1, 2)  # [b, n, h, PAGE, d]
        codes = pool[name + "_codes"][pages]
        codes = codes if name == "key" else codes.transpose(3, 4)
        before = torch.where(earlier.any(3)[..., 0], pool[name + "_scale"][pages], 0.0)
        scale = torch.maximum(before, (x * fresh).abs().amax((3, 4)).clamp_min(FLOOR) / 127.0)
        x = torch.where(earlier, codes.float() * before[..., None, None], x)
        made = torch.round(x * (1.0 / scale)[..., None, None]).clamp_(-127, 127).to(torch.int8)
        codes = torch.where(fresh | earlier, made, codes)
        pool[name + "_codes"][pages] = codes if name == "key" else codes.transpose(3, 4)
        pool[name + "_scale"][pages] = scale
    return state["lengths"] + count.to(torch.int32)


def _plain_read(state, lengths, starts, length, dtype):
    case, pool, table = state["case"], state["pool"], state["table"].long()
    device = table.device
    starts = torch.zeros_like(lengths) if starts is None else starts
    position = starts[:, None].long() + torch.arange(length, device=device)  # [b, length]
    inside = (position < lengths[:, None])[:, None, :, None]
    first = starts.long() // PAGE
    n = (length + 2 * PAGE - 2) // PAGE
    block = (first[:, None] + torch.arange(n, device=device)).clamp_max(table.size(1) - 1)
    at = (position - first[:, None] * PAGE).clamp_max(n * PAGE - 1)[:, None, :, None]
    out = []
    for name in ("key", "value"):
        x = _paged(pool, name, table.gather(1, block))
        x = x.gather(2, at.expand(-1, x.size(1), -1, x.size(3)))
        if name == "key" and "mean" in state:
            x = x + state["mean"].float()[:, :, None]
        out.append(_hnd(torch.where(inside, x, 0.0).to(dtype), case["layout"]).contiguous())
    return tuple(out)


def _plain_attend(state):
    case, pool, table = state["case"], state["pool"], state["table"].long()
    b, hq, hkv, d, lq = (case[x] for x in ("b", "hq", "hkv", "d", "lq"))
    q = _hnd(state["query"], case["layout"]).float()
    if "query_scale" in state:
        q = q * state["query_scale"].repeat_interleave(16, 2)[:, :, :lq, None]
    k, v = _paged(pool, "key", table), _paged(pool, "value", table)
    lengths = state["lengths"].long()
    count = torch.full_like(lengths, lq) if state["queries"] is None else state["queries"].long()
    row = torch.arange(lq, device=q.device)
    key = torch.arange(k.size(2), device=q.device)
    last = (lengths - count)[:, None] + row if case["causal"] else lengths[:, None].expand(b, lq) - 1
    last = torch.where(row < count[:, None], last, -1)
    seen = (key <= last[..., None])[:, None, None]  # [b, 1, 1, lq, keys]
    q = (q * d ** -0.5).reshape(b, hkv, hq // hkv * lq, d)
    s = torch.matmul(q, k.transpose(-1, -2).contiguous()).unflatten(2, (hq // hkv, lq))
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True).clamp_min(1e-30)
    o = torch.matmul(s.flatten(2, 3), v).unflatten(2, (hq // hkv, lq)) / total
    dtype = TYPES.get(case["dtype"], torch.bfloat16)
    return _hnd(o.flatten(1, 2).to(dtype), case["layout"]).contiguous()


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def _sequence(state, i, pages):
    """fp64 keys and values [h, tokens, d] of a sequence's first `pages` pages."""
    at, pool = state["table"][i, :pages].long(), state["pool"]
    k = pool["key_codes"][at].double() * pool["key_scale"][at].double()[..., None, None]
    v = pool["value_codes"][at].double() * pool["value_scale"][at].double()[..., None, None]
    return (k.permute(1, 0, 2, 3).reshape(k.size(1), -1, k.size(3)),
            v.permute(1, 0, 3, 2).reshape(v.size(1), -1, v.size(2)))


def exact(case, seed):
    state = prepare(case, seed)
    nhd = case["layout"] == "NHD"
    held = _lengths(case, case["held"])
    if case["kind"] == "attend":
        b, hq, hkv, lq, d = (case[x] for x in ("b", "hq", "hkv", "lq", "d"))
        q = (state["query"].transpose(1, 2) if nhd else state["query"]).double()
        if "query_scale" in state:
            q = q * state["query_scale"].double()[:, :, torch.arange(lq, device=DEVICE) // 16, None]
        out = torch.zeros(b, hq, lq, d, dtype=torch.float64, device=DEVICE)
        for i, (n, length) in enumerate(zip(_queries(case), held)):
            k, v = _sequence(state, i, (length + PAGE - 1) // PAGE)
            for h in range(hq):
                kv = h // (hq // hkv)
                s = (q[i, h, :n] @ k[kv, :length].t()) / math.sqrt(d)
                if case["causal"]:
                    s.masked_fill_(torch.ones_like(s, dtype=torch.bool).triu_(length - n + 1), -math.inf)
                out[i, h, :n] = s.softmax(1) @ v[kv, :length]
        return out.transpose(1, 2) if nhd else out
    if case["kind"] == "read":
        ends, starts, length = held, [0] * case["b"], case["held"]
    else:
        ends = [x + n for x, n, _ in _spans(case)]
        starts, length = [x - front for x, _, front in _spans(case)], state["back"]
    keys = torch.zeros(case["b"], case["hkv"], length, case["d"], dtype=torch.float64, device=DEVICE)
    values = torch.zeros_like(keys)
    for i, (start, end) in enumerate(zip(starts, ends)):
        if case["kind"] == "read":
            k, v = _sequence(state, i, (end + PAGE - 1) // PAGE)
            k, v = k[:, :end], v[:, :end]
        else:
            k, v = _written(state, case, i, held[i], end - held[i])
        if "mean" in state:
            k = k + state["mean"][i].double()[:, None]
        keys[i, :, :end - start], values[i, :, :end - start] = k, v
    out = [x.transpose(1, 2) if nhd else x for x in (keys, values)]
    return tuple(out) if case["kind"] == "read" else (None, *out)


def _written(state, case, i, held, new):
    """What the pages that a sequence's new tokens touch hold afterwards, from their first token on, page by page."""
    front, result = held % PAGE, []
    for name in ("key", "value"):
        x = (state[name].transpose(1, 2) if case["layout"] == "NHD" else state[name])[i, :, :new].double()
        if name == "key" and "key_scale" in state:
            x = x * state["key_scale"][i].double()[:, torch.arange(new, device=DEVICE) // PAGE, None]
        if name == "key" and "mean" in state:
            x = x - state["mean"][i].double()[:, None]
        page = int(state["table"][i, held // PAGE]) if front else 0
        codes = state["pool"][name + "_codes"][page].double()
        codes = (codes if name == "key" else codes.transpose(1, 2))[:, :front]
        before = state["pool"][name + "_scale"][page].double()
        x = torch.cat([codes * before[:, None, None], x], 1)
        pages = []
        for at in range(0, front + new, PAGE):
            part = x[:, at:at + PAGE]
            fresh = part[:, front:] if at == 0 else part
            scale = fresh.abs().amax((1, 2)).clamp_min(FLOOR) / 127
            if at == 0 and front:
                scale = torch.maximum(scale, before)
            scale = scale.float().double()[:, None, None]  # (a scale is held in 32 bits)
            pages.append((part / scale).round().clamp(-127, 127) * scale)
        result.append(torch.cat(pages, 1))
    return result
