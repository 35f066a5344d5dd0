"""The measured operators: what a DiT that serves many requests runs beside its dense attention and plain linears.

* ``select``: ``turing_sage.select_key_blocks``, which key blocks of 64 each query block of 128 attends to, by the
  product of the blocks' mean rows;
* ``attend``: ``turing_sage.key_block_attention``, the Sage attention over the selected key blocks alone;
* ``adapters``: ``turing_int8_linear_adapters``, the W8A8 projection with each request's own low-rank adapter.

The package is an inference path, so there is no backward direction.  Where ``own`` is false, ``run`` computes the
same formulas with elementary torch operations.
"""
import math
import os
import sys

import torch

own = False

DEVICE = "cuda"
QB, KB = 128, 64  # rows of a query block, keys of a key block


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

def _attention(kind, b, hq, hkv, lq, lk, d, keep, layout="HND", causal=False, blkq=128, blkk=128, sink=0, local=0,
               ragged=False):
    return {"kind": kind, "b": b, "hq": hq, "hkv": hkv, "lq": lq, "lk": lk, "d": d, "keep": keep, "layout": layout,
            "causal": causal, "blkq": blkq, "blkk": blkk, "sink": sink, "local": local, "ragged": ragged}


def _adapters(m, k, n, rank, count, rows=1, bias=True, residual=False, gate=False):
    return {"kind": "adapters", "m": m, "k": k, "n": n, "rank": rank, "count": count, "rows": rows, "bias": bias,
            "residual": residual, "gate": gate}


def listed():
    return [
        # A short prompt's blocks, grouped queries, head_dim 64: launches and latency only.
        dict(_attention("select", 2, 8, 2, 300, 300, 64, 2, layout="NHD"), name="select_short"),
        # Causal selection with the first block and the diagonal always kept, odd length, as a causal video model does.
        dict(_attention("select", 2, 16, 4, 4001, 4001, 128, 16, causal=True, blkq=16, blkk=64, sink=1, local=1),
             name="select_causal_4001"),
        # A whole 480p video (Wan 14B): 256 query blocks by 512 key blocks, a quarter of them kept.
        dict(_attention("select", 1, 40, 40, 32760, 32760, 128, 128, layout="NHD", blkq=16, blkk=64),
             name="select_32760"),
        # One query token per sample over a longer context, grouped queries: latency.
        dict(_attention("attend", 4, 16, 4, 1, 8190, 128, 32, blkq=16, blkk=64), name="attend_token"),
        # Wan 1.3B at 480p with a quarter of the keys.
        dict(_attention("attend", 1, 12, 12, 8190, 8190, 128, 32, local=1), name="attend_8190"),
        # Causal grouped-query attention at an odd length, the layout ComfyUI hands over.
        dict(_attention("attend", 2, 16, 4, 4001, 4001, 128, 16, layout="NHD", causal=True, blkq=16, blkk=64, sink=1,
                        local=1), name="attend_causal_4001"),
        # A padded batch, head_dim 64: samples of different lengths with rubbish behind their last rows.
        dict(_attention("attend", 2, 9, 9, 6000, 6000, 64, 24, ragged=True), name="attend_padded_d64"),
        # The largest: the self-attention of a whole 480p video (Wan 14B) over a fifth of the keys.
        dict(_attention("attend", 1, 40, 40, 32760, 32760, 128, 102, layout="NHD", blkq=16, blkk=64),
             name="attend_32760"),
        # The time projection of four prompts, each request with an adapter of its own: four rows.
        dict(_adapters(4, 1536, 9216, 16, 4), name="adapters_rows"),
        # Many single rows with different adapters, some without one, an odd rank.
        dict(_adapters(61, 5120, 5120, 24, 16), name="adapters_61_mixed"),
        # The fused k / v projection of four prompts' text tokens, one adapter a prompt.
        dict(_adapters(2050, 5120, 10240, 64, 3, rows=513), name="adapters_text"),
        # The largest: the output projection of a whole video with the block's gated residual, two requests.
        dict(_adapters(32760, 5120, 5120, 32, 2, rows=16380, residual=True, gate=True), name="adapters_32760"),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["select", "attend", "attend", "adapters", "adapters"])
    if kind == "adapters":
        m = _log(rng, 1, 16384)
        rows = rng.choice([1, 1, _log(rng, 2, max(2, m))])
        groups = (m + rows - 1) // rows
        k, n = 16 * _log(rng, 8, 864), 8 * _log(rng, 16, 1280)
        while 2 * m * k * n > 2 * 32760 * 5120 * 5120:
            m = max(1, m // 2)
        return _adapters(m, k, n, 8 * rng.randint(1, 12), min(32, max(1, min(groups, _log(rng, 1, 32)))), rows,
                         bias=rng.random() < 0.7, residual=rng.random() < 0.4, gate=rng.random() < 0.5)
    d = rng.choice([64, 128])
    b, hkv, group = rng.randint(1, 3), rng.randint(1, 10), rng.choice([1, 1, 2, 4])
    lk = _log(rng, 64, 32760)
    lq = 1 if kind == "attend" and rng.random() < 0.2 else lk if rng.random() < 0.7 else _log(rng, 2, 32760)
    blocks = (lk + KB - 1) // KB
    keep = max(1, min(102, int(blocks * rng.uniform(0.05, 0.5))))
    while b * hkv * group * max(lq, lk) > 40 * 32760:
        hkv = max(1, hkv // 2)
        b = 1
    while kind == "attend" and b * hkv * group * lq * keep > 40 * 32760 * 102:
        keep = max(1, keep // 2)
    blkq, blkk = rng.choice([(16, 64), (128, 128)])
    return _attention(kind, b, hkv * group, hkv, lq, lk, d, keep, rng.choice(["HND", "NHD"]),
                      causal=lq == lk and rng.random() < 0.35, blkq=blkq, blkk=blkk, sink=rng.randint(0, 1),
                      local=rng.randint(0, 2), ragged=rng.random() < 0.3)


def _lengths(case, length):
    """The samples' lengths of a padded batch."""
    return [max(1, length * (case["b"] + 1 - i) // (case["b"] + 1)) if case["ragged"] else length
            for i in range(case["b"])]


def _blocks_of(case):
    """(query blocks, key blocks, per sample: rows and visible keys' blocks of each query block)."""
    nqb, nkb = (case["lq"] + QB - 1) // QB, (case["lk"] + KB - 1) // KB
    seen = []
    for ql, kl in zip(_lengths(case, case["lq"]), _lengths(case, case["lk"])):
        for i in range((ql + QB - 1) // QB):
            rows = min(QB, ql - i * QB)
            visible = (min(kl, i * QB + rows) if case["causal"] else kl) + KB - 1
            seen.append((rows, visible // KB))
    return nqb, nkb, seen


def work(case):
    if case["kind"] == "adapters":
        m, k, n, r = case["m"], case["k"], case["n"], case["rank"]
        used = min(case["count"], (m + case["rows"] - 1) // case["rows"])
        moved = m * k + n * k + 4 * m + 4 * n * (2 if case["bias"] else 1) + 2 * used * r * (k + n) + 2 * m * n
        if case["residual"]:
            moved += 2 * m * n + (2 * n * ((m + case["rows"] - 1) // case["rows"]) if case["gate"] else 0)
        return {"bytes": moved, "flops": 2 * m * n * k + 2 * m * r * (k + n)}
    b, hq, hkv, lq, lk, d = (case[x] for x in ("b", "hq", "hkv", "lq", "lk", "d"))
    nqb, nkb, seen = _blocks_of(case)
    width = min(case["keep"], nkb)
    index = 4 * b * hq * nqb * width
    queries = hq * (d * sum(_lengths(case, lq)) + 4 * b * ((lq + case["blkq"] - 1) // case["blkq"]))
    codes = hkv * (d * sum(_lengths(case, lk)) + 4 * b * ((lk + case["blkk"] - 1) // case["blkk"]))
    if case["kind"] == "select":
        return {"bytes": queries + codes + index,
                "flops": hq * sum(2 * d * visible for _, visible in seen)
                + d * (hq * sum(_lengths(case, lq)) + hkv * sum(_lengths(case, lk)))}
    # key and value blocks that no list can name are not read
    share = min(1.0, sum(min(case["keep"], visible) for _, visible in seen) * (hq // hkv)
                / max(1, sum(_lengths(case, lk)) / KB))
    return {"bytes": queries + index + share * 3 * codes + 2 * b * hq * lq * d,
            "flops": 4 * hq * d * sum(rows * KB * min(case["keep"], visible) for rows, visible in seen)}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _rows(g, b, heads, group, length, d, coefficients):
    """bf16 rows [b, heads, length, d] that resemble their neighbours', as a video's tokens do: noise on slow waves
    whose amplitudes queries and keys of a head share."""
    t = torch.arange(length, device=DEVICE, dtype=torch.float32)[:, None] / 640.0
    f = torch.arange(1, coefficients.size(2) + 1, device=DEVICE, dtype=torch.float32)[None, :]
    waves = torch.sin(t * f + f * f)  # [length, waves]
    slow = torch.matmul(waves, coefficients.repeat_interleave(group, 1))  # [b, heads, length, d]
    return (torch.randn(b, heads, length, d, generator=g, device=DEVICE) + slow).to(torch.bfloat16)


def _codes(x, block, mean=None):
    """(int8 codes, fp32 scales) of x [b, h, l, d] per block of tokens, as the Sage prologue makes them."""
    b, h, l, d = x.shape
    x = x.float() if mean is None else x.float() - mean
    n = (l + block - 1) // block
    padded = torch.nn.functional.pad(x, (0, 0, 0, n * block - l)).view(b, h, n, block * d)
    amax = padded.abs().amax(-1).clamp_min(1e-7)
    q = torch.round(padded * (127.0 / amax)[..., None]).clamp_(-127, 127).to(torch.int8)
    return q.view(b, h, n * block, d)[:, :, :l].contiguous(), amax / 127.0


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    if case["kind"] == "adapters":
        m, k, n, r, count = case["m"], case["k"], case["n"], case["rank"], case["count"]
        groups = (m + case["rows"] - 1) // case["rows"]
        # codes of rotated rows are near normal with 127 at a row's largest value
        act = torch.randn(m, k, generator=g, device=DEVICE).mul_(30).round_().clamp_(-127, 127).to(torch.int8)
        weight = torch.randn(n, k, generator=g, device=DEVICE).mul_(30).round_().clamp_(-127, 127).to(torch.int8)
        state = {"activation": act, "weight": weight,
                 "activation_scale": 0.02 + 0.03 * torch.rand(m, 1, generator=g, device=DEVICE),
                 "weight_scale": (0.5 + torch.rand(n, generator=g, device=DEVICE)) * 0.02 / 30,
                 "bias": torch.randn(n, generator=g, device=DEVICE) * 0.02 if case["bias"] else None,
                 "down": (torch.randn(count, r, k, generator=g, device=DEVICE) * k ** -0.5).to(torch.bfloat16),
                 "up": (torch.randn(count, n, r, generator=g, device=DEVICE) * 0.05).to(torch.bfloat16),
                 "scaling": 0.5 + torch.rand(count, generator=g, device=DEVICE),
                 # one request in eight carries no adapter
                 "adapter_ids": torch.where(torch.rand(groups, generator=g, device=DEVICE) < 0.125, -1,
                                            torch.randint(0, count, (groups,), generator=g, device=DEVICE)
                                            ).to(torch.int32),
                 "adapter_rows": case["rows"], "residual": None, "gate": None, "gate_rows": 1}
        if case["residual"]:
            state["residual"] = torch.randn(m, n, generator=g, device=DEVICE).to(torch.bfloat16)
            if case["gate"]:
                state["gate"] = (torch.randn(groups, n, generator=g, device=DEVICE) * 0.5).to(torch.bfloat16)
                state["gate_rows"] = case["rows"]
        return {"case": case, "args": state}
    b, hq, hkv, lq, lk, d = (case[x] for x in ("b", "hq", "hkv", "lq", "lk", "d"))
    coefficients = torch.randn(b, hkv, 6, d, generator=g, device=DEVICE) * 0.4
    q = _rows(g, b, hq, hq // hkv, lq, d, coefficients)
    k = _rows(g, b, hkv, 1, lk, d, coefficients)
    k = k + 2 * torch.randn(b, hkv, 1, d, generator=g, device=DEVICE).to(torch.bfloat16)
    q8, qs = _codes(q, case["blkq"])
    k8, ks = _codes(k, case["blkk"], k.float().mean(2, keepdim=True))
    ql = kl = None
    if case["ragged"]:
        ql, kl = (torch.tensor(_lengths(case, n), dtype=torch.int32, device=DEVICE) for n in (lq, lk))
    state = {"query_int8": q8, "query_scale": qs, "key_int8": k8, "key_scale": ks,
             "tensor_layout": case["layout"], "is_causal": case["causal"], "blkq": case["blkq"],
             "blkk": case["blkk"], "query_lengths": ql, "key_lengths": kl}
    choice = {"keep": case["keep"], "sink_blocks": case["sink"], "local_blocks": case["local"]}
    if case["kind"] == "attend":
        index = _select(dict(state, tensor_layout="HND", **choice))
        v = torch.randn(b, hkv, d, (lk + KB - 1) // KB * KB, generator=g, device=DEVICE)
        v += torch.randn(b, hkv, d, 1, generator=g, device=DEVICE) * 0.5
        v = v.to(torch.bfloat16)
        v[..., lk:] = 0
        if case["ragged"]:  # what stands behind a sample's last key is rubbish
            v.masked_fill_(torch.arange(v.size(-1), device=DEVICE) >= kl[:, None, None, None].long(), float("nan"))
        state.update(value_t=v, block_index=index, sm_scale=d ** -0.5)
    else:
        state.update(choice)
    if case["layout"] == "NHD":
        for x in ("query_int8", "key_int8"):
            state[x] = state[x].transpose(1, 2).contiguous()
    return {"case": case, "args": state}


# ---------------------------------------------------------------------------
# The passes
# ---------------------------------------------------------------------------

def run(state):
    kind, args = state["case"]["kind"], state["args"]
    if own:
        kernel = _package()
        if kind == "adapters":
            return kernel.turing_int8_linear_adapters(**args)
        call = kernel.turing_sage.select_key_blocks if kind == "select" else kernel.turing_sage.key_block_attention
        return call(**args)
    return {"select": _select, "attend": _attend, "adapters": _linear}[kind](args)


def _heads_first(a):
    q8, k8 = a["query_int8"], a["key_int8"]
    return (q8, k8) if a["tensor_layout"] == "HND" else (q8.transpose(1, 2), k8.transpose(1, 2))


def _ends(a, lq, lk, batch, device):
    """The samples' lengths as [batch, 1, 1, 1]."""
    given = [a["query_lengths"], a["key_lengths"]]
    full = [torch.full((batch,), n, device=device) if x is None else x.long().clamp(0, n)
            for x, n in zip(given, (lq, lk))]
    return [x.view(batch, 1, 1, 1) for x in full]


def _means(codes, scale, group, block, ends):
    """fp64 mean rows [b, h, blocks, d] of the blocks' tokens in front of the sample's end."""
    b, h, l, d = codes.shape
    n = (l + block - 1) // block
    rows = scale.double().repeat_interleave(group, 2)[:, :, :l, None] * codes
    rows = rows * (torch.arange(l, device=codes.device)[:, None] < ends)
    sums = torch.nn.functional.pad(rows, (0, 0, 0, n * block - l)).view(b, h, n, block, d).sum(3)
    count = (ends - torch.arange(n, device=codes.device)[:, None] * block).clamp(0, block)
    return sums / count.clamp_min(1)


def _select(a):
    q8, k8 = _heads_first(a)
    (b, hq, lq, _), (_, hkv, lk, _) = q8.shape, k8.shape
    ql, kl = _ends(a, lq, lk, b, q8.device)
    mq = _means(q8, a["query_scale"], a["blkq"], QB, ql)
    mk = _means(k8, a["key_scale"], a["blkk"], KB, kl).repeat_interleave(hq // hkv, 1)
    # 64 bits: a choice between two near scores is a whole number, right or wrong
    score = torch.matmul(mq, mk.transpose(-1, -2).contiguous())
    nqb, nkb = score.shape[-2:]
    i = torch.arange(nqb, device=q8.device)[:, None]
    j = torch.arange(nkb, device=q8.device)[None, :]
    near = (j >= 2 * i - (a["local_blocks"] - 1)) & (j <= 2 * i + a["local_blocks"])
    forced = (j < a["sink_blocks"]) | (near & (a["local_blocks"] > 0))
    visible = (i * QB < ql) & (j * KB < kl)
    if a["is_causal"]:
        visible = visible & (j * KB < torch.minimum((i + 1) * QB, ql))
    score = score.masked_fill(forced, math.inf).masked_fill(~visible, -math.inf)
    width = min(a["keep"], nkb)
    order = torch.sort(score, dim=-1, descending=True, stable=True).indices[..., :width]
    order = torch.where(visible.expand_as(score).gather(-1, order), order, nkb).sort(-1).values
    return torch.where(order < nkb, order, -1).to(torch.int32)


def _attend(a):
    q8, k8 = _heads_first(a)
    (b, hq, lq, d), (_, hkv, lk, _) = q8.shape, k8.shape
    ql, kl = _ends(a, lq, lk, b, q8.device)
    index = a["block_index"].long()
    nqb, width = index.shape[2:]
    nkb = (lk + KB - 1) // KB
    pad = torch.nn.functional.pad
    qf = pad(q8.float(), (0, 0, 0, nqb * QB - lq)).reshape(b * hq, nqb, QB, d)
    row_scale = pad(a["query_scale"].repeat_interleave(a["blkq"], 2)[:, :, :lq], (0, nqb * QB - lq))
    row_scale = (row_scale * a["sm_scale"]).view(b * hq, nqb, QB, 1)
    kf = pad(k8.float(), (0, 0, 0, nkb * KB - lk)).reshape(b * hkv * nkb, KB, d)
    key_scale = pad(a["key_scale"].repeat_interleave(a["blkk"], 2)[:, :, :lk], (0, nkb * KB - lk))
    key_scale = key_scale.reshape(b * hkv * nkb, KB)
    key = torch.arange(nkb * KB, device=q8.device)
    vf = a["value_t"].float().masked_fill(key >= kl, 0).transpose(2, 3).reshape(b * hkv * nkb, KB, d)
    row = torch.arange(nqb * QB, device=q8.device).view(nqb, QB, 1)
    before = torch.cummax(pad(index, (1, 0), value=-1), -1).values[..., :-1]
    valid = ((index > before) & (index < nkb)).view(b * hq, nqb, width, 1)
    index = index.clamp(0, nkb - 1).view(b * hq, nqb, width)
    base = (torch.arange(b, device=q8.device)[:, None] * hkv
            + torch.arange(hq, device=q8.device) // (hq // hkv)).view(b * hq, 1, 1) * nkb
    key_end = kl.expand(b, hq, 1, 1).reshape(b * hq, 1, 1, 1)
    row_end = ql.expand(b, hq, 1, 1).reshape(b * hq, 1, 1, 1)
    out = torch.empty(b * hq, nqb, QB, d, dtype=torch.bfloat16, device=q8.device)
    # the gathered keys of all heads together can pass the card's memory: some heads at a time
    step = max(1, int(2 ** 31 / (nqb * width * KB * (2 * d + 2 * QB))))
    for c in range(0, b * hq, step):
        heads = slice(c, c + step)
        at = (base[heads] + index[heads])
        s = torch.matmul(qf[heads], kf[at].flatten(2, 3).transpose(-1, -2).contiguous())
        s = s * row_scale[heads] * key_scale[at].flatten(2, 3)[:, :, None]
        where = index[heads][..., None] * KB + torch.arange(KB, device=q8.device)
        seen = (valid[heads] & (where < key_end[heads])).flatten(2, 3)[:, :, None]
        if a["is_causal"]:
            seen = seen & (where.flatten(2, 3)[:, :, None] <= row)
        seen = seen & (row < row_end[heads])
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
        o = torch.matmul(p, vf[at].flatten(2, 3)) / p.sum(-1, keepdim=True).clamp_min(1e-30)
        out[heads] = o.to(torch.bfloat16)
    out = out.view(b, hq, nqb * QB, d)[:, :, :lq]
    return out if a["tensor_layout"] == "HND" else out.transpose(1, 2)


def _linear(a):
    act, down, up = a["activation"].float(), a["down"].float(), a["up"].float()
    m, (count, r, k) = act.size(0), down.shape
    y = torch.matmul(act, a["weight"].float().t()) * a["activation_scale"].view(m, 1) * a["weight_scale"]
    if a["bias"] is not None:
        y = y + a["bias"]
    ids = a["adapter_ids"].long().repeat_interleave(a["adapter_rows"])[:m]
    mine = (ids[:, None] == torch.arange(count, device=act.device)) * a["scaling"]  # [m, count]
    h = torch.matmul(act, down.view(count * r, k).t()) * a["activation_scale"].view(m, 1)
    h = (h.view(m, count, r) * mine[..., None]).view(m, count * r)
    y = (y + torch.matmul(h, up.transpose(1, 2).reshape(count * r, -1))).to(torch.bfloat16)
    if a["residual"] is None:
        return y
    gate = 1.0 if a["gate"] is None else a["gate"].float().repeat_interleave(a["gate_rows"], 0)[:m]
    return (y.float() * gate + a["residual"].float()).to(torch.bfloat16)


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    if case["kind"] == "select":
        return None  # whole numbers
    a = prepare(case, seed)["args"]
    if case["kind"] == "adapters":
        x = a["activation"].double() * a["activation_scale"].double().view(-1, 1)
        y = x @ (a["weight"].double() * a["weight_scale"].double()[:, None]).t()
        y += 0 if a["bias"] is None else a["bias"].double()
        ids = a["adapter_ids"].repeat_interleave(case["rows"])[:case["m"]]
        for i in range(case["count"]):
            rows = (ids == i).nonzero().view(-1)
            y[rows] += (x[rows] @ a["down"][i].double().t()) @ a["up"][i].double().t() * a["scaling"][i].double()
        if a["residual"] is not None:
            if a["gate"] is not None:
                y *= a["gate"].double().repeat_interleave(case["rows"], 0)[:case["m"]]
            y += a["residual"].double()
        return y
    b, hq, lq, lk = (case[x] for x in ("b", "hq", "lq", "lk"))
    q8, k8 = _heads_first(a)
    kept = torch.zeros(*a["block_index"].shape[:3], (lk + KB - 1) // KB + 1, dtype=torch.bool, device=DEVICE)
    kept.scatter_(3, torch.where(a["block_index"] < 0, kept.size(3) - 1, a["block_index"]).long(), True)
    out = torch.zeros(b, hq, lq, case["d"], dtype=torch.float64, device=DEVICE)
    for i, (ql, kl) in enumerate(zip(_lengths(case, lq), _lengths(case, lk))):
        for h in range(hq):
            kv = h // (hq // case["hkv"])
            k = k8[i, kv, :kl].double() * a["key_scale"][i, kv].double().repeat_interleave(case["blkk"])[:kl, None]
            q = q8[i, h, :ql].double() * a["query_scale"][i, h].double().repeat_interleave(case["blkq"])[:ql, None]
            s = (q @ k.t()) * case["d"] ** -0.5
            seen = kept[i, h].repeat_interleave(QB, 0)[:ql].repeat_interleave(KB, 1)[:, :kl]
            if case["causal"]:
                seen = seen.tril()
            some = seen.any(1)
            weights = s.masked_fill_(~seen, -math.inf)[some].softmax(1)
            out[i, h, :ql][some] = weights @ a["value_t"][i, kv, :, :kl].double().t()
    return out if case["layout"] == "HND" else out.transpose(1, 2)
