"""Plain 64-bit forms of the block-sparse attention and the adapters, and the
inputs and bounds that their tests share (test infrastructure)."""
from __future__ import annotations

import torch

QB, KB = 128, 64

# bf16 half a step relative to the value, and fp32's
BF16, FP32 = 2.0 ** -8, 2.0 ** -24


def codes(b, h, l, d, block, gen, device, layout="HND", spread=1.0):
    """int8 codes near normal with block scales, in ``layout``, and the scales."""
    c = torch.randn(b, h, l, d, generator=gen).mul(35).round().clamp(-127, 127).to(torch.int8)
    s = (0.5 + torch.rand(b, h, (l + block - 1) // block, generator=gen)) * 0.03 * spread
    c = c if layout == "HND" else c.transpose(1, 2).contiguous()
    return c.to(device), s.to(device)


def _hnd(c, layout):
    return c if layout == "HND" else c.transpose(1, 2)


def _lengths(lengths, batch, length):
    return [length] * batch if lengths is None else [min(max(int(x), 0), length) for x in lengths.tolist()]


def select(q8, qs, k8, ks, keep, layout, causal, sink, local, blkq, blkk, q_lengths=None, k_lengths=None):
    """select_key_blocks, block by block in fp64 on the CPU."""
    q8, k8, qs, ks = _hnd(q8, layout).cpu(), _hnd(k8, layout).cpu(), qs.cpu(), ks.cpu()
    (b, hq, lq, d), (_, hkv, lk, _) = q8.shape, k8.shape
    nqb, nkb = (lq + QB - 1) // QB, (lk + KB - 1) // KB
    qd = q8.double() * qs.double().repeat_interleave(blkq, 2)[:, :, :lq, None]
    kd = k8.double() * ks.double().repeat_interleave(blkk, 2)[:, :, :lk, None]
    out = torch.full((b, hq, nqb, min(keep, nkb)), -1, dtype=torch.int32)
    for i, (ql, kl) in enumerate(zip(_lengths(q_lengths, b, lq), _lengths(k_lengths, b, lk))):
        for h in range(hq):
            means = [kd[i, h // (hq // hkv), j * KB:min(kl, (j + 1) * KB)].mean(0) for j in range((kl + KB - 1) // KB)]
            for n in range((ql + QB - 1) // QB):
                end = min(ql, (n + 1) * QB)
                mq = qd[i, h, n * QB:end].mean(0)
                rank = []
                for j, mk in enumerate(means):
                    if causal and j * KB > end - 1:
                        continue
                    forced = j < sink or (local > 0 and 2 * n - (local - 1) <= j <= 2 * n + local)
                    s = float((mq * mk).sum())
                    rank.append((not forced, s != s, 0.0 if forced or s != s else -s, j))
                chosen = sorted(j for *_, j in sorted(rank)[:keep])
                out[i, h, n, :len(chosen)] = torch.tensor(chosen, dtype=torch.int32)
    return out


def attend(q8, qs, k8, ks, vt, index, layout, causal, sm_scale, blkq, blkk, q_lengths=None, k_lengths=None):
    """key_block_attention in fp64: (out, sum p |v| / sum p) in ``layout``."""
    q8, k8 = _hnd(q8, layout), _hnd(k8, layout)
    (b, hq, lq, d), (_, hkv, lk, _) = q8.shape, k8.shape
    out = torch.zeros(b, hq, lq, d, dtype=torch.float64, device=q8.device)
    size = torch.zeros_like(out)
    nkb = (lk + KB - 1) // KB
    lists = index.cpu().tolist()
    for i, (ql, kl) in enumerate(zip(_lengths(q_lengths, b, lq), _lengths(k_lengths, b, lk))):
        for h in range(hq):
            kv = h // (hq // hkv)
            for n in range((ql + QB - 1) // QB):
                rows = torch.arange(n * QB, min(ql, (n + 1) * QB), device=q8.device)
                top, named = -1, []
                for e in lists[i][h][n]:
                    if top < e < nkb:
                        named.append(e)
                    top = max(top, e)
                keys = [t for e in named for t in range(e * KB, min(kl, (e + 1) * KB))]
                if not keys:
                    continue
                keys = torch.tensor(keys, device=q8.device)
                s = q8[i, h, rows].double() @ k8[i, kv, keys].double().t()
                s = s * qs[i, h, rows // blkq].double()[:, None] * ks[i, kv, keys // blkk].double() * sm_scale
                seen = keys <= rows[:, None] if causal else torch.ones_like(s, dtype=torch.bool)
                some = seen.any(1)
                p = s.masked_fill(~seen, -float("inf"))[some].softmax(1)
                v = vt[i, kv][:, keys].double().t()
                out[i, h, rows[some]] = p @ v
                size[i, h, rows[some]] = p @ v.abs()
    return _hnd(out, layout), _hnd(size, layout)


def attend_bound(out, size):
    """|kernel - exact| per element: P and with it the row sum are rounded to
    bf16 (half a step each of sum p |v|), the exponent is formed to 2^-13 and
    its fp32 factors to a few 2^-23 of at most some hundred (together under
    2^-11 of the same), and the result is rounded to bf16."""
    return BF16 * out.abs() + (2 * BF16 + 2.0 ** -11) * size


def linear(act, weight, act_scale, w_scale, bias, down, up, scaling, ids, rows, residual=None, gate=None, gate_rows=1):
    """int8_linear_adapters in fp64: (out, per-element bound of the kernel)."""
    m, k = act.shape
    rank = down.shape[1]
    x, s = act.double(), act_scale.double().view(-1, 1)
    base = (x @ weight.double().t()) * s * w_scale.double()
    y = base if bias is None else base + bias.double()
    # float(acc), two products and a sum
    err = 3 * FP32 * base.abs() + FP32 * y.abs()
    ids = ids.repeat_interleave(rows)[:m]
    for a in range(down.shape[0]):
        mine = (ids == a).nonzero().view(-1)
        if not mine.numel():
            continue
        f = s[mine] * scaling[a].double()
        h = (x[mine] @ down[a].double().t()) * f
        h_abs = (x[mine].abs() @ down[a].double().abs().t()) * f.abs()
        u = up[a].double().t()
        y = y.index_add(0, mine, h @ u)
        # h: K products summed in fp32, then two roundings; as two bf16 terms
        # off by 2^-16 of it; 2 rank products and sums in fp32
        h_err = (k + 2) * FP32 * h_abs + 2.0 ** -16 * h.abs()
        err = err.index_add(0, mine, h_err @ u.abs() + (2 * rank + 2) * FP32 * (h.abs() @ u.abs()))
    err = err + BF16 * y.abs() + BF16 * err
    if residual is None:
        return y, err
    g = 1.0 if gate is None else gate.double().repeat_interleave(gate_rows, 0)[:m]
    out = y * g + residual.double()
    err = err * (abs(g) if gate is None else g.abs())
    return out, err + BF16 * (out.abs() + err)
