"""The paged cache's operators in 64 bits on the CPU, from their definitions: loops over
sequences, heads and pages, no code shared with the kernels' wrappers."""

import math

import torch

D = 256
E4M3_MAX = 448.0


def values(pages, scale):
    """What the pages hold, in 64 bits."""
    x = pages.to(torch.float32).double()
    return x if scale is None else x * scale.double()[:, :, None, None]


def pow2_scale(amax):
    """The least power of two s >= 2^-64 with amax <= 448 s."""
    if amax == 0.0:
        return 2.0 ** -64
    return 2.0 ** max(-64, math.ceil(math.log2(amax / E4M3_MAX)))


def attention(q, k_pages, v_pages, table, kv_len, gate, k_scale=None, v_scale=None, scale=None):
    """(out (B, T, Hq*D), tolerance of a bf16 result): half a bf16 step of the value (2^-8); on the
    weighted mean of |v| half a step of the weights' type (bf16 pages: hi + lo, 16 bits, 2^-15 for
    the weight and the sum; 8-bit pages: fp16, 2^-11) and the fp32 scores (258 roundings of 2^-24 on
    the absolute products, doubled for the sum); and for fp16 weights, whose step ends at 2^-24, half
    of that (2^-25) on the sum of |v| beside a largest weight of 1 or more.  8-bit values enter as fp16 in
    units of at most the largest scale among the sequence's pages: half of fp16's least step in these
    units, 2^-25 of that scale, on each value, so on their mean."""
    weight = 2.0 ** -14 if k_scale is None else 2.0 ** -11
    B, T, Hq, _ = q.shape
    n, Hkv, P, _ = k_pages.shape
    s = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, T, Hq, D, dtype=torch.float64)
    tol = torch.zeros_like(out)
    kd, vd = values(k_pages, k_scale), values(v_pages, v_scale)
    for b in range(B):
        L = min(max(int(kv_len[b]), 0), table.shape[1] * P)
        where = [j for j in range(L) if 0 <= int(table[b, j // P]) < n]
        if not where:
            continue
        at = torch.tensor(where)
        page, slot = table[b].long()[at // P], at % P
        hidden = at[None] > torch.arange(L - T, L)[:, None]
        for h in range(Hq):
            kb, vb = kd[page, h // (Hq // Hkv), slot], vd[page, h // (Hq // Hkv), slot]
            qb = q[b, :, h].double()
            x = (qb @ kb.T * s).masked_fill(hidden, -math.inf)
            p = torch.softmax(x, -1).nan_to_num(0.0)
            out[b, :, h] = p @ vb
            ds = 258 * 2.0 ** -24 * (qb.abs() @ kb.abs().T * s).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
            tol[b, :, h] = (weight + 2 * ds) * (p @ vb.abs())
            if k_scale is not None:
                tol[b, :, h] += 2.0 ** -25 * p.amax(-1, keepdim=True) * ((~hidden).double() @ vb.abs())
                tol[b, :, h] += 2.0 ** -25 * float(v_scale[page, h // (Hq // Hkv)].max()) * (~hidden).any(-1, keepdim=True)
    if gate is not None:
        g = torch.sigmoid(gate.double().reshape(B, T, Hq, D))
        out, tol = out * g, tol * g
    # 2^-20: the gate's fp32 sigmoid and the division
    tol = tol + (2.0 ** -8 + 2.0 ** -20) * out.abs()
    return out.reshape(B, T, Hq * D), tol.reshape(B, T, Hq * D)


def norm_rotate(x, w, eps, rd, inv_freq, pos):
    """QK-norm and rotation of (T, H, D) rows at positions pos (T,), in 64 bits."""
    x = x.double()
    x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * (1 + w.double())
    h = rd // 2
    if h == 0:
        return x
    ang = (pos.double()[:, None] * inv_freq.double())[:, None]
    a, b = x[..., :h], x[..., h:rd]
    return torch.cat([a * ang.cos() - b * ang.sin(), b * ang.cos() + a * ang.sin(), x[..., rd:]], -1)


def append(qkv, qw, kw, inv_freq, lengths, table, k_pages, v_pages, Hq, rd, eps, k_scale=None,
           v_scale=None, rope_pos=None):
    """(q in 64 bits, {"k": new, "v": new}): for each, the pool's unrounded values in 64 bits, the
    scales, and a mask of the rows that the call stores."""
    B, T, _ = qkv.shape
    n, Hkv, P, _ = k_pages.shape
    q = torch.empty(B, T, Hq, D, dtype=torch.float64)
    res = {}
    for name, pages, scale in (("k", k_pages, k_scale), ("v", v_pages, v_scale)):
        res[name] = {"values": values(pages, scale), "scale": None if scale is None else scale.double().clone(),
                     "stored": torch.zeros(n, Hkv, P, dtype=torch.bool), "kept": torch.zeros(n, Hkv, P, dtype=torch.bool)}
    for b in range(B):
        L = int(lengths[b])
        pos = torch.arange(L, L + T)
        if rope_pos is not None:
            pos = rope_pos[b].long() if rope_pos.dim() == 2 else int(rope_pos[b]) + torch.arange(T)
        q[b] = norm_rotate(qkv[b, :, :Hq * 2 * D].view(T, Hq, 2, D)[:, :, 0], qw, eps, rd, inv_freq, pos)
        kv = qkv[b, :, Hq * 2 * D:].view(T, 2, Hkv, D)
        new = {"k": norm_rotate(kv[:, 0], kw, eps, rd, inv_freq, pos), "v": kv[:, 1].double()}
        for i in range(table.shape[1]):
            p = int(table[b, i])
            rows = [t for t in range(T) if i * P <= L + t < (i + 1) * P]
            if not rows or not 0 <= p < n:
                continue
            s0 = L + rows[0] - i * P
            for name, r in res.items():
                part = new[name][rows]
                for h in range(Hkv):
                    if r["scale"] is not None:
                        fin = part[:, h][part[:, h].isfinite()]
                        s = pow2_scale(float(fin.abs().max()) if fin.numel() else 0.0)
                        if s0 > 0:
                            s = max(s, float(r["scale"][p, h]))
                        r["scale"][p, h] = s
                    r["values"][p, h, s0:s0 + len(rows)] = part[:, h]
                    r["stored"][p, h, s0:s0 + len(rows)] = True
                    r["kept"][p, h, :s0] = True
    return q, res
