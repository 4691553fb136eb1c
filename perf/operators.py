"""The paged KV cache's operators as measurable cases: appending keys and values to pages
(QK-norm and rotation on the way), and the gated attention that reads them, with pages
held in bf16 or in 8 bits (e4m3 with one power-of-two scale per page and KV head).

Sizes are those of the repository's own configurations: 32 query / 4 KV heads
(`dense_8b_config_dict`), 8 / 2 (`tiny_config_dict`), 16 / 2 (the long-context verify
benchmark) and 4 / 2 (`micro_config_dict`), head dim 256, rotary dim 64.

`listed()` gives the named cases, `draw(rng)` more of the same ranges; `prepare` makes the
inputs and the pages on the device from the seed, `run` is one pass (the plain form, or the
framework's kernels where `own` is set), `work` its unavoidable bytes and flops, `exact` its
result in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
D = 256
ROTARY = 64
THETA = 1e7
EPS = 1e-6
LARGEST = 448.0        # of e4m3
LEAST_EXPONENT = -64   # of a page's scale


# ------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------
def listed():
    return [
        # the smallest attention: one user of the tiny model, one new token
        {"name": "attend 1x1 tiny", "kind": "attend", "q_heads": 8, "kv_heads": 2, "batch": 1, "T": 1,
         "context": 131, "context_max": 131, "page": 16, "bits": 16, "idle": 0, "holes": False},
        # one decode token of a serving batch, 8-bit pages; a slot of the batch is idle
        {"name": "attend 16x1 8 bit", "kind": "attend", "q_heads": 32, "kv_heads": 4, "batch": 16, "T": 1,
         "context": 1000, "context_max": 4000, "page": 64, "bits": 8, "idle": 1, "holes": False},
        # the verify block of the speculative step: pending token and three drafts
        {"name": "attend 16x4 bf16", "kind": "attend", "q_heads": 32, "kv_heads": 4, "batch": 16, "T": 4,
         "context": 2048, "context_max": 2600, "page": 64, "bits": 16, "idle": 0, "holes": False},
        # verify blocks over long contexts of very different lengths, 8-bit pages
        {"name": "attend 8x4 8 bit ragged", "kind": "attend", "q_heads": 32, "kv_heads": 4, "batch": 8, "T": 4,
         "context": 1000, "context_max": 32000, "page": 128, "bits": 8, "idle": 0, "holes": False},
        # the long-context verify benchmark's heads and contexts in small pages
        {"name": "attend 16x4 bf16 ragged", "kind": "attend", "q_heads": 16, "kv_heads": 2, "batch": 16, "T": 4,
         "context": 1024, "context_max": 32768, "page": 16, "bits": 16, "idle": 0, "holes": False},
        # two prompts of odd length into 8-bit pages
        {"name": "attend 2x1999 8 bit", "kind": "attend", "q_heads": 32, "kv_heads": 4, "batch": 2, "T": 1999,
         "context": 0, "context_max": 0, "page": 64, "bits": 8, "idle": 0, "holes": False},
        # a chunk of a long prompt behind what is cached of it, some early pages given back
        {"name": "attend 1x512 bf16", "kind": "attend", "q_heads": 32, "kv_heads": 4, "batch": 1, "T": 512,
         "context": 7777, "context_max": 7777, "page": 32, "bits": 16, "idle": 0, "holes": True},
        # the smallest append: one token of one user
        {"name": "append 1x1 tiny", "kind": "append", "q_heads": 8, "kv_heads": 2, "batch": 1, "T": 1,
         "context": 131, "context_max": 131, "page": 16, "bits": 8, "idle": 0, "far": False},
        # one decode token of a large serving batch, pages part full
        {"name": "append 64x1 8 bit", "kind": "append", "q_heads": 32, "kv_heads": 4, "batch": 64, "T": 1,
         "context": 1000, "context_max": 30000, "page": 64, "bits": 8, "idle": 2, "far": False},
        # a verify block; drafts cross from page to page
        {"name": "append 16x4 bf16", "kind": "append", "q_heads": 32, "kv_heads": 4, "batch": 16, "T": 4,
         "context": 2048, "context_max": 2600, "page": 16, "bits": 16, "idle": 0, "far": False},
        # two prompts of odd length
        {"name": "append 2x1999 8 bit", "kind": "append", "q_heads": 32, "kv_heads": 4, "batch": 2, "T": 1999,
         "context": 0, "context_max": 0, "page": 64, "bits": 8, "idle": 0, "far": False},
        # chunks of three long prompts, positions given apart from the cache's rows
        {"name": "append 3x1500 bf16", "kind": "append", "q_heads": 32, "kv_heads": 4, "batch": 3, "T": 1500,
         "context": 300, "context_max": 900, "page": 128, "bits": 16, "idle": 0, "far": True},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attend", "attend", "attend", "append", "append"])
    hq, hkv = rng.choice([(32, 4), (32, 4), (16, 2), (8, 2), (4, 2)])
    c = {"kind": kind, "q_heads": hq, "kv_heads": hkv, "page": rng.choice([16, 32, 64, 128]),
         "bits": rng.choice([8, 16])}
    if rng.random() < 0.6:      # decode, verify and small blocks
        c["T"] = rng.choice([1, 1, rng.randint(2, 6), _log(rng, 6, 64)])
        c["batch"] = _log(rng, 1, 64 // c["T"] if c["T"] > 6 else 32)
        lo = _log(rng, 1, 8000)
        c["context"], c["context_max"] = lo, _log(rng, lo, max(lo + 1, 100000 // c["batch"]))
    else:                       # prompts and chunks of them
        c["T"] = _log(rng, 16, 3000)
        c["batch"] = _log(rng, 1, max(1, 3998 // c["T"]))
        c["context"] = c["context_max"] = rng.choice([0, 0, _log(rng, 10, 8000)])
        if c["batch"] * c["T"] * (c["T"] + 2 * c["context"]) > 2 * 1999 * 1999:
            c["context"] = c["context_max"] = 0
        if c["batch"] * c["T"] * c["T"] > 2 * 1999 * 1999:
            c["batch"] = 1
            c["T"] = min(c["T"], 2700)
    c["idle"] = rng.choice([0, 0, 1]) if c["batch"] > 1 else 0
    if kind == "attend":
        c["holes"] = rng.random() < 0.2
    else:
        c["far"] = rng.random() < 0.3
    return c


# ------------------------------------------------------------------------------------
# inputs and pages
# ------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 17)
    return g


def _power_of_two_scale(amax):
    """The least power of two s with amax <= 448 s, and at least 2^LEAST_EXPONENT."""
    m, x = torch.frexp(amax)
    e = torch.where(m <= 0.875, x - 9, x - 8).clamp(min=LEAST_EXPONENT)
    return torch.ldexp(torch.ones_like(amax), e)


def _pages(g, n, hkv, page, bits):
    """Pages of stale and live rows: (pages, scales or None), the rows of different pages and
    heads of different size, as a model's keys and values are."""
    x = torch.randn(n, hkv, page, D, device=DEV, generator=g)
    x *= torch.exp2(torch.randint(-2, 3, (n, hkv, 1, 1), device=DEV, generator=g).float() / 2)
    if bits == 16:
        return x.bfloat16(), None
    s = _power_of_two_scale(x.abs().amax((2, 3)))
    return (x / s[:, :, None, None]).to(torch.float8_e4m3fn), s


def _qkv(c, g):
    """The fused projection's output; a prompt's first token stands out, as it does in a model."""
    w = c["q_heads"] * 2 * D + 2 * c["kv_heads"] * D
    x = torch.randn(c["batch"], c["T"], w, device=DEV, generator=g)
    x *= torch.exp2(torch.randn(c["batch"], c["T"], 1, device=DEV, generator=g) / 2)
    return x.bfloat16()


def prepare(case, seed):
    c, g = case, _gen(seed)
    B, T, P, hkv = c["batch"], c["T"], c["page"], c["kv_heads"]
    ctx = torch.randint(c["context"], c["context_max"] + 1, (B,), device=DEV, generator=g)
    live = torch.arange(B, device=DEV) < B - c["idle"]
    i32 = torch.int32
    if c["kind"] == "attend":
        width = -(-(c["context_max"] + T) // P)
        n = B * width + 3
        # every sequence's pages lie anywhere in the pool
        table = torch.randperm(n, device=DEV, generator=g)[:B * width].view(B, width)
        kv_len = torch.where(live, ctx + T, 0)
        table = torch.where(torch.arange(width, device=DEV) * P < kv_len[:, None], table, -1)
        if c["holes"]:          # early pages given back: their keys are out of the window
            given = torch.randint(0, max(1, width // 2), (B, 1), device=DEV, generator=g)
            table = torch.where(torch.arange(width, device=DEV) < given, -1, table)
        k, ks = _pages(g, n, hkv, P, c["bits"])
        v, vs = _pages(g, n, hkv, P, c["bits"])
        qkv = _qkv(c, g)        # the gate stays where the projection wrote it
        q = torch.randn(B, T, c["q_heads"], D, device=DEV, generator=g).bfloat16()
        return {"case": c, "q": q, "k": k, "v": v, "ks": ks, "vs": vs, "table": table.to(i32).contiguous(),
                "kv_len": kv_len.to(i32), "gate": _gate(qkv, c["q_heads"])}
    # append: the sequences share the pages of a common prompt (a handful stand for them: an
    # append never reads them) and own those from their last part full page on
    lengths = torch.where(live, ctx, 0)
    width = -(-(c["context_max"] + T) // P)
    mine = (T + P - 2) // P + 1
    n = 4 + B * mine
    first = lengths // P
    j = torch.arange(width, device=DEV)[None] - first[:, None]
    perm = 4 + torch.randperm(B * mine, device=DEV, generator=g).view(B, mine)
    table = torch.where(j < 0, torch.arange(width, device=DEV)[None] % 4,
                        torch.gather(perm, 1, j.clamp(0, mine - 1)))
    table = torch.where((j < mine) & live[:, None], table, -1)
    k, ks = _pages(g, n, hkv, P, c["bits"])
    v, vs = _pages(g, n, hkv, P, c["bits"])
    pos = None
    if c["far"]:
        pos = torch.randint(0, 250000, (B, 1), device=DEV, generator=g) + torch.arange(T, device=DEV)
        pos = pos.to(i32).contiguous()
    idx = torch.arange(0, ROTARY, 2, dtype=torch.float32)
    return {"case": c, "qkv": _qkv(c, g), "k": k, "v": v, "ks": ks, "vs": vs,
            "table": table.to(i32).contiguous(), "lengths": lengths.to(i32), "pos": pos,
            "inv_freq": (1.0 / (THETA ** (idx / ROTARY))).to(DEV),
            "q_norm": (0.1 * torch.randn(D, device=DEV, generator=g)).bfloat16(),
            "k_norm": (0.1 * torch.randn(D, device=DEV, generator=g)).bfloat16()}


def _gate(qkv, hq):
    """The gates (B, T, Hq, D) inside the fused projection's output, [query | gate] per head."""
    B, T, _ = qkv.shape
    return qkv[:, :, :hq * 2 * D].view(B, T, hq, 2 * D)[..., D:]


# ------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        from lollm_amd import ops
        if c["kind"] == "attend":
            return ops.attn_paged(s["q"], s["k"], s["v"], s["table"], s["kv_len"], s["gate"],
                                  k_scale=s["ks"], v_scale=s["vs"])
        q, _ = ops.attn_append(s["qkv"], s["q_norm"], s["k_norm"], s["inv_freq"], s["lengths"], s["table"],
                               s["k"], s["v"], c["q_heads"], ROTARY, EPS, k_scale=s["ks"], v_scale=s["vs"],
                               rope_pos=s["pos"])
    elif c["kind"] == "attend":
        return _attend(s)
    else:
        q = _append(s)
    return [q, s["k"], s["v"]] + ([s["ks"], s["vs"]] if c["bits"] == 8 else [])


def _values(pages, scale, table):
    """The rows of the tables' pages in fp32: (B, Hkv, width * P, D)."""
    B, width = table.shape
    at = table.clamp(min=0).long()
    if scale is None:
        x = pages[at].float()
    else:
        x = pages.view(torch.uint8)[at].view(pages.dtype).float() * scale[at][..., None, None]
    return x.transpose(1, 2).reshape(B, pages.shape[1], -1, D)


def _attend(s):
    c, q, table = s["case"], s["q"], s["table"]
    B, T, hq, P, hkv = c["batch"], c["T"], c["q_heads"], c["page"], c["kv_heads"]
    rep, width = hq // hkv, table.shape[1]
    j = torch.arange(width * P, device=DEV)
    mapped = ((table >= 0) & (table < s["k"].shape[0])).repeat_interleave(P, 1)
    there = mapped & (j < s["kv_len"][:, None])                                     # (B, keys)
    k = _values(s["k"], s["ks"], table)
    v = torch.where(there[:, None, :, None], _values(s["v"], s["vs"], table), 0.0)
    qq = q.float().view(B, T, hkv, rep, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, rep * T, D)
    x = torch.matmul(qq * D ** -0.5, k.transpose(-1, -2)).view(B, hkv, rep, T, -1)
    at = s["kv_len"][:, None] - T + torch.arange(T, device=DEV)                     # (B, T)
    seen = (there[:, None] & (j <= at[..., None]))[:, None, None]
    x = torch.where(seen, x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, rep * T, -1), v).view(B, hkv, rep, T, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, T, hq, D)
    return (o * torch.sigmoid(s["gate"].float())).to(q.dtype).reshape(B, T, hq * D)


def _norm_rotate(x, w, cos, sin):
    """QK-norm with (1 + w) and the partial rotate-half rotation of (B, T, H, D) fp32 rows."""
    x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + w.float())
    h = ROTARY // 2
    a, b = x[..., :h], x[..., h:ROTARY]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., ROTARY:]], -1)


def _store(s, x, pages, scale, page, slot, ok):
    """Write (B, T, Hkv, D) fp32 rows into their pages; 8-bit pages take the larger of their
    scale and the new rows', the rows that they kept are rounded to it again."""
    x, page, slot = x[ok], page[ok], slot[ok]
    if scale is None:
        pages[page, :, slot] = x.to(pages.dtype)
        return
    n, hkv, P, _ = pages.shape
    amax = torch.where(x.isfinite(), x.abs(), 0.0).amax(-1)                          # (rows, Hkv)
    most = torch.zeros(n, hkv, device=DEV).scatter_reduce(0, page[:, None].expand(-1, hkv), amax, "amax")
    lengths = s["lengths"].long()
    have = ok[:, 0]
    kept = torch.zeros(n, dtype=torch.int64, device=DEV)
    p0 = s["table"].long().gather(1, (lengths // P)[:, None].clamp(max=s["table"].shape[1] - 1))[:, 0][have]
    kept[p0] = (lengths % P)[have]
    touched = torch.zeros(n, dtype=torch.bool, device=DEV)
    touched[page] = True
    old = scale.clone()
    new = torch.maximum(torch.where(kept[:, None] > 0, old, 0.0), _power_of_two_scale(most))
    scale.copy_(torch.where(touched[:, None], new, old))
    codes = pages.view(torch.uint8)
    again = pages.view(torch.uint8)[p0].view(pages.dtype).float() * (old[p0] / scale[p0])[..., None, None]
    keep = torch.arange(P, device=DEV) < kept[p0][:, None]
    codes[p0] = torch.where(keep[:, None, :, None], again.to(pages.dtype).view(torch.uint8), codes[p0])
    codes[page, :, slot] = (x / scale[page][..., None]).to(pages.dtype).view(torch.uint8)


def _append(s):
    c, qkv, table = s["case"], s["qkv"], s["table"].long()
    B, T, hq, hkv, P = c["batch"], c["T"], c["q_heads"], c["kv_heads"], c["page"]
    r = s["lengths"].long()[:, None] + torch.arange(T, device=DEV)                  # cache rows
    pos = r if s["pos"] is None else s["pos"]
    angle = pos.double()[..., None, None] * s["inv_freq"].double()   # far positions lose in fp32
    cos, sin = angle.cos().float(), angle.sin().float()
    q = qkv[:, :, :hq * 2 * D].view(B, T, hq, 2 * D)[..., :D].float()
    k, v = (y.reshape(B, T, hkv, D).float() for y in qkv[:, :, hq * 2 * D:].split(hkv * D, -1))
    page = table.gather(1, (r // P).clamp(max=table.shape[1] - 1))
    ok = (r // P < table.shape[1]) & (page >= 0) & (page < s["k"].shape[0])
    _store(s, _norm_rotate(k, s["k_norm"], cos, sin), s["k"], s["ks"], page, r % P, ok)
    _store(s, v, s["v"], s["vs"], page, r % P, ok)
    return _norm_rotate(q, s["q_norm"], cos, sin).to(qkv.dtype)


# ------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------
def work(case):
    c = case
    B, T, hq, hkv = c["batch"] - c["idle"], c["T"], c["q_heads"], c["kv_heads"]
    row = D * c["bits"] // 8
    if c["kind"] == "append":
        values = c["batch"] * T * hq * D + 2 * B * T * hkv * D
        return {"bytes": 2 * values + 2 * c["batch"] * T * hq * D + 2 * B * T * hkv * row,
                "flops": 10 * (c["batch"] * T * hq * D + B * T * hkv * D)}
    ctx = (c["context"] + c["context_max"]) / 2
    if c["holes"]:
        ctx = ctx - (ctx + T) / 4 if ctx > T else ctx
    pairs = B * T * (ctx + (T + 1) / 2)
    return {"bytes": 2 * B * (ctx + T) * hkv * row + 3 * c["batch"] * T * hq * D * 2,
            "flops": 4 * D * hq * pairs}


# ------------------------------------------------------------------------------------
# the same in 64 bits
# ------------------------------------------------------------------------------------
def exact(case, seed):
    """Key by key and sequence by sequence from the definitions.  An 8-bit code has the value
    that is rounded to it, x / scale."""
    c, s = case, prepare(case, seed)
    B, T, hq, hkv, P = c["batch"], c["T"], c["q_heads"], c["kv_heads"], c["page"]
    f8 = c["bits"] == 8
    kd, vd = s["k"].double(), s["v"].double()
    if c["kind"] == "attend":
        if f8:
            kd, vd = kd * s["ks"].double()[..., None, None], vd * s["vs"].double()[..., None, None]
        out = torch.zeros(B, T, hq, D, dtype=torch.float64, device=DEV)
        gate = s["gate"].double()
        for b in range(B):
            L = int(s["kv_len"][b])
            ids = [(i * P + r, p, r) for i, p in enumerate(s["table"][b].tolist()) if p >= 0
                   for r in range(P) if i * P + r < L]
            if not ids:
                continue
            where, page, slot = (torch.tensor(x, device=DEV) for x in zip(*ids))
            last = torch.arange(L - T, L, device=DEV)
            hidden = where[None] > last[:, None]
            for h in range(hq):
                kb, vb = kd[page, h // (hq // hkv), slot], vd[page, h // (hq // hkv), slot]
                score = (s["q"][b, :, h].double() @ kb.T) / math.sqrt(D)
                weight = torch.softmax(score.masked_fill(hidden, -math.inf), -1)
                out[b, :, h] = torch.nan_to_num(weight) @ vb
        return (out / (1 + torch.exp(-gate))).reshape(B, T, hq * D)
    x = s["qkv"].double()
    freq = s["inv_freq"].double()
    h = ROTARY // 2

    def turn(y, w, at):
        y = y / torch.sqrt((y * y).sum(-1, keepdim=True) / D + EPS) * (1 + w.double())
        z = torch.complex(y[..., :h], y[..., h:ROTARY]) * torch.polar(torch.ones_like(at[:, None] * freq),
                                                                     at[:, None] * freq)[:, None]
        return torch.cat([z.real, z.imag, y[..., ROTARY:]], -1)

    q_out = torch.empty(B, T, hq, D, dtype=torch.float64, device=DEV)
    ks, vs = (s["ks"].double(), s["vs"].double()) if f8 else (None, None)
    for b in range(B):
        L = int(s["lengths"][b])
        rows = torch.arange(L, L + T, device=DEV)
        at = rows.double() if s["pos"] is None else s["pos"][b].double()
        q_out[b] = turn(x[b, :, :hq * 2 * D].view(T, hq, 2, D)[:, :, 0], s["q_norm"], at)
        new_k = turn(x[b, :, hq * 2 * D:][:, :hkv * D].view(T, hkv, D), s["k_norm"], at)
        new_v = x[b, :, hq * 2 * D:][:, hkv * D:].view(T, hkv, D)
        for i in range(L // P, (L + T - 1) // P + 1):
            p = int(s["table"][b, i])
            if p < 0:
                continue
            lo, hi = max(L, i * P), min(L + T, (i + 1) * P)
            for pool, scale, new in ((kd, ks, new_k), (vd, vs, new_v)):
                part = new[lo - L:hi - L].transpose(0, 1)                            # (Hkv, rows, D)
                if f8:
                    need = torch.exp2(torch.ceil(torch.log2(part.abs().amax((1, 2)) / LARGEST)).clamp(min=LEAST_EXPONENT))
                    if lo > i * P:
                        need = torch.maximum(need, scale[p])
                        pool[p, :, :lo - i * P] *= (scale[p] / need)[:, None, None]
                    scale[p] = need
                    part = part / need[:, None, None]
                pool[p, :, lo - i * P:hi - i * P] = part
    return [q_out, kd, vd] + ([ks, vs] if f8 else [])
