"""The operators of a verify step over a tree of drafted tokens with 4-bit weights as measurable
cases: products with 4-bit weights and group scales, the gated attention of the tree's nodes over
the cache (slabs, bf16 pages, 8-bit pages), and the Gated DeltaNet layer over the tree.

Sizes are those of the repository's own configurations: hidden 4096 / 32 query and 4 KV heads /
16 key and 32 value heads of the recurrent layers (`dense_8b_config_dict`), 1024 / 8 and 2 / 8 and
16 (`tiny_config_dict`), the long-context verify benchmark's 16 / 2 heads, 256 / 4 and 2 / 2 and 4
(`micro_config_dict`).  A tree has at most 64 nodes, node i's parent before it; node 0 is the
pending token.

`listed()` gives the named cases, `draw(rng)` more of the same ranges; `prepare` makes the inputs
on the device from the seed, `run` is one pass (the plain form, or the framework's kernels where
`own` is set), `work` its unavoidable bytes and flops, `exact` its result in 64 bits.
"""

import math

import torch

own = False

DEV = "cuda"
D = 256          # of an attention head
DG = 128         # of a recurrent head
TAPS = 4         # of the convolution
EPS = 1e-6
MOST = 1999 * 18432 * 4096      # products of the largest listed matrix


# ------------------------------------------------------------------------------------
# the cases
# ------------------------------------------------------------------------------------
def listed():
    return [
        # one token of the tiny model through its output projection
        {"name": "q4 1 row 1024x2048", "kind": "q4", "rows": 1, "N": 1024, "K": 2048, "group": 32, "zeros": False,
         "swiglu": False},
        # one user's token through the largest layer product, SwiGLU with it
        {"name": "q4 1 row gate|up", "kind": "q4", "rows": 1, "N": 24576, "K": 4096, "group": 128, "zeros": True,
         "swiglu": True},
        # a draft position of 16 sequences
        {"name": "q4 16 rows down", "kind": "q4", "rows": 16, "N": 4096, "K": 12288, "group": 64, "zeros": False,
         "swiglu": False},
        # one tree of an odd number of nodes into a recurrent layer
        {"name": "q4 61 rows in_proj", "kind": "q4", "rows": 61, "N": 12352, "K": 4096, "group": 128, "zeros": True,
         "swiglu": False},
        # trees of 16 sequences at once
        {"name": "q4 256 rows o_proj", "kind": "q4", "rows": 256, "N": 4096, "K": 8192, "group": 128, "zeros": False,
         "swiglu": False},
        # a prompt of odd length
        {"name": "q4 1999 rows q|k|v", "kind": "q4", "rows": 1999, "N": 18432, "K": 4096, "group": 128,
         "zeros": False, "swiglu": False},
        # the smallest tree of one user, slab cache
        {"name": "attend 1x7 tiny slab", "kind": "attend", "q_heads": 8, "kv_heads": 2, "batch": 1, "T": 7,
         "context": 131, "context_max": 131, "cache": "slab", "page": 0, "idle": 0, "spread": 3},
        # a serving batch's trees over bf16 pages; one slot is idle
        {"name": "attend 16x16 bf16 pages", "kind": "attend", "q_heads": 32, "kv_heads": 4, "batch": 16, "T": 16,
         "context": 2048, "context_max": 2600, "cache": "pages", "page": 64, "idle": 1, "spread": 6},
        # large trees over long ragged contexts in 8-bit pages
        {"name": "attend 4x63 8 bit ragged", "kind": "attend", "q_heads": 32, "kv_heads": 4, "batch": 4, "T": 63,
         "context": 1000, "context_max": 30000, "cache": "pages8", "page": 128, "idle": 0, "spread": 20},
        # one user's small tree through a recurrent layer of the tiny model
        {"name": "gdn 1x7 tiny", "kind": "gdn", "k_heads": 8, "v_heads": 16, "batch": 1, "T": 7, "slots": 7,
         "spread": 3},
        # a serving batch's trees
        {"name": "gdn 16x16", "kind": "gdn", "k_heads": 16, "v_heads": 32, "batch": 16, "T": 16, "slots": 16,
         "spread": 6},
        # large trees of an odd size
        {"name": "gdn 8x63", "kind": "gdn", "k_heads": 16, "v_heads": 32, "batch": 8, "T": 63, "slots": 64,
         "spread": 20},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


PRODUCTS = [(18432, 4096, False), (12352, 4096, False), (4096, 4096, False), (4096, 8192, False),
            (4096, 12288, False), (24576, 4096, True), (5120, 1024, False), (6208, 1024, False),
            (1024, 2048, False), (6144, 1024, True), (256, 512, False), (1024, 256, True)]


def draw(rng):
    kind = rng.choice(["q4", "q4", "attend", "attend", "gdn"])
    if kind == "q4":
        N, K, swiglu = rng.choice(PRODUCTS)
        rows = rng.choice([1, rng.randint(2, 16), rng.randint(17, 64), _log(rng, 65, 2000)])
        return {"kind": kind, "rows": max(1, min(rows, MOST // (N * K))), "N": N, "K": K,
                "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5, "swiglu": swiglu}
    T = rng.choice([rng.randint(1, 8), rng.randint(9, 32), rng.randint(33, 64)])
    spread = rng.choice([1, rng.randint(2, 8), 64])          # 1: a chain, 64: parents anywhere
    if kind == "gdn":
        hk, hv = rng.choice([(16, 32), (16, 32), (8, 16), (2, 4)])
        return {"kind": kind, "k_heads": hk, "v_heads": hv, "batch": _log(rng, 1, min(32, 512 // T)), "T": T,
                "slots": rng.randint(T, 64), "spread": spread}
    hq, hkv = rng.choice([(32, 4), (32, 4), (16, 2), (8, 2), (4, 2)])
    cache = rng.choice(["slab", "pages", "pages8"])
    batch = _log(rng, 1, min(32, 512 // T))
    lo = _log(rng, 1, 4000)
    return {"kind": kind, "q_heads": hq, "kv_heads": hkv, "batch": batch, "T": T, "context": lo,
            "context_max": _log(rng, lo, max(lo, 60000 // batch)), "cache": cache,
            "page": 0 if cache == "slab" else rng.choice([16, 32, 64, 128]),
            "idle": rng.choice([0, 0, 1]) if batch > 1 else 0, "spread": spread}


# ------------------------------------------------------------------------------------
# inputs
# ------------------------------------------------------------------------------------
def _gen(seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed) * 1000003 + 29)
    return g


def _tree(g, B, T, spread):
    """(parents (B, T) int64, -1 above node 0; ancestor bitmaps (B, T) int64, a node's own bit
    among them).  Node i hangs on one of the `spread` nodes before it."""
    i = torch.arange(T, device=DEV)
    back = (torch.rand(B, T, device=DEV, generator=g) * i.clamp(max=spread)).long() + 1
    parents = torch.where(i > 0, i - back, -1)
    mask = torch.zeros(B, T, dtype=torch.int64, device=DEV)
    one = torch.ones((), dtype=torch.int64, device=DEV)
    for n in range(T):
        above = mask.gather(1, parents[:, n:n + 1].clamp(min=0))[:, 0] if n else 0
        mask[:, n] = above | (one << n)
    return parents, mask


def _q4_inputs(c, g):
    """Normal weights of different size per output, quantised to 16 levels a group, and rows of
    activations some of whose channels stand out, as a model's do."""
    N, K, G = c["N"], c["K"], c["group"]
    w = torch.randn(N, K // G, G, device=DEV, generator=g)
    w *= 0.02 * torch.exp2(torch.randn(N, 1, 1, device=DEV, generator=g) / 2)
    if c["zeros"]:
        lo, hi = w.amin(-1, keepdim=True).clamp(max=0), w.amax(-1, keepdim=True).clamp(min=0)
        scale = ((hi - lo) / 15).bfloat16()
        zero = torch.round(-lo / scale.float()).clamp(0, 15)
    else:
        scale = (w.abs().amax(-1, keepdim=True) / 7.5).bfloat16()
        zero = torch.full_like(scale, 8, dtype=torch.float32)
    code = (torch.round(w / scale.float()) + zero).clamp(0, 15).to(torch.uint8).view(N, K)
    x = torch.randn(c["rows"], K, device=DEV, generator=g)
    x *= torch.where(torch.rand(K, device=DEV, generator=g) < 0.01, 16.0, 1.0)
    x *= torch.exp2(torch.randn(c["rows"], 1, device=DEV, generator=g) / 2)
    s = {"case": c, "x": x.bfloat16(), "codes": code[:, 0::2] | (code[:, 1::2] << 4), "scales": scale[..., 0],
         "zeros": zero[..., 0].to(torch.uint8) if c["zeros"] else None}
    if own:      # laid out once, when a model is loaded
        from lollm_amd import ops
        s["weight"] = ops.q4_pack(s["codes"], s["scales"], s["zeros"],
                                  epilogue=ops.GEMM_SWIGLU if c["swiglu"] else ops.GEMM_NONE)
    return s


def _attend_inputs(c, g):
    B, T, hq, hkv, P = c["batch"], c["T"], c["q_heads"], c["kv_heads"], c["page"]
    ctx = torch.randint(c["context"], c["context_max"] + 1, (B,), device=DEV, generator=g)
    kv_len = torch.where(torch.arange(B, device=DEV) < B - c["idle"], ctx + T, 0)
    _, mask = _tree(g, B, T, c["spread"])
    q = torch.randn(B, T, hq, D, device=DEV, generator=g).bfloat16()
    # the gate lies where the fused projection wrote it, [query | gate] of each head
    qkv = torch.randn(B, T, hq * 2 * D + 2 * hkv * D, device=DEV, generator=g).bfloat16()
    gate = qkv[:, :, :hq * 2 * D].view(B, T, hq, 2 * D)[..., D:]
    s = {"case": c, "q": q, "kv_len": kv_len.to(torch.int32), "mask": mask, "ks": None, "vs": None, "table": None}
    longest = c["context_max"] + T

    def rows(n, m):      # rows of different pages (or runs) and heads of different size
        x = torch.randn(n, hkv, m, D, device=DEV, generator=g)
        return x.mul_(torch.exp2(torch.randint(-2, 3, (n, hkv, 1, 1), device=DEV, generator=g).float() / 2))

    if c["cache"] == "slab":
        s["k"], s["v"] = rows(B, longest + 5).bfloat16(), rows(B, longest + 5).bfloat16()
        s["gate"] = gate.reshape(B, T, hq * D)
        return s
    width = -(-longest // P)
    n = B * width + 3
    table = torch.randperm(n, device=DEV, generator=g)[:B * width].view(B, width)
    table = torch.where(torch.arange(width, device=DEV) * P < kv_len[:, None], table, -1)
    s["gate"], s["table"] = gate, table.to(torch.int32).contiguous()
    for name, scale in (("k", "ks"), ("v", "vs")):
        x = rows(n, P)
        if c["cache"] == "pages":
            s[name] = x.bfloat16()
        else:            # e4m3 codes, one power of two a page and head
            s[scale] = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448)))
            s[name] = (x / s[scale][:, :, None, None]).to(torch.float8_e4m3fn)
    return s


def _gdn_inputs(c, g):
    B, T, hk, hv, S = c["batch"], c["T"], c["k_heads"], c["v_heads"], c["slots"]
    C, W = 2 * hk * DG + hv * DG, TAPS - 1 + S

    def randn(*shape):
        return torch.randn(*shape, device=DEV, generator=g)

    def randint(lo, hi, *shape):
        return torch.randint(lo, hi, shape, device=DEV, generator=g)

    _, mask = _tree(g, B, T, c["spread"])
    width = -(-(C + hv * DG + 2 * hv) // 64) * 64        # the projection's columns come in 64s
    # records of an earlier call: keys and values as they left the convolution, decay, beta, 1 / |k|
    kv = torch.nn.functional.silu(randn(B, 2, hv, S, 2 * DG)).bfloat16()
    norm = torch.rsqrt(kv[..., :DG].float().square().sum(-1) + EPS)
    scalars = torch.stack([torch.exp(-torch.rand(B, 2, hv, S, device=DEV, generator=g)),
                           torch.sigmoid(randn(B, 2, hv, S)), norm, torch.zeros_like(norm)], -1)
    rep = torch.cat([kv.view(torch.uint8), scalars.view(torch.uint8)], -1)
    half = randint(0, 2, B)
    return {"case": c, "mask": mask, "proj": randn(B, T, width).bfloat16(),
            "conv_w": (0.3 * randn(C, TAPS)).bfloat16(),
            "A_log": torch.log(torch.rand(hv, device=DEV, generator=g) * 1.9 + 0.1), "dt_bias": 0.5 * randn(hv),
            "norm_w": (1 + 0.1 * randn(DG)).bfloat16(), "win": randn(B, 2 * W, C).bfloat16(),
            "conv_off": (half * W + randint(0, S + 1, B)).to(torch.int32),
            "rec": 0.1 * randn(B, 2, hv, DG, DG), "rec_half": half.to(torch.int32), "rep": rep.contiguous(),
            "replay": randint(0, min(S, 6) + 1, B).to(torch.int32)}


def prepare(case, seed):
    return {"q4": _q4_inputs, "attend": _attend_inputs, "gdn": _gdn_inputs}[case["kind"]](case, _gen(seed))


# ------------------------------------------------------------------------------------
# one pass
# ------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if not own:
        return {"q4": _q4, "attend": _attend, "gdn": _gdn}[c["kind"]](s)
    from lollm_amd import ops
    if c["kind"] == "q4":
        return ops.gemm_q4(s["x"], s["weight"])
    if c["kind"] == "attend":
        if c["cache"] == "slab":
            return ops.attn_verify(s["q"], s["k"], s["v"], s["kv_len"], s["gate"], tree=s["mask"])
        return ops.attn_paged(s["q"], s["k"], s["v"], s["table"], s["kv_len"], s["gate"], k_scale=s["ks"],
                              v_scale=s["vs"], tree=s["mask"])
    out = ops.gdn_layer(s["proj"], s["conv_w"], s["A_log"], s["dt_bias"], s["norm_w"], s["win"], s["conv_off"],
                        s["rec"], s["rec_half"], s["rep"], s["replay"], False, c["batch"], c["T"], c["k_heads"],
                        c["v_heads"], DG, TAPS, EPS, tree=s["mask"])
    return _gdn_outputs(s, out)


def _gdn_outputs(s, out):
    """The layer's output and its updated state: states, conv windows, the records' keys and values
    and their scalars."""
    return [out, s["rec"], s["win"], s["rep"][..., :4 * DG].view(torch.bfloat16),
            s["rep"][..., 4 * DG:].view(torch.float32)]


def _q4(s):
    c = s["case"]
    N, K, G = c["N"], c["K"], c["group"]
    code = torch.stack([s["codes"] & 15, s["codes"] >> 4], -1).view(N, K // G, G).float()
    zero = 8.0 if s["zeros"] is None else s["zeros"].float()[..., None]
    w = ((code - zero) * s["scales"].float()[..., None]).view(N, K)
    y = torch.matmul(s["x"].float(), w.t())
    if c["swiglu"]:
        gate, up = y.chunk(2, -1)
        y = gate * torch.sigmoid(gate) * up
    return y.to(s["x"].dtype)


def _bits(mask, T):
    """(B, T, T): whether node j is node i or above it."""
    j = torch.arange(T, device=DEV)
    return ((mask[..., None] >> j) & 1).bool()


def _attend(s):
    c, q = s["case"], s["q"]
    B, T, hq, hkv = c["batch"], c["T"], c["q_heads"], c["kv_heads"]
    if s["table"] is None:
        k, v = s["k"].float(), s["v"].float()
    else:
        at = s["table"].clamp(min=0).long()

        def values(pages, scale):
            if scale is None:
                x = pages[at].float()
            else:
                x = pages.view(torch.uint8)[at].view(pages.dtype).float() * scale[at][..., None, None]
            return x.transpose(1, 2).reshape(B, hkv, -1, D)

        k, v = values(s["k"], s["ks"]), values(s["v"], s["vs"])
    keys = k.shape[2]
    j = torch.arange(keys, device=DEV)
    first = s["kv_len"].long()[:, None] - T                                  # the row of node 0
    node = (j - first)[:, None]                                              # (B, 1, keys)
    bit = _bits(s["mask"], T).gather(2, node.clamp(0, T - 1).expand(B, T, keys))
    seen = (j < s["kv_len"][:, None])[:, None] & ((node < 0) | bit)          # (B, T, keys)
    v = torch.where((j < s["kv_len"][:, None])[:, None, :, None], v, 0.0)
    rep = hq // hkv
    qq = q.float().view(B, T, hkv, rep, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, rep * T, D)
    x = torch.matmul(qq * D ** -0.5, k.transpose(-1, -2).contiguous()).view(B, hkv, rep, T, keys)
    x = torch.where(seen[:, None, None], x, -math.inf)
    m = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(m == -math.inf, 0.0, m))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(B, hkv, rep * T, keys), v).view(B, hkv, rep, T, D)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(B, T, hq, D)
    gate = s["gate"].view(B, T, hq, D) if s["gate"].dim() == 3 else s["gate"]
    return (o * torch.sigmoid(gate.float())).to(q.dtype).reshape(B, T, hq * D)


def _gdn(s):
    """Node after node from the parent's state.  Queries, keys and values are bf16 tensors, as the
    records hold the latter two for the next call."""
    c = s["case"]
    B, T, hk, hv, S = c["batch"], c["T"], c["k_heads"], c["v_heads"], c["slots"]
    C, W, per = 2 * hk * DG + hv * DG, TAPS - 1 + S, hv // hk
    b = torch.arange(B, device=DEV)
    half, other = s["rec_half"].long(), 1 - s["rec_half"].long()
    above = _bits(s["mask"], T) & ~torch.eye(T, dtype=torch.bool, device=DEV)
    i = torch.arange(T, device=DEV)
    parent = torch.where(above, i, -1).amax(-1)                              # (B, T), -1: the root
    # the convolution's inputs of a node: itself and its next three ancestors, then the window's rows
    raw = s["proj"][..., :C]
    rows = s["conv_off"].long()[:, None] + torch.arange(TAPS - 1, device=DEV)
    source = torch.cat([s["win"][b[:, None], rows], raw], 1).float()         # (B, 3 + T, C)
    up = torch.cat([torch.full((B, TAPS - 1), 0, device=DEV, dtype=torch.long), parent + TAPS - 1], 1)
    up = torch.where(up < TAPS - 1, TAPS - 2, up)                            # above a root: the window's last row
    up[:, :TAPS - 1] = torch.arange(-1, TAPS - 2, device=DEV).clamp(min=0)   # and the rows before that
    at = (i + TAPS - 1).expand(B, T)
    acc = torch.zeros(B, T, C, device=DEV)
    for tap in range(TAPS - 1, -1, -1):
        acc += source[b[:, None], at] * s["conv_w"][:, tap].float()
        at = up.gather(1, at)
    act = (acc * torch.sigmoid(acc)).to(s["proj"].dtype).float()
    q = act[..., :hk * DG].view(B, T, hk, DG).repeat_interleave(per, 2)
    k = act[..., hk * DG:2 * hk * DG].view(B, T, hk, DG).repeat_interleave(per, 2)
    v = act[..., 2 * hk * DG:].view(B, T, hv, DG)
    z = s["proj"][..., C:C + hv * DG].float().view(B, T, hv, DG)
    beta = torch.sigmoid(s["proj"][..., C + hv * DG:C + hv * DG + hv].float())
    a = s["proj"][..., C + hv * DG + hv:C + hv * DG + 2 * hv].float() + s["dt_bias"]
    gamma = torch.exp(-torch.exp(s["A_log"]) * torch.where(a > 20, a, torch.log1p(torch.exp(a.clamp(max=20)))))
    rk = torch.rsqrt(k.square().sum(-1) + EPS)
    rq = torch.rsqrt(q.square().sum(-1) + EPS) * DG ** -0.5

    def rule(state, k, v, gamma, beta):      # (n, hv, DG, DG) from (n, hv, DG) and (n, hv)
        state = state * gamma[..., None, None]
        u = (v - torch.matmul(k[..., None, :], state)[..., 0, :]) * beta[..., None]
        return state + k[..., :, None] * u[..., None, :]

    # the committed state: the half's, with its first `replay` records applied
    state = s["rec"][b, half]
    kv = s["rep"][..., :4 * DG].view(torch.bfloat16)[b, half].float()
    scalars = s["rep"][..., 4 * DG:].view(torch.float32)[b, half]
    for n in range(S):
        live = s["replay"] > n
        if n >= 6:                           # (a call of few tokens leaves few)
            break
        x = scalars[:, :, n]
        new = rule(state, kv[:, :, n, :DG] * x[..., 2:3], kv[:, :, n, DG:], x[..., 0], x[..., 1])
        state = torch.where(live[:, None, None, None], new, state)
    states = torch.empty(T + 1, B, hv, DG, DG, device=DEV)
    states[T] = state                        # (index -1: the root's)
    o = torch.empty(B, T, hv, DG, device=DEV)
    for n in range(T):
        states[n] = rule(states[parent[:, n], b], k[:, n] * rk[:, n, :, None], v[:, n], gamma[:, n], beta[:, n])
        o[:, n] = torch.matmul((q[:, n] * rq[:, n, :, None])[..., None, :], states[n])[..., 0, :]
    y = o * torch.rsqrt(o.square().mean(-1, keepdim=True) + EPS) * s["norm_w"].float() * z * torch.sigmoid(z)
    # the written half: the committed state, a record a node, the window's rows and the inputs
    s["rec"][b, other] = state
    s["rep"][..., :4 * DG].view(torch.bfloat16)[b, other, :, :T] = torch.cat([k, v], -1).transpose(1, 2).bfloat16()
    s["rep"][..., 4 * DG:].view(torch.float32)[b, other, :, :T] = torch.stack(
        [gamma, beta, rk, torch.zeros_like(rk)], -1).transpose(1, 2)
    to = torch.where(s["conv_off"].long() >= W, 0, W)[:, None] + torch.arange(TAPS - 1 + T, device=DEV)
    s["win"][b[:, None], to] = source.bfloat16()
    return _gdn_outputs(s, y.to(s["proj"].dtype).reshape(B, T, hv * DG))


# ------------------------------------------------------------------------------------
# what a pass cannot do without
# ------------------------------------------------------------------------------------
def work(case):
    c = case
    if c["kind"] == "q4":
        M, N, K = c["rows"], c["N"], c["K"]
        groups = N * K // c["group"]
        return {"bytes": N * K // 2 + groups * (3 if c["zeros"] else 2) + 2 * M * (K + (N // 2 if c["swiglu"] else N)),
                "flops": 2 * M * N * K}
    B, T = c["batch"], c["T"]
    if c["kind"] == "attend":
        live, hq, hkv = B - c["idle"], c["q_heads"], c["kv_heads"]
        ctx = (c["context"] + c["context_max"]) / 2
        row = D * (1 if c["cache"] == "pages8" else 2)
        return {"bytes": 2 * live * (ctx + T) * hkv * row + 3 * B * T * hq * D * 2 + 8 * B * T,
                "flops": 4 * D * hq * live * T * (ctx + min(T, 6))}
    hk, hv = c["k_heads"], c["v_heads"]
    C = 2 * hk * DG + hv * DG
    state, rec = B * hv * DG * DG * 4, 4 * DG + 16
    rows = B * T * (2 * (C + 2 * hv * DG + 2 * hv) + hv * rec) + 2 * B * (2 * (TAPS - 1) + T) * C + 8 * B * T
    return {"bytes": 2 * state + rows + B * hv * min(c["slots"], 6) // 2 * rec,
            "flops": B * hv * (T * 8 * DG * DG + 4 * TAPS * T * DG)}


# ------------------------------------------------------------------------------------
# the same in 64 bits
# ------------------------------------------------------------------------------------
def exact(case, seed):
    """From the definitions: a product group by group, attention sequence by sequence, the delta
    rule down each node's own path from the root."""
    s = prepare(case, seed)
    return {"q4": _q4_exact, "attend": _attend_exact, "gdn": _gdn_exact}[case["kind"]](case, s)


def _q4_exact(c, s):
    N, K, G = c["N"], c["K"], c["group"]
    y = torch.zeros(c["rows"], N, dtype=torch.float64, device=DEV)
    x = s["x"].double()
    for k in range(0, K, G):
        low = s["codes"][:, k // 2:(k + G) // 2].long()
        zero = 8 if s["zeros"] is None else s["zeros"][:, k // G, None].long()
        w = torch.empty(N, G, dtype=torch.float64, device=DEV)
        w[:, 0::2] = (low % 16 - zero).double()
        w[:, 1::2] = (low // 16 - zero).double()
        y += (x[:, k:k + G] @ w.t().contiguous()) * s["scales"][:, k // G].double()
    if c["swiglu"]:
        y = y[:, :N // 2] / (1 + torch.exp(-y[:, :N // 2])) * y[:, N // 2:]
    return y


def _attend_exact(c, s):
    B, T, hq, hkv, P = c["batch"], c["T"], c["q_heads"], c["kv_heads"], c["page"]
    rep = hq // hkv
    out = torch.zeros(B, T, hq, D, dtype=torch.float64, device=DEV)
    lengths, masks = s["kv_len"].tolist(), s["mask"].tolist()
    for b in range(B):
        L = lengths[b]
        if not L:
            continue
        if s["table"] is None:
            k, v = s["k"][b, :, :L].double(), s["v"][b, :, :L].double()
        else:
            pages = s["table"][b, :-(-L // P)].long()

            def rows(pool, scale):
                x = pool.view(torch.uint8)[pages].view(pool.dtype).double() if scale is not None else pool[pages].double()
                x = x if scale is None else x * scale[pages].double()[..., None, None]
                return torch.cat(list(x), 1)[:, :L]

            k, v = rows(s["k"], s["ks"]), rows(s["v"], s["vs"])
        hidden = torch.ones(T, L, dtype=torch.bool)
        hidden[:, :L - T] = False
        for i in range(T):
            for j in range(i + 1):
                hidden[i, L - T + j] = not (masks[b][i] >> j) & 1
        hidden = hidden.to(DEV)
        for h in range(hq):
            x = (s["q"][b, :, h].double() @ k[h // rep].t().contiguous()) / math.sqrt(D)
            out[b, :, h] = torch.softmax(x.masked_fill(hidden, -math.inf), -1) @ v[h // rep]
    gate = s["gate"].reshape(B, T, hq, D).double()
    return (out / (1 + torch.exp(-gate))).view(B, T, hq * D)


def _gdn_exact(c, s):
    B, T, hk, hv, S = c["batch"], c["T"], c["k_heads"], c["v_heads"], c["slots"]
    C, W = 2 * hk * DG + hv * DG, TAPS - 1 + S
    f64 = torch.float64
    rec, win = s["rec"].double(), s["win"].double()
    kv_all, scal_all = (x.double() for x in (s["rep"][..., :4 * DG].view(torch.bfloat16),
                                             s["rep"][..., 4 * DG:].view(torch.float32)))
    out = torch.zeros(B, T, hv, DG, dtype=f64, device=DEV)
    masks = s["mask"].tolist()
    offs, halves, replays = s["conv_off"].tolist(), s["rec_half"].tolist(), s["replay"].tolist()
    proj, taps = s["proj"].double(), s["conv_w"].double()
    for b in range(B):
        window = win[b, offs[b]:offs[b] + TAPS - 1].clone()
        paths = [[j for j in range(i + 1) if (masks[b][i] >> j) & 1] for i in range(T)]
        conv = torch.zeros(T, C, dtype=f64, device=DEV)
        for i in range(T):
            line = torch.cat([window, proj[b, paths[i], :C]])[-TAPS:]
            conv[i] = (line * taps.t()).sum(0)
        held = (conv / (1 + torch.exp(-conv)))
        act = held.float().bfloat16().double()       # (the tensors that the rule consumes are bf16)
        tail = proj[b, :, C:]
        z, bb, aa = tail[:, :hv * DG].view(T, hv, DG), tail[:, hv * DG:hv * DG + hv], tail[:, hv * DG + hv:hv * DG + 2 * hv]
        beta = 1 / (1 + torch.exp(-bb))
        gamma = torch.exp(-torch.exp(s["A_log"].double()) * torch.log1p(torch.exp(aa + s["dt_bias"].double())))
        head = torch.arange(hv, device=DEV) // (hv // hk)
        q = act[:, :hk * DG].view(T, hk, DG)[:, head]
        k = act[:, hk * DG:2 * hk * DG].view(T, hk, DG)[:, head]
        v = act[:, 2 * hk * DG:].view(T, hv, DG)
        rk = 1 / torch.sqrt((k * k).sum(-1) + EPS)
        qn = q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS) / math.sqrt(DG)

        def after(state, key, value, decay, rate):
            err = value - decay[:, None] * (state * key[:, :, None]).sum(1)
            return decay[:, None, None] * state + key[:, :, None] * (rate[:, None] * err)[:, None, :]

        root = rec[b, halves[b]].clone()
        for n in range(replays[b]):
            key, value = kv_all[b, halves[b], :, n, :DG], kv_all[b, halves[b], :, n, DG:]
            x = scal_all[b, halves[b], :, n]
            root = after(root, key * x[:, 2:3], value, x[:, 0], x[:, 1])
        known = {(): root}
        for i in range(T):
            path = tuple(paths[i])
            for n in range(len(path)):
                if path[:n + 1] not in known:
                    j = path[n]
                    known[path[:n + 1]] = after(known[path[:n]], k[j] * rk[j][:, None], v[j], gamma[j], beta[j])
            out[b, i] = (known[path] * qn[i][:, :, None]).sum(1)
        known.clear()
        out[b] = out[b] / torch.sqrt((out[b] ** 2).mean(-1, keepdim=True) + EPS) * s["norm_w"].double() * z / (1 + torch.exp(-z))
        to = 1 - halves[b]
        rec[b, to] = root
        keys = held[:, hk * DG:2 * hk * DG].view(T, hk, DG)[:, head]
        kv_all[b, to, :, :T] = torch.cat([keys, held[:, 2 * hk * DG:].view(T, hv, DG)], -1).transpose(0, 1)
        scal_all[b, to, :, :T] = torch.stack([gamma, beta, rk, torch.zeros_like(rk)], -1).transpose(0, 1)
        start = 0 if offs[b] >= W else W
        win[b, start:start + TAPS - 1] = window
        win[b, start + TAPS - 1:start + TAPS - 1 + T] = proj[b, :, :C]
    return [out.view(B, T, hv * DG), rec, win, kv_all, scal_all]
