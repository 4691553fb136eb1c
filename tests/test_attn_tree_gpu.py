"""Attention for a tree of drafted tokens over slabs and pages (lollm_attn_tree, lollm_attn_paged_tree)
against 64 bits, and the words of a tree (lollm_tree_masks)."""

import math

import pytest
import torch

D = 256


def tree(B, T, spread, seed):
    """(parents (B, T), words (B, T)): node i hangs on one of the `spread` nodes before it, some nodes
    on the context."""
    g = torch.Generator().manual_seed(seed)
    parents = torch.full((B, T), -1, dtype=torch.int32)
    words = torch.zeros(B, T, dtype=torch.int64)
    for b in range(B):
        for i in range(T):
            p = i - 1 - int(torch.randint(0, min(spread, i) if i else 1, (), generator=g)) if i else -1
            if spread > 3 and int(torch.randint(0, 9, (), generator=g)) == 0:
                p = -1
            parents[b, i] = p
            w = (int(words[b, p]) if p >= 0 else 0) | 1 << i
            words[b, i] = w - (1 << 64) if w >= 1 << 63 else w
    return parents, words


def inputs(B, T, hq, hkv, lens, seed):
    g = torch.Generator().manual_seed(seed)
    longest = max(max(lens), T)
    q = torch.randn(B, T, hq, D, generator=g).bfloat16()
    k = torch.randn(B, hkv, longest, D, generator=g).bfloat16()
    v = torch.randn(B, hkv, longest, D, generator=g).bfloat16()
    gate = torch.randn(B, T, hq, D, generator=g).bfloat16()
    return q, k, v, gate


def reference(q, k, v, gate, lens, words):
    """(output, sum of |terms|) in 64 bits, row by row; a row that sees nothing is 0."""
    B, T, hq, _ = q.shape
    rep = hq // k.shape[1]
    out, mag = torch.zeros(B, T, hq, D, dtype=torch.float64), torch.zeros(B, T, hq, D, dtype=torch.float64)
    for b in range(B):
        L = lens[b]
        if L == 0:
            continue
        seen = torch.zeros(T, L, dtype=torch.bool)
        for i in range(T):
            w = int(words[b, i])
            for j in range(L):
                n = j - (L - T)
                seen[i, j] = n < 0 or (n <= i and (w >> n) & 1)
        kk, vv = k[b, :, :L].double().repeat_interleave(rep, 0), v[b, :, :L].double().repeat_interleave(rep, 0)
        x = q[b].double().transpose(0, 1) @ kk.transpose(1, 2) / math.sqrt(D)
        x = x.masked_fill(~seen, -math.inf)
        p = torch.softmax(x, -1)
        p = torch.where(seen.any(-1)[None, :, None], p, torch.zeros_like(p))
        p = torch.where(seen, p, torch.zeros_like(p))
        out[b], mag[b] = (p @ vv).transpose(0, 1), (p @ vv.abs()).transpose(0, 1)
    s = 1.0 if gate is None else torch.sigmoid(gate.double())
    return out * s, mag * s


def close(got, ref, mag):
    """The output's rounding (2^-9 of it, twice) and the weights', bf16 at worst: 2^-9 of sum p |v|, twice."""
    err = (got.double().cpu().view(ref.shape) - ref).abs()
    bad = err > ref.abs() * 2 ** -8 + mag * 2 ** -8 + 1e-30
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, largest {err.max().item()}"


def to_pages(k, v, lens, page, bits, seed):
    """Pools with the sequences' rows in pages anywhere, what no sequence holds NaN (bf16) or the
    largest code; (k_pages, v_pages, scales or None x 2, table, values as the pages hold them)."""
    g = torch.Generator().manual_seed(seed)
    B, hkv, longest, _ = k.shape
    width = -(-longest // page)
    n = B * width + 2
    table = torch.randperm(n, generator=g)[:B * width].view(B, width).to(torch.int32)
    pools, scales, held = [], [], []
    for x in (k, v):
        rows = torch.zeros(B, hkv, width * page, D)
        rows[:, :, :longest] = x.float()
        pg = rows.view(B, hkv, width, page, D).permute(0, 2, 1, 3, 4)          # (B, width, hkv, page, D)
        if bits == 16:
            pool = torch.full((n, hkv, page, D), float("nan")).bfloat16()
            pool[table.long()] = pg.bfloat16()
            held.append(x)
            scales.append(None)
        else:
            s = torch.exp2(torch.ceil(torch.log2(pg.abs().amax((3, 4)) / 448 + 1e-30)).clamp(min=-20))
            codes = (pg / s[..., None, None]).to(torch.float8_e4m3fn)
            pool = torch.full((n, hkv, page, D), 126, dtype=torch.uint8)
            pool[table.long()] = codes.view(torch.uint8)
            pool = pool.view(torch.float8_e4m3fn)
            sc = torch.ones(n, hkv)
            sc[table.long()] = s
            scales.append(sc)
            back = codes.float() * s[..., None, None]
            held.append(back.permute(0, 2, 1, 3, 4).reshape(B, hkv, width * page, D)[:, :, :longest])
        pools.append(pool)
    for b in range(B):
        table[b, -(-lens[b] // page):] = -1
    return pools, scales, table, held


CASES = [  # B, T, q heads, kv heads, keys with the tree's, spread
    (1, 1, 2, 2, [1], 1), (1, 7, 8, 2, [138], 3), (2, 5, 4, 2, [5, 133], 2), (3, 16, 32, 4, [16, 300, 0], 6),
    (2, 33, 16, 2, [33, 160], 8), (1, 64, 8, 1, [64], 64), (2, 64, 32, 4, [400, 129], 20), (1, 63, 32, 1, [200], 20),
    (2, 9, 6, 2, [4, 9], 3), (9, 17, 16, 4, [17, 18, 40, 127, 128, 129, 145, 256, 300], 5),
    (1, 40, 2, 2, [1000], 9),
]


def run(kind, q, k, v, gate, lens, words, **kw):
    from lollm_amd import ops
    kl = torch.tensor(lens, dtype=torch.int32).cuda()
    w = words.cuda()
    B, T, hq, _ = q.shape
    if kind == "slab":
        return ops.attn_verify(q.cuda(), k.cuda(), v.cuda(), kl, None if gate is None else gate.reshape(B, T, hq * D).cuda(),
                               tree=w, **kw), k, v
    page, bits = kind
    (kp, vp), (ks, vs), table, (kh, vh) = to_pages(k, v, lens, page, bits, 5)
    args = {} if ks is None else {"k_scale": ks.cuda(), "v_scale": vs.cuda()}
    return ops.attn_paged(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), kl, None if gate is None else gate.cuda(),
                          tree=w, **args, **kw), kh, vh


KINDS = ("slab", (16, 16), (64, 16), (128, 16), (16, 8), (64, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("case", CASES, ids=str)
def test_attn_tree_matches_64_bits(case, kind):
    B, T, hq, hkv, lens, spread = case
    print("case tree attention", case, kind, flush=True)
    q, k, v, gate = inputs(B, T, hq, hkv, lens, sum(lens) + T)
    _, words = tree(B, T, spread, T)
    got, kh, vh = run(kind, q, k, v, gate, lens, words)
    close(got, *reference(q, kh, vh, gate, lens, words))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("B,T,hq,hkv", [(24, 33, 32, 4), (20, 64, 16, 2)])
def test_attn_tree_many_nodes(B, T, hq, hkv, kind):
    """Enough query rows for the tiles of long calls; no gate."""
    lens = [T + (37 * b) % 400 for b in range(B)]
    print("case tree attention", B, T, hq, hkv, kind, flush=True)
    q, k, v, _ = inputs(B, T, hq, hkv, lens, 3)
    _, words = tree(B, T, 12, 1)
    got, kh, vh = run(kind, q, k, v, None, lens, words)
    close(got, *reference(q, kh, vh, None, lens, words))


RAGGED = [(70, 12, 8, 1, [12 + (b * b * 7) % 300 if b % 5 else 0 for b in range(70)]),       # more sequences than lanes
          (4, 63, 32, 4, [0, 63, 900, 5000]), (3, 33, 16, 2, [33, 2000, 40]), (1, 64, 32, 4, [3000]),
          (2, 24, 32, 4, [24, 24]), (65, 17, 8, 1, [17] * 64 + [1500])]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ((16, 16), (128, 16), (16, 8), (128, 8)), ids=str)
@pytest.mark.parametrize("case", RAGGED, ids=lambda c: f"{c[0]}x{c[1]}")
def test_attn_tree_keys_dealt_out_by_length(case, kind):
    """Query tiles whose keys go to workgroups by the sequences' lengths: none, few and many keys, empty
    sequences between, one that takes nearly all."""
    B, T, hq, hkv, lens = case
    print("case tree attention by length", B, T, hq, hkv, kind, flush=True)
    q, k, v, gate = inputs(B, T, hq, hkv, lens, 8)
    _, words = tree(B, T, 9, 3)
    got, kh, vh = run(kind, q, k, v, gate, lens, words)
    again, _, _ = run(kind, q, k, v, gate, lens, words)
    assert torch.equal(got, again)
    close(got, *reference(q, kh, vh, gate, lens, words))
    for b in range(B):
        if lens[b] == 0:
            assert (got[b] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS, ids=str)
def test_attn_tree_any_words(kind):
    """Words that are no tree's: rows that see no node (and, with nothing cached, nothing at all: zeros),
    bits past the query itself and past T, which count for nothing; keys of unseen nodes that are NaN."""
    B, T, hq, hkv = 2, 12, 8, 2
    lens = [T, 90]
    q, k, v, gate = inputs(B, T, hq, hkv, lens, 9)
    g = torch.Generator().manual_seed(4)
    words = torch.randint(-2 ** 62, 2 ** 62, (B, T), generator=g)
    words[0, 3] = 0
    words[1, 5] = -1 << 20
    words &= ~(1 << 7)          # no query sees node 7
    for b in range(B):
        if kind == "slab" or kind[1] == 16:
            k[b, :, lens[b] - T + 7] = float("nan")
    clean = torch.where(k.isnan(), torch.zeros_like(k), k)
    print("case tree attention, any words", kind, flush=True)
    got, kh, vh = run(kind, q, k, v, gate, lens, words)
    kh = clean if kind == "slab" or kind[1] == 16 else kh
    ref, mag = reference(q, kh, vh, gate, lens, words)
    assert (ref[0, 3] == 0).all()
    close(got, ref, mag)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ("slab", (64, 16), (64, 8)), ids=str)
def test_attn_tree_that_is_a_chain_equals_the_plain_call(kind):
    """Same kernels, same grid: the same bits."""
    from lollm_amd import ops
    B, T, hq, hkv = 3, 6, 32, 4
    lens = [6, 200, 1500]
    q, k, v, gate = inputs(B, T, hq, hkv, lens, 2)
    words = ((torch.ones(1, dtype=torch.int64) << torch.arange(1, T + 1)) - 1).expand(B, T).contiguous()
    got, _, _ = run(kind, q, k, v, gate, lens, words, grid=200)
    kl = torch.tensor(lens, dtype=torch.int32).cuda()
    if kind == "slab":
        want = ops.attn_verify(q.cuda(), k.cuda(), v.cuda(), kl, gate.reshape(B, T, hq * D).cuda(), grid=200)
    else:
        (kp, vp), (ks, vs), table, _ = to_pages(k, v, lens, *kind, 5)
        args = {} if ks is None else {"k_scale": ks.cuda(), "v_scale": vs.cuda()}
        want = ops.attn_paged(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), kl, gate.cuda(), grid=200, **args)
    assert torch.equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ("slab", (32, 16), (32, 8)), ids=str)
def test_attn_tree_in_a_graph(kind):
    """A captured call follows the words and lengths that it is replayed over."""
    from lollm_amd import ops
    B, T, hq, hkv = 2, 20, 16, 2
    lens, other = [20, 700], [333, 41]
    q, k, v, gate = inputs(B, T, hq, hkv, [700, 700], 6)
    _, w1 = tree(B, T, 6, 1)
    _, w2 = tree(B, T, 2, 2)
    kl, w = torch.tensor(lens, dtype=torch.int32).cuda(), w1.cuda()
    if kind == "slab":
        args = (q.cuda(), k.cuda(), v.cuda(), kl, gate.reshape(B, T, hq * D).cuda())
        call = lambda: ops.attn_verify(*args, tree=w)   # noqa: E731
    else:
        (kp, vp), (ks, vs), table, _ = to_pages(k, v, [700, 700], *kind, 5)
        args = (q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), kl, gate.cuda())
        kw = {} if ks is None else {"k_scale": ks.cuda(), "v_scale": vs.cuda()}
        call = lambda: ops.attn_paged(*args, tree=w, **kw)   # noqa: E731
    want = []
    for ln, ww in ((lens, w1), (other, w2)):
        kl.copy_(torch.tensor(ln, dtype=torch.int32))
        w.copy_(ww)
        want.append(call().clone())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for turn in range(4):
        kl.copy_(torch.tensor((lens, other)[turn % 2], dtype=torch.int32))
        w.copy_((w1, w2)[turn % 2])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[turn % 2])
        call()


@pytest.mark.gpu
def test_attn_tree_refusals():
    from lollm_amd import ops
    dev = "cuda"
    q = torch.zeros(1, 65, 4, D, dtype=torch.bfloat16, device=dev)
    k = torch.zeros(1, 2, 128, D, dtype=torch.bfloat16, device=dev)
    kl = torch.full((1,), 65, dtype=torch.int32, device=dev)
    pages = torch.zeros(3, 2, 64, D, dtype=torch.bfloat16, device=dev)
    table = torch.zeros(1, 2, dtype=torch.int32, device=dev)
    words = torch.ones(1, 65, dtype=torch.int64, device=dev)
    for w, T in ((words, 65), (words[:, :4].int(), 4), (words[:, :5], 4), (words[:, :4].cpu(), 4),
                 (torch.ones(2, 4, dtype=torch.int64, device=dev), 4)):
        with pytest.raises((ValueError, TypeError)):
            ops.attn_verify(q[:, :T].contiguous(), k, k, kl, tree=w)
        with pytest.raises((ValueError, TypeError)):
            ops.attn_paged(q[:, :T].contiguous(), pages, pages, table, kl, tree=w)
    with pytest.raises(ValueError):
        ops.attn_paged_workspace_bytes(1, 65, 4, 2, D, tree=True)
    with pytest.raises(RuntimeError):
        ops.attn_paged(q[:, :4].contiguous(), pages, pages, table, kl, tree=words[:, :4].contiguous(),
                       workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    for bad in (torch.zeros(1, 65, dtype=torch.int32, device=dev), torch.zeros(4, dtype=torch.int32, device=dev),
                torch.zeros(1, 4, dtype=torch.int64, device=dev), torch.zeros(1, 4, dtype=torch.int32)):
        with pytest.raises((ValueError, TypeError)):
            ops.tree_masks(bad)


@pytest.mark.gpu
@pytest.mark.parametrize("T,spread", [(1, 1), (2, 1), (7, 2), (33, 5), (63, 64), (64, 1), (64, 64)])
def test_tree_masks(T, spread):
    from lollm_amd import ops
    B = 5
    print("case words", T, spread, flush=True)
    parents, words = tree(B, T, spread, 8)
    mask, depth = ops.tree_masks(parents.cuda())
    assert torch.equal(mask.cpu(), words)
    assert depth.cpu().tolist() == [[bin(int(w) & (1 << 64) - 1).count("1") - 1 for w in row] for row in words]


@pytest.mark.gpu
def test_tree_masks_takes_what_is_no_node_for_the_context():
    from lollm_amd import ops
    parents = torch.tensor([[0, 0, 2, 7, -5, 4, 2 ** 31 - 1, -2 ** 31]], dtype=torch.int32).cuda()
    mask, depth = ops.tree_masks(parents)
    assert mask.tolist() == [[1, 3, 4, 8, 16, 48, 64, 128]]
    assert depth.tolist() == [[0, 1, 0, 0, 0, 1, 0, 0]]


def test_tree_entry_points_check_before_any_launch():
    from lollm_amd import _lib
    L = _lib.lib()
    p = 4096     # an address that no check reads
    assert L.lollm_tree_masks(None, p, None, 1, 4, None) == 1
    assert L.lollm_tree_masks(p, p, None, 1, 65, None) == 2
    assert L.lollm_tree_masks(p, p + 4, None, 1, 4, None) == 1
    assert L.lollm_tree_masks(p, p, None, 0, 4, None) == 1
    tail = (4, 2, D, 128, 2 * 128 * D, 128 * D, 8, 0.0625, None)
    assert L.lollm_attn_tree(p, p, p, p, None, None, p, p, 1 << 30, 1, 4, *tail) == 1
    assert L.lollm_attn_tree(p, p, p, p, p, None, p, p, 1 << 30, 1, 65, *tail) == 2
    assert L.lollm_attn_tree(p, p, p, p, p + 4, None, p, p, 1 << 30, 1, 4, *tail) == 1
    head = (p, p, p, None, None, 0, p, 2, 2, 3, 64, p)
    assert L.lollm_attn_paged_tree(*head, None, None, 0, 0, p, p, 1 << 30, 1, 4, 4, 2, D, 8, 0.0625, None) == 1
    assert L.lollm_attn_paged_tree(*head, p, None, 0, 0, p, p, 1 << 30, 1, 65, 4, 2, D, 8, 0.0625, None) == 2
    assert L.lollm_attn_paged_tree_workspace_bytes(1, 65, 4, 2, D, 0, 8) == -1


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,hq,hkv,lens,max_len", [(2, 5, 8, 2, [131, 40], 131), (1, 16, 32, 4, [600], 9001),
                                                     (3, 7, 8, 1, [7, 0, 1021], 1021), (1, 3, 2, 2, [3], 3)], ids=str)
def test_attn_tree_slabs_that_end_anywhere(B, T, hq, hkv, lens, max_len):
    """Capacities that no block divides, sequences that fill them, long slabs with few keys; rows past the
    lengths are NaN."""
    from lollm_amd import ops
    print("case tree attention, slabs of", max_len, lens, flush=True)
    q, k, v, gate = inputs(B, T, hq, hkv, [max_len] * B, 4)
    _, words = tree(B, T, 4, 2)
    kc, vc = k.clone(), v.clone()
    for b in range(B):
        kc[b, :, lens[b]:] = float("nan")
        vc[b, :, lens[b]:] = float("nan")
    got = ops.attn_verify(q.cuda(), kc.cuda(), vc.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(),
                          gate.reshape(B, T, hq * D).cuda(), tree=words.cuda())
    close(got, *reference(q, k, v, gate, lens, words))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", (16, 8))
def test_attn_tree_parts_of_rows_of_any_size(bits):
    """Keys dealt out in parts whose values differ by powers of two from part to part and head to head, from
    2^-40 to 2^60 in bf16: a part's pieces are in units of their own."""
    B, T, hq, hkv, lens = 2, 24, 32, 4, [1500, 777]
    print("case tree attention, sizes of values", bits, flush=True)
    q, k, v, gate = inputs(B, T, hq, hkv, lens, 21)
    step = torch.arange(1500) // 96
    size = (step * 7 % 11 - 4) * (10 if bits == 16 else 1)
    v = (v.float() * torch.exp2(size.float())[None, None, :, None] * torch.tensor([1.0, 2.0 ** 10, 2.0 ** -10, 1.0])[None, :, None, None]).bfloat16()
    _, words = tree(B, T, 6, 5)
    got, kh, vh = run((64, bits), q, k, v, gate, lens, words)
    close(got, *reference(q, kh, vh, gate, lens, words))
