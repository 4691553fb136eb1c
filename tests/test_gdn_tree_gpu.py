"""The Gated DeltaNet layer over a tree of drafts (lollm_gdn_layer_tree) against the definition in 64
bits: every node's own path from the root, walked alone."""

import pytest
import torch

D, K, EPS = 128, 4, 1e-6


def tree(B, T, spread, seed):
    g = torch.Generator().manual_seed(seed)
    words = torch.zeros(B, T, dtype=torch.int64)
    for b in range(B):
        for i in range(T):
            p = i - 1 - int(torch.randint(0, min(spread, i) if i else 1, (), generator=g)) if i else -1
            if spread > 3 and int(torch.randint(0, 9, (), generator=g)) == 0:
                p = -1
            w = (int(words[b, p]) if p >= 0 else 0) | 1 << i
            words[b, i] = w - (1 << 64) if w >= 1 << 63 else w
    return words


def layer(B, T, Hk, Hv, slots, seed, replay_max=3):
    g = torch.Generator().manual_seed(seed)
    C, W = 2 * Hk * D + Hv * D, K - 1 + slots
    P = -(-(C + Hv * D + 2 * Hv) // 8) * 8
    rn = lambda *s: torch.randn(*s, generator=g)   # noqa: E731
    kv = torch.nn.functional.silu(rn(B, 2, Hv, slots, 2 * D)).bfloat16()
    norm = torch.rsqrt(kv[..., :D].float().square().sum(-1) + EPS)
    sc = torch.stack([torch.exp(-torch.rand(B, 2, Hv, slots, generator=g)), torch.sigmoid(rn(B, 2, Hv, slots)), norm,
                      torch.zeros_like(norm)], -1)
    half = torch.randint(0, 2, (B,), generator=g)
    return {"proj": rn(B, T, P).bfloat16(), "conv_w": (0.3 * rn(C, K)).bfloat16(),
            "A_log": torch.log(torch.rand(Hv, generator=g) * 1.9 + 0.1), "dt_bias": 0.5 * rn(Hv),
            "norm_w": (1 + 0.1 * rn(D)).bfloat16(), "win": rn(B, 2 * W, C).bfloat16(),
            "conv_off": (half * W + torch.randint(0, slots + 1, (B,), generator=g)).int(),
            "rec": 0.1 * rn(B, 2, Hv, D, D), "rec_half": half.int(),
            "rep": torch.cat([kv.view(torch.uint8), sc.view(torch.uint8)], -1).contiguous(),
            "replay": torch.randint(0, min(slots, replay_max) + 1, (B,), generator=g).int()}


def call(s, words, B, T, Hk, Hv, fresh=False, **kw):
    """(out, the state tensors after the call, on the CPU)"""
    from lollm_amd import ops
    d = {n: t.cuda() for n, t in s.items()}
    out = ops.gdn_layer(d["proj"], d["conv_w"], d["A_log"], d["dt_bias"], d["norm_w"], d["win"], d["conv_off"], d["rec"],
                        d["rec_half"], d["rep"], d["replay"], fresh, B, T, Hk, Hv, D, K, EPS, tree=words.cuda(), **kw)
    return out.cpu(), {n: d[n].cpu() for n in ("win", "rec", "rep")}


def after(state, k, v, gamma, beta):
    u = (v - gamma[:, None] * (state * k[:, :, None]).sum(1)) * beta[:, None]
    return gamma[:, None, None] * state + k[:, :, None] * u[:, None]


def reference(s, words, B, T, Hk, Hv, slots, fresh=False):
    """In 64 bits: outputs, committed states, and per node (k and v before their rounding, gamma,
    beta, 1 / |k|)."""
    C, W = 2 * Hk * D + Hv * D, K - 1 + slots
    per = torch.arange(Hv) // (Hv // Hk)
    outs, states, recs = [], [], []
    for b in range(B):
        off, half, n = int(s["conv_off"][b]), int(s["rec_half"][b]), int(s["replay"][b])
        window, proj = s["win"][b, off:off + K - 1].double(), s["proj"][b].double()
        root = torch.zeros(Hv, D, D, dtype=torch.float64) if fresh else s["rec"][b, half].double()
        kv = s["rep"][b, half, ..., :4 * D].contiguous().view(torch.bfloat16).double()
        sc = s["rep"][b, half, ..., 4 * D:].contiguous().view(torch.float32).double()
        for j in range(0 if fresh else n):
            root = after(root, kv[:, j, :D] * sc[:, j, 2:3], kv[:, j, D:], sc[:, j, 0], sc[:, j, 1])
        paths = [[j for j in range(i) if (int(words[b, i]) >> j) & 1] + [i] for i in range(T)]
        act = torch.zeros(T, C, dtype=torch.float64)
        for i in range(T):
            line = torch.cat([window, proj[paths[i], :C]])[-K:]
            act[i] = (line * s["conv_w"].double().t()).sum(0)
        act = act * torch.sigmoid(act)
        held = act.float().bfloat16().double()
        q, k = held[:, :Hk * D].view(T, Hk, D)[:, per], held[:, Hk * D:2 * Hk * D].view(T, Hk, D)[:, per]
        v = held[:, 2 * Hk * D:].view(T, Hv, D)
        z = proj[:, C:C + Hv * D].view(T, Hv, D)
        beta = torch.sigmoid(proj[:, C + Hv * D:C + Hv * D + Hv])
        a = proj[:, C + Hv * D + Hv:C + Hv * D + 2 * Hv] + s["dt_bias"].double()
        gamma = torch.exp(-torch.exp(s["A_log"].double()) * torch.nn.functional.softplus(a, threshold=1e9))
        rk = 1 / torch.sqrt((k * k).sum(-1) + EPS)
        qn = q / torch.sqrt((q * q).sum(-1, keepdim=True) + EPS) * D ** -0.5
        known = {(): root}
        o = torch.zeros(T, Hv, D, dtype=torch.float64)
        for i in range(T):
            p = tuple(paths[i])
            for m in range(len(p)):
                if p[:m + 1] not in known:
                    j = p[m]
                    known[p[:m + 1]] = after(known[p[:m]], k[j] * rk[j][:, None], v[j], gamma[j], beta[j])
            o[i] = (known[p] * qn[i][:, :, None]).sum(1)
        y = o / torch.sqrt((o * o).mean(-1, keepdim=True) + EPS) * s["norm_w"].double() * z * torch.sigmoid(z)
        keys = act[:, Hk * D:2 * Hk * D].view(T, Hk, D)[:, per]
        outs.append(y.view(T, Hv * D))
        states.append(root)
        recs.append((keys, act[:, 2 * Hk * D:].view(T, Hv, D), gamma, beta, rk))
    return torch.stack(outs), torch.stack(states), recs


def check(s, words, B, T, Hk, Hv, slots, fresh=False):
    out, st = call(s, words, B, T, Hk, Hv, fresh)
    ref, states, recs = reference(s, words, B, T, Hk, Hv, slots, fresh)
    # the output's rounding, 2^-9 of it (twice), and the operands' of the two products with the state,
    # 2^-17 of the terms, whose sums over 128 are at most some 30 times their typical result: 2^-11 of a
    # head's root mean square
    rms = ref.view(B, T, Hv, D).square().mean(-1, keepdim=True).sqrt().expand(-1, -1, -1, D).reshape(ref.shape)
    err = (out.double() - ref).abs()
    assert (err <= ref.abs() * 2 ** -8 + rms * 2 ** -8).all(), f"largest {(err / rms).max().item()} of the rms"
    W = K - 1 + slots
    for b in range(B):
        half, off = int(s["rec_half"][b]), int(s["conv_off"][b])
        # the committed half and everything behind the nodes' rows stay as they were
        assert torch.equal(st["rec"][b, half], s["rec"][b, half])
        assert torch.equal(st["rep"][b, half], s["rep"][b, half])
        assert torch.equal(st["rep"][b, 1 - half, :, T:], s["rep"][b, 1 - half, :, T:])
        # fp32 steps of the rule: each of the (at most 3) records rounds sums of 128 products
        got = st["rec"][b, 1 - half].double()
        assert (got - states[b]).abs().max() <= 2 ** -17 * states[b].abs().max().clamp(min=1e-3)
        keys, v, gamma, beta, rk = recs[b]
        kv = st["rep"][b, 1 - half, :, :T, :4 * D].contiguous().view(torch.bfloat16).double().transpose(0, 1)
        for got, want in ((kv[..., :D], keys), (kv[..., D:], v)):
            # one rounding of fp32 sums of four products (2^-21 of their size covers those)
            assert ((got - want).abs() <= want.abs() * 2 ** -8 * 1.01 + 2 ** -18).all()
        sc = st["rep"][b, 1 - half, :, :T, 4 * D:].contiguous().view(torch.float32).double().transpose(0, 1)
        # gamma = e^g: a relative error d of g, a product of e^A_log and a softplus in fp32 (2^-22 each, 2^-24
        # of |A_log| < 31 for the first, and g's own rounding: below 2^-20), moves e^g by |g| d of itself
        room = 2 ** -17 + 2 ** -20 * gamma.clamp(min=1e-300).log().abs()
        assert ((sc[..., 0] - gamma).abs() <= gamma * room + 1e-30).all()
        assert ((sc[..., 1] - beta).abs() <= beta * 2 ** -17).all()
        # 1 / |k| of rounded keys, which may have gone the other way at a tie
        assert ((sc[..., 2] - rk).abs() <= rk * 2 ** -14).all() and (sc[..., 3] == 0).all()
        base = 0 if off >= W else W
        want = torch.cat([s["win"][b, off:off + K - 1], s["proj"][b, :, :st["win"].shape[2]]])
        assert torch.equal(st["win"][b, base:base + K - 1 + T], want)
        rest = torch.ones(2 * W, dtype=torch.bool)
        rest[base:base + K - 1 + T] = False
        assert torch.equal(st["win"][b, rest], s["win"][b, rest])


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,Hk,Hv,slots,spread", [
    (1, 1, 1, 1, 1, 1), (2, 1, 2, 4, 4, 1), (1, 2, 1, 2, 2, 1), (2, 7, 8, 16, 7, 3), (3, 8, 2, 2, 9, 8),
    (2, 15, 2, 4, 16, 4), (2, 16, 2, 4, 16, 1), (2, 16, 2, 8, 20, 64), (2, 17, 1, 2, 17, 5), (1, 31, 2, 4, 64, 2),
    (2, 32, 2, 4, 32, 9), (1, 33, 2, 2, 40, 6), (2, 48, 1, 3, 48, 64), (1, 63, 2, 4, 64, 20), (2, 64, 2, 4, 64, 1),
    (1, 64, 2, 4, 64, 64)])
def test_gdn_tree_matches_64_bits(B, T, Hk, Hv, slots, spread):
    print("case gdn tree", B, T, Hk, Hv, slots, spread, flush=True)
    check(layer(B, T, Hk, Hv, slots, T + slots), tree(B, T, spread, T), B, T, Hk, Hv, slots)


@pytest.mark.gpu
@pytest.mark.parametrize("T", (3, 20, 50))
def test_gdn_tree_fresh_sequences(T):
    """No committed state: zeros, whatever the buffers hold (NaN here)."""
    B, Hk, Hv, slots = 2, 2, 4, 50
    s = layer(B, T, Hk, Hv, slots, 1)
    words = tree(B, T, 5, 2)
    print("case gdn tree fresh", T, flush=True)
    check(s, words, B, T, Hk, Hv, slots, fresh=True)
    clean, _ = call(s, words, B, T, Hk, Hv, fresh=True)
    s["rec"][:] = float("nan")
    dirty, st = call(s, words, B, T, Hk, Hv, fresh=True)
    assert torch.equal(clean, dirty)
    for b in range(B):
        assert (st["rec"][b, 1 - int(s["rec_half"][b])] == 0).all()


@pytest.mark.gpu
def test_gdn_tree_many_records_and_strong_decays():
    """All slots replayed; decays whose products leave fp32's range, and none at all."""
    B, T, Hk, Hv, slots = 2, 30, 2, 4, 33
    s = layer(B, T, Hk, Hv, slots, 8)
    s["replay"][:] = torch.tensor([slots, 17])
    s["A_log"][:] = torch.tensor([4.0, -30.0, 0.0, 2.0])
    # 33 steps of the rule, each within 2^-22 of the state: three records' 2^-17 covers them (checked there)
    print("case gdn tree decays", flush=True)
    check(s, tree(B, T, 1, 3), B, T, Hk, Hv, slots)
    check(s, tree(B, T, 7, 3), B, T, Hk, Hv, slots)


@pytest.mark.gpu
def test_gdn_tree_bits_of_no_ancestor_count_for_nothing():
    """Bits at and past the node itself."""
    B, T, Hk, Hv, slots = 2, 20, 2, 4, 20
    s, words = layer(B, T, Hk, Hv, slots, 5), tree(B, T, 6, 1)
    want, st = call(s, words, B, T, Hk, Hv)
    past = words.clone()
    for i in range(T):
        past[:, i] = (words[:, i] & ((1 << i) - 1)) | (-1 << (i + 1))
    print("case gdn tree bits", flush=True)
    got, st2 = call(s, past, B, T, Hk, Hv)
    assert torch.equal(want, got) and all(torch.equal(st[n], st2[n]) for n in st)


@pytest.mark.gpu
def test_gdn_tree_that_is_a_chain_is_the_short_call():
    """The plain short call rounds the convolution's output before the activation and beta to bf16 besides:
    outputs within a few bf16 steps of each other's typical size, records within two."""
    from lollm_amd import ops
    B, T, Hk, Hv, slots = 3, 5, 2, 4, 8
    s = layer(B, T, Hk, Hv, slots, 2)
    words = tree(B, T, 1, 1)
    got, st = call(s, words, B, T, Hk, Hv)
    d = {n: t.cuda() for n, t in s.items()}
    want = ops.gdn_layer(d["proj"], d["conv_w"], d["A_log"], d["dt_bias"], d["norm_w"], d["win"], d["conv_off"],
                         d["rec"], d["rec_half"], d["rep"], d["replay"], False, B, T, Hk, Hv, D, K, EPS).cpu()
    rms = want.double().square().mean().sqrt()
    assert (got.double() - want.double()).square().mean().sqrt() <= 2 ** -6 * rms
    assert torch.equal(st["win"], d["win"].cpu())
    for b in range(B):
        o = 1 - int(s["rec_half"][b])
        a, c = (x[b, o, :, :T, :4 * D].contiguous().view(torch.bfloat16).double() for x in (st["rep"], d["rep"].cpu()))
        assert ((a - c).abs() <= c.abs() * 2 ** -6 + 2 ** -10).all()


@pytest.mark.gpu
def test_gdn_tree_in_a_graph():
    from lollm_amd import ops
    B, T, Hk, Hv, slots = 2, 12, 2, 4, 12
    s = layer(B, T, Hk, Hv, slots, 6)
    trees = [tree(B, T, 4, 1), tree(B, T, 1, 2)]
    want = [call(s, w, B, T, Hk, Hv)[0] for w in trees]
    d = {n: t.cuda() for n, t in s.items()}
    words = trees[0].cuda()

    def run():
        return ops.gdn_layer(d["proj"], d["conv_w"], d["A_log"], d["dt_bias"], d["norm_w"], d["win"], d["conv_off"],
                             d["rec"], d["rec_half"], d["rep"], d["replay"], False, B, T, Hk, Hv, D, K, EPS, tree=words)
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for turn in range(4):
        words.copy_(trees[turn % 2])
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu(), want[turn % 2])
        run()


@pytest.mark.gpu
def test_gdn_tree_refusals():
    B, T, Hk, Hv, slots = 1, 6, 2, 4, 6
    s, words = layer(B, T, Hk, Hv, slots, 6), tree(B, T, 2, 1)
    for change in ({"rep": s["rep"][:, :, :, :5].contiguous()}, {"win": s["win"][:, :16].contiguous()},
                   {"proj": s["proj"][..., :-8].contiguous()}, {"conv_w": s["conv_w"][:, :3].contiguous()},
                   {"proj": s["proj"].float()}, {"win": s["win"][..., :-8].contiguous()}, {"A_log": s["A_log"][:2]},
                   {"norm_w": s["norm_w"].float()}):
        with pytest.raises((ValueError, TypeError)):
            call({**s, **change}, words, B, T, Hk, Hv)
    for w in (words.int(), words[:, :5].contiguous(), torch.cat([words, words])):
        with pytest.raises((ValueError, TypeError)):
            call(s, w, B, T, Hk, Hv)
    big = layer(1, 65, 1, 1, 65, 1)
    with pytest.raises(ValueError):
        call(big, torch.ones(1, 65, dtype=torch.int64), 1, 65, 1, 1)


def test_gdn_tree_entry_point_checks_before_any_launch():
    from lollm_amd import _lib
    p = 4096     # an address that no check reads
    f = _lib.lib().lollm_gdn_layer_tree

    def rc(tree=p, T=6, slots=6, win=9, Hk=2, Hv=4, Dk=128, taps=4, stride=2048, proj=p):
        return f(proj, stride, p, p, p, p, p, p, win, p, p, p, p, slots, 0, tree, p, 1, T, Hk, Hv, Dk, Dk, taps, 1e-6, None)

    assert rc(tree=None) == 1 and rc(tree=p + 4) == 1 and rc(slots=5) == 1 and rc(win=8) == 1
    assert rc(T=65, slots=65, win=68) == 2 and rc(Dk=64) == 2 and rc(taps=3) == 2
    assert rc(Hv=3) == 1 and rc(stride=1024) == 1 and rc(proj=p + 2) == 1 and rc(T=0) == 1
