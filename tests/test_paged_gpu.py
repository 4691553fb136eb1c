"""The paged cache's kernels against their definitions in 64 bits (tests/paged_oracle.py): pages
of every size in bf16 and 8 bits, unmapped pages, rows past the lengths, odd sizes, strides; the
refusals of their wrappers; append and attention together, as a decoder uses them, eager and in
a replayed graph.  Tolerances count roundings: they are derived beside the oracle."""

import pytest
import torch

import paged_oracle as O

pytestmark = pytest.mark.gpu
D = 256
EPS = 1e-6


def gen(seed):
    return torch.Generator().manual_seed(seed)


def pool(g, n, hkv, P, bits, junk=True):
    """A pool whose rows hold NaN (a caller overwrites the ones that live) or random rows."""
    x = torch.randn(n, hkv, P, D, generator=g) * torch.exp2(torch.randint(-3, 4, (n, hkv, 1, 1), generator=g).float())
    if bits == 16:
        return x.bfloat16(), None
    s = torch.tensor([[O.pow2_scale(float(x[i, h].abs().max())) for h in range(hkv)] for i in range(n)])
    return (x / s[:, :, None, None]).to(torch.float8_e4m3fn), s.float()


def attend_case(seed, B, T, Hq, Hkv, lens, P, bits, holes=(), spare=2):
    """Sequences in shuffled pages; every row that no query may see is NaN."""
    g = gen(seed)
    width = max(1, max(-(-L // P) for L in lens))
    n = sum(-(-L // P) for L in lens) + spare
    first = lens[0] == 0 or (0, 0) in holes            # page 0 of the pool is nobody's now and then
    k, ks = pool(g, n, Hkv, P, bits)
    v, vs = pool(g, n, Hkv, P, bits)
    perm = [p for p in torch.randperm(n, generator=g).tolist() if not first or p]
    table = torch.full((B, width), -1, dtype=torch.int32)
    dead = torch.ones(n, P, dtype=torch.bool)
    for b, L in enumerate(lens):
        for i in range(-(-L // P)):
            if (b, i) in holes:
                table[b, i] = (-1, n, n + 100, -2 ** 31)[i % 4]
                continue
            p = perm.pop()
            table[b, i] = p
            dead[p, :max(0, min(P, L - i * P))] = False
    if bits == 8:                                      # pages of nobody have no scale either
        nobody = dead.all(1)
        ks[nobody], vs[nobody] = float("nan"), float("nan")
    nan = torch.tensor(float("nan"))
    for x in (k, v):
        x.view(torch.uint8 if bits == 8 else torch.bfloat16).masked_fill_(
            dead[:, None, :, None], 0x7f if bits == 8 else nan)
    q = (2 * torch.randn(B, T, Hq, D, generator=g)).bfloat16()
    qkv = torch.randn(B, T, Hq * 2 * D + 2 * Hkv * D, generator=g).bfloat16()
    return q, k, v, table, torch.tensor(lens, dtype=torch.int32), qkv, ks, vs


def gates(qkv, Hq):
    B, T, _ = qkv.shape
    return qkv[:, :, :Hq * 2 * D].view(B, T, Hq, 2 * D)[..., D:]


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def clean(pages):
    """The oracle's pages: what must not be used as zeros."""
    return pages.float().nan_to_num(0.0).to(pages.dtype) if pages.dtype != torch.float8_e4m3fn else \
        pages.float().nan_to_num(0.0).to(torch.float8_e4m3fn)


def check_attention(case, Hq, **kw):
    from lollm_amd import ops
    q, k, v, table, lens, qkv, ks, vs = case
    gate = gates(qkv, Hq)
    ref, tol = O.attention(q, clean(k), clean(v), table, lens, gate, ks, vs, kw.get("scale"))
    qd, kd, vd, td, ld, gd, ksd, vsd = cuda(q, k, v, table, lens, qkv, ks, vs)
    out = ops.attn_paged(qd, kd, vd, td, ld, gates(gd, Hq), k_scale=ksd, v_scale=vsd, **kw)
    torch.cuda.synchronize()
    # nothing of what lay in the workspace counts
    ws = torch.full((ops.attn_paged_workspace_bytes(*q.shape[:3], k.shape[1], D, k.dtype, kw.get("grid", 0)),), 255,
                    dtype=torch.uint8, device="cuda")
    again = ops.attn_paged(qd, kd, vd, td, ld, gates(gd, Hq), k_scale=ksd, v_scale=vsd, workspace=ws, **kw)
    assert torch.equal(again, out)
    got = out.cpu().double()
    assert got.isfinite().all()
    worst = ((got - ref).abs() - tol).max()
    assert worst <= 0, f"off by {float(worst)} more than {float(tol.max())}"
    return out


CASES = [
    # B, T, Hq, Hkv, lens, page, grid
    (1, 1, 8, 2, [1], 16, 0),
    (2, 1, 4, 2, [131, 0], 16, 0),                   # an idle slot
    (3, 1, 32, 4, [5, 128, 1000], 64, 0),
    (3, 4, 16, 2, [4, 37, 700], 32, 0),
    (2, 2, 8, 2, [2, 129], 128, 3),
    (2, 8, 16, 2, [8, 300], 16, 4),                  # two query blocks a pair
    (5, 3, 8, 2, [3, 64, 65, 190, 7], 64, 7),        # ranges over several sequences
    (3, 4, 16, 2, [4, 600, 130], 32, 1),             # one workgroup walks every pair
    (3, 4, 16, 2, [4, 600, 130], 16, 1024),          # more workgroups than blocks
    (2, 5, 8, 1, [3, 0], 16, 0),                     # fewer keys than queries: rows that see none
    (1, 1, 32, 1, [9000], 128, 1),                   # more blocks than a lookup holds
    (2, 3, 6, 2, [77, 4100], 64, 2),                 # 3 query heads a KV head
    (1, 33, 4, 2, [50], 32, 0),
    (2, 70, 8, 2, [70, 213], 16, 0),                 # query tiles
    (1, 100, 8, 2, [1501], 16, 0),                   # their keys in parts
    (2, 67, 32, 4, [2100, 67], 64, 0),               # one sequence in parts, one whole
    (3, 65, 6, 2, [700, 0, 65], 32, 0),              # an idle slot; 3 query heads a KV head
    (1, 600, 32, 4, [1111], 128, 0),                 # several tiles a part
]


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("B,T,Hq,Hkv,lens,P,grid", CASES)
def test_attention(B, T, Hq, Hkv, lens, P, grid, bits):
    print(f"case {B} {T} {Hq}/{Hkv} {lens} page {P} grid {grid} bits {bits}", flush=True)
    check_attention(attend_case(sum(lens) + T + P, B, T, Hq, Hkv, lens, P, bits), Hq, grid=grid)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("P", [16, 32, 64, 128])
def test_attention_unmapped_pages(P, bits):
    print(f"case holes page {P} bits {bits}", flush=True)
    lens = [10 * P, 3 * P + 5, 2 * P, 1]
    # pages inside, the first, a whole sequence, the only one
    holes = {(0, 1), (0, 4), (0, 5), (0, 6), (0, 7), (1, 0), (2, 0), (2, 1), (3, 0)}
    out = check_attention(attend_case(P, 4, 2, 8, 2, lens, P, bits, holes), 8)
    assert (out[2] == 0).all() and (out[3] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("P", [16, 64])
def test_attention_window_of_a_chunk(P, bits):
    """Query tiles over a window: the early pages given back, of one sequence to the last of them
    that no query sees, of one all; a hole inside."""
    print(f"case window page {P} bits {bits}", flush=True)
    lens = [1900, 1300, 700]
    holes = {(0, i) for i in range(1000 // P)} | {(1, i) for i in range(1300 // P - 1)} | {(2, i) for i in range(-(-700 // P))}
    holes |= {(0, 1200 // P), (0, 1300 // P + 1)}
    out = check_attention(attend_case(P, 3, 72, 8, 2, lens, P, bits, holes), 8)
    assert (out[2] == 0).all()


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("B,T,lens,P,given,holes", [
    (1, 520, [2300], 64, 1000, (19, 25)),            # a window, holes behind it
    (1, 513, [1501], 16, 0, (3, 40, 41, 60, 92)),    # holes that end inside a block
    (2, 300, [1300, 0], 32, 200, (38,)),             # an idle slot
    (2, 257, [140, 3000], 128, 0, (1,)),             # more rows than keys
])
def test_attention_many_tiles(B, T, lens, P, given, holes, bits):
    """Tiles that share a CU two by two, their keys in parts."""
    print(f"case tiles {B} {T} {lens} page {P} bits {bits}", flush=True)
    holes = {(0, i) for i in range(given // P)} | {(0, i) for i in holes}
    check_attention(attend_case(sum(lens) + P, B, T, 32, 4, lens, P, bits, holes), 32)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_scale_and_large_values(bits):
    """A maximum that moves by more than the rescale threshold between blocks, and a scale."""
    q, k, v, table, lens, qkv, ks, vs = attend_case(3, 2, 2, 8, 2, [900, 300], 32, bits)
    q = (q.float() * 6).bfloat16()
    check_attention((q, k, v, table, lens, qkv, ks, vs), 8, scale=0.11)


@pytest.mark.parametrize("T", [2, 72])
@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("spread", [4, 12, 40])
def test_attention_scales_far_apart(spread, P, T):
    """Pages whose values lie up to 2^(2 spread) apart, in both directions along a sequence."""
    print(f"case spread {spread} page {P} T {T}", flush=True)
    q, k, v, table, lens, qkv, ks, vs = attend_case(20 + spread, 3, T, 8, 2, [1030, 300, 75], P, 8)
    vs = vs * torch.exp2(torch.randint(-spread, spread + 1, vs.shape, generator=gen(spread)).float())
    check_attention((q, k, v, table, lens, qkv, ks, vs), 8)


@pytest.mark.parametrize("T", [15, 72])
def test_attention_far_scale_of_a_later_page(T):
    """The last page's values are 2^20 of the others': rows before it see none of that but the
    units of its scale."""
    q, k, v, table, lens, qkv, ks, vs = attend_case(31, 2, T, 8, 2, [1030, 75], 16, 8)
    for b, L in enumerate(lens.tolist()):
        vs[table[b, (L - 1) // 16]] *= 2.0 ** 20
    check_attention((q, k, v, table, lens, qkv, ks, vs), 8)


@pytest.mark.parametrize("T", [1, 80])
@pytest.mark.parametrize("bits", [16, 8])
def test_attention_light_weights_add_up(bits, T):
    """One key of value 0 outweighs each of the others by 2^16 or more: what they add up to counts."""
    print(f"case light T {T} bits {bits}", flush=True)
    q, k, v, table, lens, qkv, ks, vs = attend_case(30, 1, T, 8, 2, [2000], 64, bits)
    q = torch.zeros_like(q)
    q[..., 0] = 16.0                                  # the scores: k's first column
    k, v = torch.zeros_like(k.float()), torch.ones_like(v.float())
    first = int(table[0, 0])
    k[first, :, 3, 0] = 11.5                          # e^11.5 = 2^16.6
    v[first, :, 3] = 0.0
    k, v = (x.to(torch.bfloat16 if bits == 16 else torch.float8_e4m3fn) for x in (k, v))
    if bits == 8:
        ks, vs = torch.ones_like(ks), torch.ones_like(vs)
    check_attention((q, k, v, table, lens, qkv, ks, vs), 8)


def test_attention_gate_forms_and_strided_table():
    from lollm_amd import ops
    q, k, v, table, lens, qkv, ks, vs = cuda(*attend_case(4, 3, 2, 8, 2, [40, 1, 333], 16, 8))
    want = ops.attn_paged(q, k, v, table, lens, gates(qkv, 8), k_scale=ks, v_scale=vs)
    dense = gates(qkv, 8).contiguous()
    wide = torch.full((3, table.shape[1] + 5), 10 ** 6, dtype=torch.int32, device="cuda")
    wide[:, :table.shape[1]] = table
    got = ops.attn_paged(q, k, v, wide[:, :table.shape[1]], lens, dense, k_scale=ks, v_scale=vs)
    assert torch.equal(got, want)
    got = ops.attn_paged(q, k, v, wide, lens, dense.view(3, 2, -1), k_scale=ks, v_scale=vs)
    assert torch.equal(got, want)
    plain = ops.attn_paged(q, k, v, table, lens, k_scale=ks, v_scale=vs).float()
    torch.testing.assert_close(want.float(), plain * torch.sigmoid(dense.float().view(3, 2, -1)), rtol=2 ** -6, atol=1e-6)


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T", [2, 70])
def test_attention_shared_pages(T, bits):
    """Two sequences over the pages of a common prompt, and a page named twice in one table."""
    print(f"case shared T {T} bits {bits}", flush=True)
    q, k, v, table, lens, qkv, ks, vs = attend_case(32, 3, T, 8, 2, [500, 333, 200], 32, bits)
    table[1, :6] = table[0, :6]
    table[2, 2] = table[2, 0]
    check_attention((q, k, v, table, lens, qkv, ks, vs), 8)


@pytest.mark.parametrize("bits", [16, 8])
def test_attention_largest_batch(bits):
    print(f"case 512 sequences bits {bits}", flush=True)
    lens = [(37 * b) % 150 for b in range(512)]
    check_attention(attend_case(33, 512, 1, 4, 2, lens, 16, bits), 4)


@pytest.mark.parametrize("bits", [16, 8])
def test_pools_past_4_gb(bits):
    """Pages whose bytes begin past 2^32, where neither 32 bits of bytes nor 31 of values reach."""
    from lollm_amd import ops
    print(f"case large pool bits {bits}", flush=True)
    Hkv, P = 2, 128
    n = (2 ** 32 + 2 ** 28) // (Hkv * P * D * bits // 8)
    for T in (3, 80):
        q, k, v, table, lens, qkv, ks, vs = cuda(*attend_case(34, 2, T, 8, Hkv, [700, 333], P, bits))
        want = ops.attn_paged(q, k, v, table, lens, gates(qkv, 8), k_scale=ks, v_scale=vs)
        m = k.shape[0]
        far = torch.where(table >= 0, table + (n - m), table)

        def grown(x):
            y = torch.empty((n, *x.shape[1:]), dtype=x.dtype, device="cuda")
            y[n - m:].view(torch.uint8).copy_(x.view(torch.uint8))
            return y

        big = [None if x is None else grown(x) for x in (k, v, ks, vs)]
        assert torch.equal(ops.attn_paged(q, big[0], big[1], far, lens, gates(qkv, 8), k_scale=big[2], v_scale=big[3]), want)
        w, inv = torch.zeros(D, dtype=torch.bfloat16, device="cuda"), torch.ones(32, device="cuda")
        for pools, tb in (((k, v, ks, vs), table), (big, far)):
            ops.attn_append(qkv, w, w, inv, lens - T, tb, pools[0], pools[1], 8, 64, EPS, k_scale=pools[2], v_scale=pools[3])
        torch.cuda.synchronize()
        for x, y in zip((k, v, ks, vs), big):
            assert x is None or torch.equal(x.view(torch.uint8), y[n - m:].view(torch.uint8))
        del big


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("T", [3, 90, 520])
def test_attention_lengths_outside_the_table(T, bits):
    """A length past what the table names counts as that much, a negative one as none."""
    print(f"case lengths T {T} bits {bits}", flush=True)
    q, k, v, table, lens, qkv, ks, vs = attend_case(35, 3, T, 16, 4, [640, 600, 64], 64, bits)
    lens = torch.tensor([2 ** 31 - 1, 600, -7], dtype=torch.int32)
    out = check_attention((q, k, v, table, lens, qkv, ks, vs), 16)
    assert (out[2] == 0).all()


def test_outputs_of_the_caller():
    from lollm_amd import ops
    q, k, v, table, lens, qkv, ks, vs = cuda(*attend_case(36, 2, 3, 8, 2, [40, 90], 16, 8))
    want = ops.attn_paged(q, k, v, table, lens, gates(qkv, 8), k_scale=ks, v_scale=vs)
    out = torch.full((2, 3, 8 * D), 7.0, dtype=torch.bfloat16, device="cuda")
    assert ops.attn_paged(q, k, v, table, lens, gates(qkv, 8), k_scale=ks, v_scale=vs, out=out) is out
    assert torch.equal(out, want)
    w, inv = torch.zeros(D, dtype=torch.bfloat16, device="cuda"), torch.ones(32, device="cuda")
    args = (qkv, w, w, inv, lens - 3, table, k, v, 8, 64, EPS)
    want, _ = ops.attn_append(*args, k_scale=ks, v_scale=vs)
    got, _ = ops.attn_append(*args, k_scale=ks, v_scale=vs, q_out=torch.empty_like(q))
    assert torch.equal(got, want)
    for bad in (torch.empty_like(q)[:, :2], torch.empty_like(q).float(), torch.empty_like(q).cpu()):
        with pytest.raises((ValueError, TypeError)):
            ops.attn_append(*args, k_scale=ks, v_scale=vs, q_out=bad)
        with pytest.raises((ValueError, TypeError)):
            ops.attn_paged(q, k, v, table, lens, None, k_scale=ks, v_scale=vs, out=bad)


def test_attention_repeats_bit_for_bit():
    from lollm_amd import ops
    q, k, v, table, lens, qkv, ks, vs = cuda(*attend_case(5, 4, 4, 16, 2, [900, 40, 2000, 333], 64, 8))
    outs = [ops.attn_paged(q, k, v, table, lens, gates(qkv, 16), k_scale=ks, v_scale=vs) for _ in range(4)]
    assert all(torch.equal(o, outs[0]) for o in outs)


# ------------------------------------------------------------------------------------
# append
# ------------------------------------------------------------------------------------
APPENDS = [
    # B, T, Hq, Hkv, lengths, page, rotary, positions
    (1, 1, 8, 2, [0], 16, 64, None),
    (3, 1, 8, 2, [15, 16, 17], 16, 64, None),         # the last slot, the first, the second
    (2, 4, 32, 4, [126, 61], 64, 64, "start"),        # across a page's end
    (2, 37, 4, 2, [5, 0], 16, 64, "token"),           # several pages
    (2, 130, 8, 2, [100, 128], 128, 256, None),       # every value rotated
    (1, 40, 3, 3, [31], 32, 76, "far"),               # a rotation that is not a multiple of 8
    (2, 9, 4, 1, [3, 64], 32, 0, None),               # none
    (1, 1100, 4, 2, [7], 64, 64, "far"),              # a workgroup per token
    (2, 6, 4, 2, [-3, 10], 16, 64, None),             # rows before the first are dropped
]


def append_case(seed, B, T, Hq, Hkv, lengths, P, rd, pos, bits, short=0):
    g = gen(seed)
    width = max(1, max(-(-(max(L, 0) + T) // P) for L in lengths) - short)
    n = B * width + 2
    k, ks = pool(g, n, Hkv, P, bits)
    v, vs = pool(g, n, Hkv, P, bits)
    table = torch.randperm(n, generator=g)[:B * width].view(B, width).to(torch.int32)
    qkv = (torch.randn(B, T, Hq * 2 * D + 2 * Hkv * D, generator=g) * torch.exp2(torch.randn(B, T, 1, generator=g))).bfloat16()
    qw, kw = ((0.1 * torch.randn(D, generator=g)).bfloat16() for _ in range(2))
    inv = 1.0 / (1e7 ** (torch.arange(0, rd, 2, dtype=torch.float32) / max(rd, 1)))
    rope = None
    if pos == "start":
        rope = torch.randint(0, 5000, (B,), generator=g).to(torch.int32)
    elif pos in ("token", "far"):
        rope = torch.randint(0, 300000 if pos == "far" else 4000, (B, T), generator=g).to(torch.int32)
    return qkv, qw, kw, inv, torch.tensor(lengths, dtype=torch.int32), table, k, v, ks, vs, rope


def check_append(case, Hq, rd):
    """Runs the append on the device and compares; returns the device pools."""
    from lollm_amd import ops
    qkv, qw, kw, inv, lengths, table, k, v, ks, vs, rope = case
    ref_q, ref = O.append(qkv, qw, kw, inv, lengths, table, k, v, Hq, rd, EPS, ks, vs, rope)
    d = cuda(qkv, qw, kw, inv, lengths, table, k.clone(), v.clone(), ks, vs, rope)
    kd, vd, ksd, vsd = d[6], d[7], d[8], d[9]
    q, gate = ops.attn_append(d[0], d[1], d[2], d[3] if rd else None, d[4], d[5], kd, vd, Hq, rd, EPS,
                              k_scale=ksd, v_scale=vsd, rope_pos=d[10])
    torch.cuda.synchronize()
    assert torch.equal(gate.cpu(), gates(qkv, Hq)) and gate.data_ptr() == d[0].data_ptr() + 2 * D
    # fp32 arithmetic (the norm, sines of 2^-20, two products): 2^-17 of the row's largest value
    def slack(x):
        return 2.0 ** -17 * x.abs().amax(-1, keepdim=True)
    got = q.cpu().double()
    assert ((got - ref_q).abs() <= 2.0 ** -8 * ref_q.abs() + slack(ref_q)).all()
    for name, pages, scale, before, sbefore in (("k", kd, ksd, k, ks), ("v", vd, vsd, v, vs)):
        r = ref[name]
        raw = pages.cpu()
        stored, kept = r["stored"], r["kept"]
        code = torch.uint8 if scale is not None else torch.int16
        other = ~(stored | kept)
        assert torch.equal(raw.view(code)[other], before.view(code)[other]), f"{name}: rows beside the call's changed"
        exact = r["values"]
        if scale is None:
            assert torch.equal(raw.view(code)[kept], before.view(code)[kept])
            x = raw.double()
            tol = 2.0 ** -8 * exact.abs() + (slack(exact) if name == "k" else 0.0)
            fine = exact.isfinite()
            assert ((x - exact).abs() <= tol)[fine & stored[..., None]].all(), name
            assert (~x.isfinite())[~fine & stored[..., None]].all()
            continue
        sc = scale.cpu().double()
        assert torch.equal(sc, r["scale"]), f"{name}: scales"
        # kept rows: the codes rounded to the new scale, which a power of two makes exact
        want = (before.float() * (sbefore / scale.cpu())[..., None, None]).to(torch.float8_e4m3fn)
        assert torch.equal(raw.view(code)[kept], want.view(code)[kept]), f"{name}: kept rows"
        x = raw.float().double() * sc[..., None, None]
        # half a step of e4m3: 2^-4 of a normal code's value, 2^-10 of the scale below
        tol = torch.maximum(2.0 ** -4 * exact.abs(), 2.0 ** -10 * sc[..., None, None]) + (slack(exact) if name == "k" else 0.0)
        fine = exact.isfinite()
        assert ((x - exact).abs() <= tol)[fine & stored[..., None]].all(), name
        assert x.isnan()[~fine & stored[..., None]].all()
        if name == "v":   # bf16 values, exact scale: torch's own rounding, to the bit
            w = torch.where(stored[..., None] & fine, exact / sc[..., None, None], 0.0).float().to(torch.float8_e4m3fn)
            at = (stored[..., None] & fine).expand(raw.shape)
            assert torch.equal(raw.view(code)[at], w.view(code)[at]), "v: codes"
    return d


@pytest.mark.parametrize("bits", [16, 8])
@pytest.mark.parametrize("B,T,Hq,Hkv,lengths,P,rd,pos", APPENDS)
def test_append(B, T, Hq, Hkv, lengths, P, rd, pos, bits):
    print(f"case append {B} {T} {Hq}/{Hkv} {lengths} page {P} rotary {rd} {pos} bits {bits}", flush=True)
    check_append(append_case(sum(lengths) + T + P, B, T, Hq, Hkv, lengths, P, rd, pos, bits), Hq, rd)


@pytest.mark.parametrize("bits", [16, 8])
def test_append_drops_rows_without_a_page(bits):
    """A table too short for the call, and entries that name no page of the pool."""
    case = list(append_case(9, 3, 20, 4, 2, [14, 3, 30], 16, 64, None, bits, short=1))
    case[5][0, 1] = -1
    case[5][1, 0] = case[6].shape[0]
    case[5][2, 1] = -2 ** 31
    check_append(tuple(case), 4, 64)


def test_append_scales():
    """Rows of zeros, of one huge value, of values that are not finite; scales that grow, that
    stay, and that restart on a page's first row."""
    case = list(append_case(10, 5, 3, 2, 1, [4, 4, 0, 4, 4], 16, 0, None, 8))
    qkv = case[0]
    v = qkv[:, :, 2 * 2 * D + D:]
    v[0] = 0.0                                        # no larger than anything: the scale stays
    v[1] = v[1] * 2.0 ** 40                           # kept rows fall below its least code
    v[2] = v[2] * 2.0 ** -40                          # a first row: the stale scale is forgotten
    v[3, 1, 5] = float("inf")
    v[3, 2, 7] = float("nan")
    v[4] = 448.0 * 2.0 ** -3                          # exactly the largest code
    check_append(tuple(case), 2, 0)
    case = list(append_case(11, 1, 2, 2, 1, [0], 16, 0, None, 8))
    case[0][:] = 0.0                                  # a page of zeros: the least scale
    d = check_append(tuple(case), 2, 0)
    assert float(d[9][int(case[5][0, 0]), 0]) == 2.0 ** -64


def test_append_token_by_token_equals_one_call_in_bf16():
    from lollm_amd import ops
    qkv, qw, kw, inv, lengths, table, k, v, _, _, _ = cuda(*append_case(12, 2, 70, 8, 2, [5, 40], 32, 64, None, 16))
    k1, v1 = k.clone(), v.clone()
    q, _ = ops.attn_append(qkv, qw, kw, inv, lengths, table, k, v, 8, 64, EPS)
    for t in range(70):
        qt, _ = ops.attn_append(qkv[:, t:t + 1].contiguous(), qw, kw, inv, lengths + t, table, k1, v1, 8, 64, EPS)
        assert torch.equal(qt[:, 0], q[:, t])
    assert torch.equal(k, k1) and torch.equal(v, v1)


# ------------------------------------------------------------------------------------
# together, and what is refused
# ------------------------------------------------------------------------------------
@pytest.mark.parametrize("bits", [16, 8])
def test_decode_steps_eager_and_replayed(bits):
    """A prompt, then steps of 3 tokens of which 1 .. 3 are kept, each an append and an attention:
    against the oracle's attention over what the pools hold, and the same from a captured graph."""
    from lollm_amd import ops
    B, Hq, Hkv, P, rd = 3, 8, 2, 16, 64
    qkv, qw, kw, inv, _, table, k, v, ks, vs, _ = cuda(*append_case(13, B, 75, Hq, Hkv, [40] * B, P, rd, None, bits))
    g = gen(14)

    def state():
        return [None if x is None else x.clone() for x in (k, v, ks, vs)] + [torch.zeros(B, dtype=torch.int32, device="cuda")]

    def step(x, s, T):
        kk, vv, sk, sv, length = s
        q, gate = ops.attn_append(x, qw, kw, inv, length, table, kk, vv, Hq, rd, EPS, k_scale=sk, v_scale=sv)
        return q, ops.attn_paged(q, kk, vv, table, length + T, gate, k_scale=sk, v_scale=sv)

    s = state()
    q, out = step(qkv, s, 75)
    ref, tol = O.attention(q.cpu(), s[0].cpu(), s[1].cpu(), table.cpu(), torch.full((B,), 75), gates(qkv, Hq).cpu(),
                           None if bits == 16 else s[2].cpu(), None if bits == 16 else s[3].cpu())
    assert ((out.cpu().double() - ref).abs() <= tol).all()
    s[4] += 75
    s2 = [None if x is None else x.clone() for x in s]
    x = qkv[:, :3].contiguous().clone()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        keep = [None if y is None else y.clone() for y in s2]
        step(x, keep, 3)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gq, gout = step(x, s2, 3)
    for i in range(6):
        x.copy_(torch.randn(x.shape, generator=g).bfloat16())
        q, out = step(x, s, 3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, gout) and torch.equal(q, gq)
        assert all(a is None or torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(s[:4], s2[:4]))
        ref, tol = O.attention(q.cpu(), s[0].cpu(), s[1].cpu(), table.cpu(), (s[4] + 3).cpu(), gates(x, Hq).cpu(),
                               None if bits == 16 else s[2].cpu(), None if bits == 16 else s[3].cpu())
        assert ((out.cpu().double() - ref).abs() <= tol).all()
        kept = torch.randint(1, 4, (B,), generator=g).to(torch.int32).cuda()   # the others are rolled back
        s[4] += kept
        s2[4].copy_(s[4])


def test_other_stream_and_caller_workspace():
    from lollm_amd import ops
    q, k, v, table, lens, qkv, ks, vs = cuda(*attend_case(15, 4, 2, 8, 2, [400, 40, 20, 333], 64, 8))
    want = ops.attn_paged(q, k, v, table, lens, gates(qkv, 8), k_scale=ks, v_scale=vs)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    ws = torch.empty(ops.attn_paged_workspace_bytes(4, 2, 8, 2, D, k.dtype), dtype=torch.uint8, device="cuda")
    with torch.cuda.stream(st):
        got = ops.attn_paged(q, k, v, table, lens, gates(qkv, 8), k_scale=ks, v_scale=vs, workspace=ws)
    st.synchronize()
    assert torch.equal(got, want)


@pytest.mark.parametrize("T", [2, 72])
def test_two_streams_at_once(T):
    from lollm_amd import ops
    cases = [cuda(*attend_case(40 + i, 3, T, 8, 2, [900, 77, 300 + i], 32, 8)) for i in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]

    def call(c):
        q, k, v, table, lens, qkv, ks, vs = c
        return ops.attn_paged(q, k, v, table, lens, gates(qkv, 8), k_scale=ks, v_scale=vs)

    want = [call(c) for c in cases]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(5):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                outs[i].append(call(cases[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in range(2) for o in outs[i])


@pytest.mark.parametrize("T", [2, 72])
def test_two_graphs_share_a_workspace(T):
    """Replayed in turn on one stream, over lengths that move between the replays."""
    from lollm_amd import ops
    cases = [cuda(*attend_case(50 + i, 3, T, 8, 2, [900, 80, 300 + i], 32, 8)) for i in range(2)]
    ws = torch.empty(ops.attn_paged_workspace_bytes(3, T, 8, 2, D, cases[0][1].dtype), dtype=torch.uint8, device="cuda")

    def call(c, workspace):
        q, k, v, table, lens, qkv, ks, vs = c
        return ops.attn_paged(q, k, v, table, lens, gates(qkv, 8), k_scale=ks, v_scale=vs, workspace=workspace)

    graphs, outs = [], []
    for c in cases:
        call(c, None)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(call(c, ws))
        graphs.append(g)
    for i in range(5):
        for c in cases:
            c[4].sub_(i)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for c, out in zip(cases, outs):
            assert torch.equal(out, call(c, None))


def test_refusals():
    from lollm_amd import ops
    q, k, v, table, lens, qkv, ks, vs = cuda(*attend_case(16, 2, 2, 8, 2, [40, 20], 16, 8))
    gate = gates(qkv, 8)
    ok = dict(k_scale=ks, v_scale=vs)
    bad = [
        (ValueError, lambda: ops.attn_paged(q, k, v, table, lens, gate)),                      # no scales
        (ValueError, lambda: ops.attn_paged(q, k, v, table, lens, gate, k_scale=ks)),
        (ValueError, lambda: ops.attn_paged(q, k, v, table, lens, gate, k_scale=ks[:, :1].contiguous(), v_scale=vs)),
        (TypeError, lambda: ops.attn_paged(q, k.view(torch.float8_e5m2), v, table, lens, gate, **ok)),
        (ValueError, lambda: ops.attn_paged(q, k[:, :, :8].contiguous(), v[:, :, :8].contiguous(), table, lens, gate, **ok)),
        (ValueError, lambda: ops.attn_paged(q, k, v[:1].contiguous(), table, lens, gate, **ok)),
        (ValueError, lambda: ops.attn_paged(q, k, v, table[:1], lens, gate, **ok)),
        (ValueError, lambda: ops.attn_paged(q, k, v, table.long(), lens, gate, **ok)),
        (ValueError, lambda: ops.attn_paged(q, k, v, table.t().contiguous().t(), lens, gate, **ok)),
        (TypeError, lambda: ops.attn_paged(q, k, v, table, lens.long(), gate, **ok)),
        (TypeError, lambda: ops.attn_paged(q.float(), k, v, table, lens, gate, **ok)),
        (TypeError, lambda: ops.attn_paged(q, k, v, table, lens, gate.float(), **ok)),
        (ValueError, lambda: ops.attn_paged(q, k, v, table, lens, gate[:, :, :4], **ok)),
        (ValueError, lambda: ops.attn_paged(q, k, v, table, lens, gate.transpose(-1, -2).contiguous().transpose(-1, -2), **ok)),
        (ValueError, lambda: ops.attn_paged(q[:, :, :7].contiguous(), k, v, table, lens, None, **ok)),
        (RuntimeError, lambda: ops.attn_paged(q, k, v, table, lens, gate, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"), **ok)),
        (RuntimeError, lambda: ops.attn_paged(q, k, v, table, lens, gate, grid=1, workspace=torch.empty(64, dtype=torch.uint8, device="cuda"), **ok)),
        (ValueError, lambda: ops.attn_paged(q, k, v, table, lens, gate, grid=2000, **ok)),
        (ValueError, lambda: ops.attn_paged(q.cpu(), k, v, table, lens, gate, **ok)),
    ]
    w = torch.zeros(D, dtype=torch.bfloat16, device="cuda")
    inv = torch.ones(32, device="cuda")

    def app(x=qkv, w1=w, f=inv, ln=lens, tb=table, Hq=8, rd=64, **kw):
        return ops.attn_append(x, w1, w, f, ln, tb, k, v, Hq, rd, EPS, **{**ok, **kw})

    bad += [
        (ValueError, lambda: app(Hq=7)),
        (ValueError, lambda: app(x=qkv.view(-1))),
        (TypeError, lambda: app(x=qkv.float())),
        (ValueError, lambda: app(f=inv[:16])),
        (RuntimeError, lambda: app(rd=63, f=inv[:31].clone())),
        (TypeError, lambda: app(ln=lens.long())),
        (ValueError, lambda: app(rope_pos=lens[:1].clone())),
        (ValueError, lambda: app(k_scale=None)),
        (ValueError, lambda: app(tb=table[:, :0])),
    ]
    before = k.view(torch.uint8).clone()
    for i, (err, call) in enumerate(bad):
        with pytest.raises(err):
            call()
            pytest.fail(f"call {i} was taken")
    torch.cuda.synchronize()
    assert torch.equal(before, k.view(torch.uint8))
