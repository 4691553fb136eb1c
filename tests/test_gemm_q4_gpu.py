"""Products with 4-bit weights (lollm_gemm_q4) against 64 bits, its packing and quantising, and its
refusals."""

import pytest
import torch


def weight(N, K, group, zeros, seed):
    """(codes as numbers (N, K), scales, zeros or None) on the CPU."""
    g = torch.Generator().manual_seed(seed)
    code = torch.randint(0, 16, (N, K), generator=g, dtype=torch.uint8)
    scale = (torch.rand(N, K // group, generator=g) * 0.05 + 0.001).bfloat16()
    zero = torch.randint(0, 16, (N, K // group), generator=g, dtype=torch.uint8) if zeros else None
    return code, scale, zero


def bytes_of(code):
    return (code[:, 0::2] | (code[:, 1::2] << 4)).contiguous()


def values(code, scale, zero, group):
    """The weight in 64 bits."""
    N, K = code.shape
    z = 8.0 if zero is None else zero.double()[..., None]
    return ((code.double().view(N, K // group, group) - z) * scale.double()[..., None]).view(N, K)


def expected(x, w, swiglu):
    y = x.double() @ w.t()
    mag = x.double().abs() @ w.abs().t()
    if not swiglu:
        return y, mag
    gate, up = y.chunk(2, -1)
    mg, mu = mag.chunk(2, -1)
    # |d silu| <= 1.1 |d gate|
    return gate * torch.sigmoid(gate) * up, 1.1 * mg * up.abs() + gate.abs() * mu


def close(got, x, w, scale, swiglu, group):
    """A bf16 rounding (2^-8 of the value covers its half step twice), and the fp32 sums: a group's
    terms are at most (16 + 16) |x| s, K / 32 additions and what a matrix instruction adds inside, each
    2^-24 of the partial sums; 2^-18 of sum 32 |x| s covers 64 of them."""
    ref, _ = expected(x, w, swiglu)
    N, K = w.shape
    room = (x.double().abs().view(-1, K // group, group).sum(-1) @ scale.double().t()) * 32 * 2 ** -18
    if swiglu:
        y = x.double() @ w.t()
        gate, up = y.chunk(2, -1)
        rg, ru = room.chunk(2, -1)
        room = 1.1 * rg * up.abs() + gate.abs() * ru
    err = (got.double().cpu().view(ref.shape) - ref).abs()
    bad = err > ref.abs() * 2 ** -8 + room
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}, largest {err.max().item()}"


ROWS = (1, 2, 15, 16, 17, 31, 33, 48, 64, 65, 130)


@pytest.mark.gpu
@pytest.mark.parametrize("swiglu", (False, True))
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("N,K", [(64, 128), (128, 256), (192, 1152), (320, 2176)])
def test_gemm_q4_matches_64_bits(N, K, group, zeros, swiglu):
    from lollm_amd import ops
    code, scale, zero = weight(N, K, group, zeros, N + K + group)
    w = values(code, scale, zero, group)
    packed = ops.q4_pack(bytes_of(code).cuda(), scale.cuda(), None if zero is None else zero.cuda(),
                         ops.GEMM_SWIGLU if swiglu else ops.GEMM_NONE)
    g = torch.Generator().manual_seed(7)
    for M in ROWS:
        print(f"case q4 {M} x {N} x {K} group {group} zeros {zeros} swiglu {swiglu}", flush=True)
        x = torch.randn(M, K, generator=g).bfloat16()
        oc = N // 2 if swiglu else N
        buf = torch.full((M + 2, oc), 7.0, dtype=torch.bfloat16, device="cuda")
        got = ops.gemm_q4(x.cuda(), packed, out=buf[:M])
        close(got, x, w, scale, swiglu, group)
        assert (buf[M:] == 7.0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("M,N,K,group,swiglu", [(1, 24576, 4096, 128, True), (61, 12352, 4096, 128, False),
                                                (16, 4096, 12288, 64, False), (200, 6208, 1024, 32, False),
                                                (700, 4096, 8192, 128, False)])
def test_gemm_q4_at_the_models_sizes(M, N, K, group, swiglu):
    """Against fp64 on the device; activations with channels that stand out."""
    from lollm_amd import ops
    print(f"case q4 {M} x {N} x {K} group {group} swiglu {swiglu}", flush=True)
    code, scale, _ = weight(N, K, group, False, 5)
    w = values(code, scale, None, group).cuda()
    packed = ops.q4_pack(bytes_of(code).cuda(), scale.cuda(), None, ops.GEMM_SWIGLU if swiglu else ops.GEMM_NONE)
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(M, K, generator=g) * torch.where(torch.rand(K, generator=g) < 0.01, 16.0, 1.0)).bfloat16()
    got = ops.gemm_q4(x.cuda(), packed)
    ref, _ = expected(x.cuda(), w, swiglu)
    room = (x.double().abs().view(M, K // group, group).sum(-1) @ scale.double().t()) * 32 * 2 ** -18
    if swiglu:
        gate, up = (x.double().cuda() @ w.t()).cpu().chunk(2, -1)
        rg, ru = room.chunk(2, -1)
        room = 1.1 * rg * up.abs() + gate.abs() * ru
    err = (got.double() - ref).abs().cpu()
    assert (err <= ref.abs().cpu() * 2 ** -8 + room).all()


@pytest.mark.gpu
@pytest.mark.parametrize("swiglu", (False, True))
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128))
def test_gemm_q4_with_many_rows(group, zeros, swiglu):
    """The form for many rows, chosen by sizes: tiles that end inside (one row, 64 columns), one to nine
    stages of K, a workspace that the call asks for; the whole sum's room as for few rows, the product over
    the groups' three-part sums within it."""
    from lollm_amd import ops
    N = 6208
    for M, K in ((513, 1152), (640, 128), (900, 256), (1000, 640)):
        print(f"case q4 many rows {M} x {N} x {K} group {group} zeros {zeros} swiglu {swiglu}", flush=True)
        assert ops._q4_workspace_bytes(M, N, K, group, torch.cuda.current_device()) > 0
        code, scale, zero = weight(N, K, group, zeros, M + K)
        w = values(code, scale, zero, group).cuda()
        packed = ops.q4_pack(bytes_of(code).cuda(), scale.cuda(), None if zero is None else zero.cuda(),
                             ops.GEMM_SWIGLU if swiglu else ops.GEMM_NONE)
        g = torch.Generator().manual_seed(K)
        x = (torch.randn(M, 2 * K, generator=g) * torch.where(torch.rand(2 * K, generator=g) < 0.01, 16.0, 1.0)).bfloat16()
        x = x.cuda()[:, K:]
        buf = torch.full((M + 1, N // 2 if swiglu else N), 7.0, dtype=torch.bfloat16, device="cuda")
        got = ops.gemm_q4(x, packed, out=buf[:M])
        ref, _ = expected(x, w, swiglu)
        room = (x.double().abs().reshape(M, K // group, group).sum(-1) @ scale.cuda().double().t()) * 32 * 2 ** -18
        if swiglu:
            gate, up = (x.double() @ w.t()).chunk(2, -1)
            rg, ru = room.chunk(2, -1)
            room = 1.1 * rg * up.abs() + gate.abs() * ru
        assert ((got.double() - ref).abs() <= ref.abs() * 2 ** -8 + room).all()
        assert (buf[M:] == 7.0).all() and torch.equal(ops.gemm_q4(x, packed), got)


@pytest.mark.gpu
def test_gemm_q4_many_rows_captured_and_refused_without_a_workspace():
    from lollm_amd import _lib, ops
    M, N, K, group = 513, 6208, 256, 128
    code, scale, _ = weight(N, K, group, False, 6)
    packed = ops.q4_pack(bytes_of(code).cuda(), scale.cuda())
    xs = [torch.randn(M, K, generator=torch.Generator().manual_seed(i)).bfloat16().cuda() for i in range(2)]
    want = [ops.gemm_q4(x, packed).clone() for x in xs]
    need = _lib.lib().lollm_gemm_q4_workspace_bytes(M, N, K, group)
    assert need == 6 * M * 32
    out = torch.zeros(M, N, dtype=torch.bfloat16, device="cuda")
    ws = torch.empty(need, dtype=torch.uint8, device="cuda")
    for at, size in ((None, need), (ws.data_ptr(), need - 1), (ws.data_ptr() + 8, need)):
        assert _lib.lib().lollm_gemm_q4(xs[0].data_ptr(), K, packed.packed.data_ptr(), 0, out.data_ptr(), N, at, size, M, N, K,
                                        group, 0, None) == 1
    torch.cuda.synchronize()
    assert not out.any()
    buf = xs[0].clone()
    graphs = []
    for _ in range(2):      # two graphs, each with its own workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.gemm_q4(buf, packed)
        graphs.append((graph, y))
    for turn in range(4):
        buf.copy_(xs[turn % 2])
        for graph, y in graphs:
            graph.replay()
            assert torch.equal(y, want[turn % 2])
        ops.gemm_q4(xs[1 - turn % 2], packed)


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", (False, True))
def test_gemm_q4_rows_do_not_depend_on_each_other(zeros):
    """A row's bits are the same in calls of any number of rows, and over calls."""
    from lollm_amd import ops
    N, K, group = 256, 2176, 64
    code, scale, zero = weight(N, K, group, zeros, 11)
    packed = ops.q4_pack(bytes_of(code).cuda(), scale.cuda(), None if zero is None else zero.cuda())
    x = torch.randn(300, K, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    whole = ops.gemm_q4(x, packed)
    for lo, hi in ((0, 1), (5, 9), (30, 47), (100, 164), (64, 300)):
        print(f"case q4 rows {lo}:{hi}", flush=True)
        assert torch.equal(ops.gemm_q4(x[lo:hi], packed), whole[lo:hi])


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("N,K", [(4224, 1152), (12352, 640), (24640, 1152), (33088, 2432), (4096, 5504)])
def test_gemm_q4_a_rows_bits_at_any_number_of_columns(N, K, group, zeros):
    """The same over the forms that the number of columns chooses: one or several column tiles a
    workgroup, whole and partial sets of the stages that a wave holds."""
    from lollm_amd import ops
    code, scale, zero = weight(N, K, group, zeros, N + group)
    packed = ops.q4_pack(bytes_of(code).cuda(), scale.cuda(), None if zero is None else zero.cuda())
    x = torch.randn(64, K, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    whole = ops.gemm_q4(x, packed)
    for lo, hi in ((0, 1), (5, 9), (16, 32), (30, 47), (17, 49), (0, 33)):
        print(f"case q4 {N} x {K} group {group} zeros {zeros} rows {lo}:{hi}", flush=True)
        assert torch.equal(ops.gemm_q4(x[lo:hi], packed), whole[lo:hi])


@pytest.mark.gpu
def test_gemm_q4_leading_shapes_strides_and_no_rows():
    from lollm_amd import ops
    N, K = 128, 256
    code, scale, _ = weight(N, K, 128, False, 2)
    packed = ops.q4_pack(bytes_of(code).cuda(), scale.cuda())
    x = torch.randn(3, 5, 2 * K, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    part = x[..., K:]
    y = ops.gemm_q4(part, packed)
    assert y.shape == (3, 5, N) and torch.equal(y, ops.gemm_q4(part.contiguous().view(15, K), packed).view(3, 5, N))
    assert ops.gemm_q4(x[:0, :, :K], packed).shape == (0, 5, N)


@pytest.mark.gpu
def test_gemm_q4_on_another_stream_and_in_a_graph():
    from lollm_amd import ops
    N, K = 192, 1152
    code, scale, zero = weight(N, K, 32, True, 4)
    packed = ops.q4_pack(bytes_of(code).cuda(), scale.cuda(), zero.cuda())
    torch.cuda.synchronize()
    x = torch.randn(40, K, generator=torch.Generator().manual_seed(8)).bfloat16().cuda()
    other = torch.randn(40, K, generator=torch.Generator().manual_seed(9)).bfloat16().cuda()
    want, want2 = ops.gemm_q4(x, packed).clone(), ops.gemm_q4(other, packed).clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.gemm_q4(x, packed)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    buf = x.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.gemm_q4(buf, packed)
    for turn in range(4):
        buf.copy_(other if turn % 2 else x)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want2 if turn % 2 else want)
        ops.gemm_q4(other, packed)


@pytest.mark.gpu
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("zeros", (False, True))
def test_q4_quantize_rounds_to_nearest(group, zeros):
    """Every value is within half a step of its code's (with one step's worth of the scale's own
    rounding to bf16 over up to 15 steps), and codes, scales and zeros are those of the rule."""
    from lollm_amd import ops
    N, K = 64, 384
    g = torch.Generator().manual_seed(group)
    w = (torch.randn(N, K, generator=g) * torch.exp(torch.randn(N, 1, generator=g))).bfloat16()
    w[0] = 0
    w[1, :group] = 0.5          # one sign only
    w[2, :group] = -0.25
    print(f"case quantise group {group} zeros {zeros}", flush=True)
    codes, scales, zero = ops.q4_quantize(w.cuda(), group, zeros)
    v = w.double().view(N, K // group, group)
    lo, hi = v.amin(-1).clamp(max=0), v.amax(-1).clamp(min=0)
    step = (hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7.5
    s = scales.double().cpu()
    assert ((s - step).abs() <= step * 2 ** -8).all()
    assert (zero is None) == (not zeros)
    code = torch.stack([codes & 15, codes >> 4], -1).view(N, K).cpu()
    back = values(code, scales.cpu(), None if zero is None else zero.cpu(), group).view(v.shape)
    # half a step, the range's ends moved by the scale's rounding: 15 steps x 2^-9; and a zero that is
    # itself rounded: half a step more
    room = s[..., None] * ((1.0 if zeros else 0.5) + 15 * 2 ** -8)
    if not zeros:
        room = room + torch.where(v >= 7.49 * s[..., None], 0.5 * s[..., None], 0.0)   # 7.5 goes to 7
    assert ((back - v).abs() <= room).all()


@pytest.mark.gpu
def test_q4_refusals():
    from lollm_amd import ops
    dev = "cuda"

    def pack(N=64, K=256, group=64, **kw):
        codes = torch.zeros(N, K // 2, dtype=torch.uint8, device=dev)
        scales = torch.ones(N, max(K // group, 1), dtype=torch.bfloat16, device=dev)
        return ops.q4_pack(kw.pop("codes", codes), kw.pop("scales", scales), **kw)

    for bad in (dict(N=60), dict(K=192), dict(group=16), dict(group=256), dict(scales=torch.ones(64, 4, device=dev)),
                dict(codes=torch.zeros(64, 128, dtype=torch.int32, device=dev)),
                dict(scales=torch.ones(32, 4, dtype=torch.bfloat16, device=dev)),
                dict(zeros=torch.zeros(64, 3, dtype=torch.uint8, device=dev)),
                dict(zeros=torch.zeros(64, 4, device=dev)), dict(epilogue=2),
                dict(codes=torch.zeros(64, 128, dtype=torch.uint8))):
        with pytest.raises((ValueError, TypeError)):
            pack(**bad)
    w = pack()
    x = torch.zeros(3, 256, dtype=torch.bfloat16, device=dev)
    for bad in (x[:, :128], x.float(), x.cpu()):
        with pytest.raises((ValueError, TypeError)):
            ops.gemm_q4(bad, w)
    for out in (torch.empty(3, 32, dtype=torch.bfloat16, device=dev), torch.empty(3, 64, device=dev),
                torch.empty(64, 3, dtype=torch.bfloat16, device=dev).t()):
        with pytest.raises((ValueError, TypeError)):
            ops.gemm_q4(x, w, out=out)
    with pytest.raises(ValueError):
        ops.q4_quantize(torch.zeros(64, 100, dtype=torch.bfloat16, device=dev))
    with pytest.raises((ValueError, TypeError)):
        ops.q4_quantize(torch.zeros(64, 128, device=dev))


def test_q4_entry_points_check_before_any_launch():
    from lollm_amd import _lib
    L = _lib.lib()
    assert L.lollm_q4_packed_bytes(64, 256, 128, 0) == 64 * 128 + 2 * 128
    assert L.lollm_q4_packed_bytes(64, 256, 32, 1) == 64 * 128 + 3 * 64 * 8
    for shape in ((60, 256, 128), (64, 200, 128), (64, 256, 16), (0, 256, 32), (64, -128, 32)):
        assert L.lollm_q4_packed_bytes(*shape, 0) == -1
    p = 4096     # an address that no check reads
    assert L.lollm_gemm_q4(None, 256, p, 0, p, 64, None, 0, 1, 64, 256, 128, 0, None) == 1
    assert L.lollm_gemm_q4(p, 256, p, 0, p, 64, None, 0, 0, 64, 256, 128, 0, None) == 1
    assert L.lollm_gemm_q4(p, 256, p, 0, p, 64, None, 0, 1, 64, 256, 96, 0, None) == 2
    assert L.lollm_gemm_q4(p, 248, p, 0, p, 64, None, 0, 1, 64, 256, 128, 0, None) == 1
    assert L.lollm_gemm_q4(p, 256, p, 0, p, 60, None, 0, 1, 64, 256, 128, 0, None) == 1
    assert L.lollm_gemm_q4(p, 256, p, 0, p, 64, None, 0, 1, 64, 256, 128, 2, None) == 1
    assert L.lollm_gemm_q4(p + 8, 256, p, 0, p, 64, None, 0, 1, 64, 256, 128, 0, None) == 1
    assert L.lollm_q4_pack(p, None, None, p, 64, 256, 128, 0, None) == 1
    assert L.lollm_q4_pack(p, p, None, p + 4, 64, 256, 128, 0, None) == 1
    assert L.lollm_q4_quantize(None, p, p, None, 64, 256, 128, None) == 1
