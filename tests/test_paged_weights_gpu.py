"""Attention over 8-bit pages where one key outweighs the others by far, as a prompt's first token
does in a model: the light keys' share of a result is as exact as their share of the row's sum.

The tolerance, on the weighted mean of |V|, which is the result itself where every light key's value
is 1 and the heavy one's 0: half a step of the output's bf16 (2^-8), half a step of fp16 weights
(2^-11), and half of fp16's least step, 2^-25, where the row's largest weight counts 2^10: 2^-35 of the
heavy weight on each light one, which is e^-nats of it.  The score is one product of exact values and
the two sums are of fp32 (keys / 32 + 8 roundings of 2^-24 at most).
"""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D = 256


def heavy_case(keys, T, nats, at, P=64, Hq=8, Hkv=2):
    """One sequence of `keys` keys whose key `at` scores `nats` above all others, with the value 0
    beside their 1.  A score is q_0 k_0 / 16."""
    n = -(-keys // P)
    q = torch.zeros(1, T, Hq, D)
    q[..., 0] = float(nats)
    k, v = torch.zeros(n, Hkv, P, D), torch.ones(n, Hkv, P, D)
    k[at // P, :, at % P, 0] = 16.0
    v[at // P, :, at % P] = 0.0
    f8 = torch.float8_e4m3fn
    one = torch.ones(n, Hkv)
    table = torch.arange(n, dtype=torch.int32)[None]
    return [x.cuda() for x in (q.bfloat16(), k.to(f8), v.to(f8), table.contiguous(),
                               torch.tensor([keys], dtype=torch.int32), one, one.clone())]


def check(keys, T, nats, at, grid):
    from lollm_amd import ops
    q, k, v, table, lens, ks, vs = heavy_case(keys, T, nats, at)
    got = ops.attn_paged(q, k, v, table, lens, k_scale=ks, v_scale=vs, grid=grid).double().cpu()[0]
    light = math.exp(-nats)
    seen = torch.arange(keys - T, keys).double()[:, None]      # light keys of each query
    want = (seen * light / (1 + seen * light)).expand_as(got)
    tol = (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -35 / light + (keys / 32 + 8) * 2.0 ** -24) * want
    worst = ((got - want).abs() / tol).max()
    assert worst <= 1, f"{float(worst)} of the tolerance, {float(tol.max() / want.max())} of the result"


@pytest.mark.parametrize("nats", [8, 12, 17, 18, 20])
@pytest.mark.parametrize("keys,T,at,grid", [
    (2000, 1, 3, 1),          # one workgroup: the heavy key's wave walks a quarter of the keys
    (100000, 1, 0, 8),
    (700, 1, 350, 0),
    (700, 80, 3, 0),          # query tiles, one part
    (2000, 80, 0, 0),         # the keys of a tile in parts
    (2000, 80, 1900, 0),      # the heavy key comes last
    (9000, 300, 3, 0),
])
def test_light_keys_beside_a_heavy_one(keys, T, at, grid, nats):
    print(f"case heavy key {at} of {keys} by {nats} nats, T {T} grid {grid}", flush=True)
    check(keys, T, nats, at, grid)


@pytest.mark.parametrize("P", [16, 64])
@pytest.mark.parametrize("nats", [6, 13, 18])
@pytest.mark.parametrize("keys,T,grid", [(3001, 2, 1), (3001, 2, 0), (733, 70, 0), (5003, 260, 0)])
def test_random_keys_beside_a_heavy_one(keys, T, grid, nats, P):
    """Normal scores and values in pages of different scales, and a first key of value 0 above them.
    The tolerance is the kernel's published bound, term by term."""
    from lollm_amd import ops
    print(f"case first of {keys} keys by {nats} nats, T {T} grid {grid} page {P}", flush=True)
    g = torch.Generator().manual_seed(keys + T + nats)
    Hq, Hkv, n, f8 = 8, 2, -(-keys // P), torch.float8_e4m3fn
    q = torch.randn(1, T, Hq, D, generator=g)
    q[..., 0] = float(nats)
    k, v = (torch.randn(n, Hkv, P, D, generator=g) for _ in range(2))
    k[..., 0] = 0.0
    k[0, :, 0] = 0.0
    k[0, :, 0, 0] = 16.0
    v[0, :, 0] = 0.0
    q, k, v = q.bfloat16(), (k / 0.25).to(f8), (v * 16).to(f8)
    ks = torch.full((n, Hkv), 0.25)
    vs = torch.exp2(torch.randint(-6, -1, (n, Hkv), generator=g).float())
    table = torch.arange(n, dtype=torch.int32)[None].contiguous()
    lens = torch.tensor([keys], dtype=torch.int32)
    got = ops.attn_paged(q.cuda(), k.cuda(), v.cuda(), table.cuda(), lens.cuda(), k_scale=ks.cuda(), v_scale=vs.cuda(),
                         grid=grid).double().cpu().view(T, Hq, D)
    hidden = torch.arange(keys)[None] > torch.arange(keys - T, keys)[:, None]
    worst = 0.0
    for h in range(Hq):
        kv = h // (Hq // Hkv)
        kd = (k[:, kv].float().double() * 0.25).reshape(-1, D)[:keys]
        vd = (v[:, kv].float().double() * vs[:, kv, None, None].double()).reshape(-1, D)[:keys]
        qd = q[0, :, h].double()
        p = torch.softmax((qd @ kd.T / 16).masked_fill(hidden, -math.inf), -1)
        ds = 258 * 2.0 ** -24 * (qd.abs() @ kd.abs().T / 16).amax(-1, keepdim=True)
        want = p @ vd
        tol = ((2.0 ** -11 + 2 * ds + keys / 16 * 2.0 ** -24) * (p @ vd.abs())
               + 2.0 ** -35 * p.amax(-1, keepdim=True) * ((~hidden).double() @ vd.abs())
               + 2.0 ** -25 * float(vs[:, kv].max()) + (2.0 ** -8 + 2.0 ** -20) * want.abs())
        worst = max(worst, float(((got[:, h] - want).abs() / tol).max()))
    assert worst <= 1, worst
