"""The paged cache's C entry points refuse what they do not take before any launch (no GPU)."""

import ctypes

import pytest

from lollm_amd import _lib

P = ctypes.c_void_p(4096)   # never dereferenced: every call below is refused on the host
Z = None


def attn(**kw):
    a = dict(q=P, k=P, v=P, ks=Z, vs=Z, dt=0, table=P, ts=4, tw=4, n=8, page=16, kv_len=P, gate=Z, gr=0, gh=0,
             out=P, ws=Z, wsb=0, B=1, T=1, Hq=8, Hkv=2, D=256, grid=4, scale=1.0, st=Z)
    a.update(kw)
    return _lib.lib().lollm_attn_paged(*a.values())


def append(**kw):
    a = dict(qkv=P, qw=P, kw=P, inv=P, ln=P, pos=Z, per=0, table=P, ts=4, tw=4, n=8, page=16, dt=0, B=1, T=1, Hq=8,
             Hkv=2, D=256, rd=64, eps=1e-6, q=P, k=P, v=P, ks=Z, vs=Z, st=Z)
    a.update(kw)
    return _lib.lib().lollm_attn_append(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(q=Z), 1), (dict(k=Z), 1), (dict(v=Z), 1), (dict(table=Z), 1), (dict(kv_len=Z), 1), (dict(out=Z), 1),
    (dict(dt=1), 2), (dict(dt=2), 1), (dict(dt=2, ks=P), 1), (dict(ts=3), 1), (dict(tw=0), 1), (dict(n=0), 1),
    (dict(page=8), 2), (dict(page=48), 2), (dict(page=256), 2), (dict(ts=2 ** 28, tw=2 ** 28), 2),
    (dict(B=0), 1), (dict(T=0), 1), (dict(Hq=7), 1), (dict(D=128), 2), (dict(B=513), 2), (dict(Hq=66), 2),
    (dict(grid=-1), 1), (dict(grid=1025), 1), (dict(gate=P, gr=100, gh=256), 1), (dict(gate=P, gr=2048, gh=128), 1),
    (dict(gate=P, gr=2049, gh=256), 1), (dict(T=2 ** 20), 2), (dict(wsb=10 ** 9), 1), (dict(ws=P, wsb=100), 1),
])
def test_attn_paged_refuses(kw, rc):
    assert attn(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(qkv=Z), 1), (dict(qw=Z), 1), (dict(kw=Z), 1), (dict(inv=Z), 1), (dict(ln=Z), 1), (dict(table=Z), 1),
    (dict(q=Z), 1), (dict(k=Z), 1), (dict(v=Z), 1), (dict(per=1), 1), (dict(ts=3), 1), (dict(tw=0), 1),
    (dict(n=0), 1), (dict(page=8), 2), (dict(page=256), 2), (dict(dt=1), 2), (dict(dt=2), 1), (dict(dt=2, ks=P), 1),
    (dict(B=0), 1), (dict(T=0), 1), (dict(Hq=0), 1), (dict(Hkv=0), 1), (dict(D=128), 2), (dict(rd=63), 2),
    (dict(rd=258), 2), (dict(rd=-2), 2), (dict(ts=2 ** 28, tw=2 ** 28), 2), (dict(B=2 ** 16, T=2 ** 16), 2),
])
def test_attn_append_refuses(kw, rc):
    assert append(**kw) == rc


def test_workspace_bytes():
    f = _lib.lib().lollm_attn_paged_workspace_bytes
    # one fp32 piece of 32 x 256 values and 2 x 32 sums per workgroup and pair, 16 bytes a pair
    assert f(2, 1, 8, 2, 256, 0, 7) == (7 + 4) * (64 + 8192) * 4 + 4 * 16 == f(2, 1, 8, 2, 256, 2, 7)
    assert f(2, 1, 8, 3, 256, 0, 7) == -1
    assert f(2, 1, 8, 2, 128, 0, 7) == -1
    assert f(2, 1, 8, 2, 256, 1, 7) == -1
    assert f(2, 1, 8, 2, 256, 0, 1025) == -1
