"""The paged cache without a GPU: its C entry points refuse what they do not take before any
launch; Qwen3_5PagedCache hands pages out and takes them back on the host."""

import ctypes

import pytest
import torch

from lollm_amd import _lib
from lollm_amd.qwen3_5 import Qwen3_5Config, Qwen3_5PagedCache
from lollm_amd.qwen3_5.config import micro_config_dict

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
    (dict(scale=0.0), 1), (dict(scale=-1.0), 1), (dict(scale=float("nan")), 1), (dict(scale=float("inf")), 1),
])
def test_attn_paged_refuses(kw, rc):
    assert attn(**kw) == rc


@pytest.mark.parametrize("kw,rc", [
    (dict(qkv=Z), 1), (dict(qw=Z), 1), (dict(kw=Z), 1), (dict(inv=Z), 1), (dict(ln=Z), 1), (dict(table=Z), 1),
    (dict(q=Z), 1), (dict(k=Z), 1), (dict(v=Z), 1), (dict(per=1), 1), (dict(ts=3), 1), (dict(tw=0), 1),
    (dict(n=0), 1), (dict(page=8), 2), (dict(page=256), 2), (dict(dt=1), 2), (dict(dt=2), 1), (dict(dt=2, ks=P), 1),
    (dict(B=0), 1), (dict(T=0), 1), (dict(Hq=0), 1), (dict(Hkv=0), 1), (dict(D=128), 2), (dict(rd=63), 2),
    (dict(rd=258), 2), (dict(rd=-2), 2), (dict(ts=2 ** 28, tw=2 ** 28), 2), (dict(B=2 ** 16, T=2 ** 16), 2),
    (dict(Hkv=65536), 2), (dict(Hq=2 ** 22), 2),
])
def test_attn_append_refuses(kw, rc):
    assert append(**kw) == rc


def test_gate_strides():
    """The stride of a head is 32 bits in the C call: a wider one is refused, not cut."""
    from lollm_amd import ops

    def gate(head):
        return torch.empty(2 * head, dtype=torch.bfloat16, device="meta").as_strided((1, 1, 2, 256), (1, 1, head, 1))

    for head in (256, 512, 2 ** 31 - 8):
        assert ops._gate_arg(gate(head), 1, 1, 2, 256, -1) == (0, 2 * head, head)
    for head in (2 ** 31, 2 ** 32 + 256, 128, 260):
        with pytest.raises(ValueError):
            ops._gate_arg(gate(head), 1, 1, 2, 256, -1)


def test_workspace_bytes():
    f = _lib.lib().lollm_attn_paged_workspace_bytes
    # one fp32 piece of 32 x 256 values and 2 x 32 sums per workgroup and pair, 16 bytes a pair
    assert f(2, 1, 8, 2, 256, 0, 7) == (7 + 4) * (64 + 8192) * 4 + 4 * 16 == f(2, 1, 8, 2, 256, 2, 7)
    assert f(2, 1, 8, 3, 256, 0, 7) == -1
    assert f(2, 1, 8, 2, 128, 0, 7) == -1
    assert f(2, 1, 8, 2, 256, 1, 7) == -1
    assert f(2, 1, 8, 2, 256, 0, 1025) == -1


def cache(batch=3, max_len=100, **kw):
    return Qwen3_5PagedCache(Qwen3_5Config.from_hf(micro_config_dict()), batch, max_len, device="cpu", **kw)


def pages_of(c):
    return [[int(p) for p in row if p >= 0] for row in c.table]


def test_cache_hands_pages_out_as_sequences_grow():
    c = cache(page=16)
    assert c.table.shape == (3, 7) and c.n_pages == 21 and pages_of(c) == [[], [], []]
    c.advance(16)
    assert [len(p) for p in pages_of(c)] == [1, 1, 1]
    c.advance(1)
    assert [len(p) for p in pages_of(c)] == [2, 2, 2]
    c.reserve(15)                                    # what is held suffices
    assert [len(p) for p in pages_of(c)] == [2, 2, 2]
    c.advance(83)
    every = sum(pages_of(c), [])
    assert len(every) == len(set(every)) == 21 and not c.free and c.seen_tokens == 100
    with pytest.raises(RuntimeError, match="capacity"):
        c.reserve(1)


def test_cache_pool_smaller_than_every_sequence_at_max_len():
    c = cache(page=16, n_pages=7)
    c.advance(20)                                    # 2 pages each, 1 free
    with pytest.raises(RuntimeError, match="pool exhausted"):
        c.reserve(13)
    before = pages_of(c)
    c.release(1)
    assert pages_of(c) == [before[0], [], before[2]] and len(c.free) == 3 and int(c.lengths[1]) == 0
    c.reserve(13)                                    # the released one takes none
    assert [len(p) for p in pages_of(c)] == [3, 0, 3] and len(c.free) == 1


def test_cache_goes_by_the_lengths_where_the_bound_is_short_of_pages():
    c = cache(page=16, n_pages=7)
    c.advance(20)
    c.lengths.copy_(torch.tensor([20, 5, 9], dtype=torch.int32))   # rolled back since
    c.len_bound = 40                                 # the bound would take 9 pages
    c.reserve(10)
    assert [len(p) for p in pages_of(c)] == [2, 2, 2] and c.len_bound == 20


def test_cache_takes_idle_pages_back_before_the_pool_is_short():
    """A long bound gave both sequences four pages; the second fills two when the first needs a fifth."""
    c = cache(batch=2, page=16, n_pages=8)
    c.reserve(60)
    c.lengths.copy_(torch.tensor([60, 28], dtype=torch.int32))
    c.grew(60)
    assert c.held == [4, 4] and not c.free
    mine, other = pages_of(c)
    c.lengths.copy_(torch.tensor([64, 29], dtype=torch.int32))
    c.grew(4)
    c.reserve(4)
    now = pages_of(c)
    assert now[0][:4] == mine and len(now[0]) == 5 and now[1] == other[:3] and c.held == [5, 3]
    assert torch.equal(c.table, c._host_table) and (c.table[1, 3:] == -1).all()


@pytest.mark.parametrize("kept", [(4, 1), (1, 4), (4, 4), (2, 3)])
def test_cache_serves_until_the_real_need_passes_the_pool(kept):
    """Steps of 4 rows of which a sequence keeps its own number: the first step that is refused is
    the first whose rows do not fit, and rows that are there keep their pages until then."""
    c = cache(batch=2, max_len=2000, page=16, n_pages=40)
    c.advance(32)
    for step in range(1000):
        need = [-(-(int(n) + 4) // 16) for n in c.lengths]
        full = [-(-int(n) // 16) for n in c.lengths]
        before = pages_of(c)
        if sum(need) > 40:
            with pytest.raises(RuntimeError, match="pool exhausted"):
                c.reserve(4)
            assert pages_of(c) == before
            break
        c.reserve(4)
        now = pages_of(c)
        assert all(n[:f] == b[:f] for n, b, f in zip(now, before, full))
        assert all(len(n) >= m for n, m in zip(now, need)) and [len(n) for n in now] == c.held
        every = sum(now, [])
        assert sorted(every + c.free) == list(range(40)) and c.len_bound >= int(c.lengths.max())
        c.lengths += torch.tensor(kept, dtype=torch.int32)
        c.grew(4)
    else:
        raise AssertionError("never refused")


def test_cache_reads_the_lengths_only_where_the_pool_is_short():
    """Bounds are each sequence's own once read: a page at a time, not all of the batch's longest."""
    c = cache(batch=2, max_len=2000, page=16, n_pages=41)
    c.advance(32)
    reads = []
    measure = c._measure
    c._measure = lambda: (reads.append(1), measure())
    for _ in range(84):
        c.reserve(4)
        c.lengths += torch.tensor([4, 1], dtype=torch.int32)
        c.grew(4)
    assert c.held[1] < c.held[0] and 1 <= len(reads) <= 4


def test_cache_append_read_and_clone():
    g = torch.Generator().manual_seed(1)
    c = cache(page=16)
    k, v = (torch.randn(3, 2, 37, 256, generator=g).bfloat16() for _ in range(2))
    layer = 3
    assert c.read_kv(0) is None
    for a, b in ((0, 5), (5, 20), (20, 37)):
        kk, vv = c.append_kv(layer, k[:, :, a:b], v[:, :, a:b])
        assert torch.equal(kk, k[:, :, :b]) and torch.equal(vv, v[:, :, :b])
        c.advance(b - a)
    d = c.clone()
    assert type(d) is Qwen3_5PagedCache and d.nbytes() == c.nbytes()
    d.append_kv(layer, k[:, :, :20], v[:, :, :20])
    d.advance(20)
    assert len(c.free) == 12 and len(d.free) == 9 and c.seen_tokens == 37
    assert torch.equal(c.read_kv(layer)[0], k) and torch.equal(d.read_kv(layer)[1][:, :, 37:], v[:, :, :20])


def test_cache_refusals():
    with pytest.raises(ValueError):
        cache(page=48)
    with pytest.raises(TypeError):
        cache(kv_dtype=torch.float16)
    with pytest.raises(ValueError):
        cache(n_pages=0)
    c = cache(page=32, kv_dtype=torch.float8_e4m3fn)
    x = torch.zeros(3, 2, 1, 256, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="attn_append"):
        c.append_kv(3, x, x)
    assert set(c.layers[3]) == {"k", "v", "ks", "vs"} and set(c.layers[0]) == {"win", "rec", "rep"}


def test_cache_refuses_rows_of_a_released_sequence():
    c = cache(batch=1, page=16)
    x = torch.zeros(1, 2, 5, 256, dtype=torch.bfloat16)
    c.append_kv(3, x, x)
    c.release(0)
    c.release(0)                                     # again: nothing to give back
    assert len(c.free) == 7
    for call in (lambda: c.append_kv(3, x, x), lambda: c.read_kv(3)):
        with pytest.raises(RuntimeError, match="released"):
            call()


def test_released_sequence_takes_no_capacity():
    """Steps go on adding to a released sequence's length, here more than to the live one's: it is
    cleared before each, and the live one reaches max_len."""
    c = cache(batch=2, max_len=64, page=16)
    c.advance(32)
    c.release(1)
    for n in range(32, 61):
        c.reserve(4)
        assert c.lengths.tolist() == [n, 0] and c.held[1] == 0
        c.lengths += torch.tensor([1, 4], dtype=torch.int32)
        c.grew(4)
    with pytest.raises(RuntimeError, match="capacity"):
        c.reserve(4)
    assert c.len_bound == 61
    d = c.clone()
    d.release(0)
    d.reserve(4)                                     # no one left: nothing to refuse
    assert d.lengths.tolist() == [0, 0] and d.len_bound == 0 and c.live == [True, False]


def test_released_sequence_takes_no_output_capacity():
    from lollm_amd.qwen3_5 import SpecDecoder
    d = SpecDecoder.__new__(SpecDecoder)
    d.k, d.cache, d.out_capacity, d.out_bound = 3, cache(batch=2, max_len=64, page=16), 16, 0
    d.out_count = torch.tensor([9, 30], dtype=torch.int32)
    d.cache.release(1)
    d.out_bound = 14
    d._reserve()                                     # 9 + 4 <= 16
    assert d.out_bound == 9
    d.out_count[0], d.out_bound = 13, 16
    with pytest.raises(RuntimeError, match="output capacity"):
        d._reserve()


def test_new_cache_takes_what_it_is_given():
    from lollm_amd.qwen3_5 import Qwen3_5Cache, Qwen3_5Model

    class Model:
        cfg, device = Qwen3_5Config.from_hf(micro_config_dict()), torch.device("cpu")
        new_cache = Qwen3_5Model.new_cache

    assert type(Model().new_cache(1, 50)) is Qwen3_5Cache
    c = Model().new_cache(1, 50, kv_dtype=torch.float8_e4m3fn)
    assert (c.page, c.kv_dtype, c.n_pages) == (64, torch.float8_e4m3fn, 1)
    assert Model().new_cache(1, 50, n_pages=3).kv_dtype == torch.bfloat16
    with pytest.raises(ValueError):
        Model().new_cache(1, 50, page=0)
