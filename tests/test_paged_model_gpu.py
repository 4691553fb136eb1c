"""The hybrid decoder over paged caches: logits against the oracle at the model's own bf16 bar with
bf16 pages, what 8-bit pages hold against the bf16 pages of the same forward, and the speculative
decoder eager and replayed, out of pages, and with a released sequence."""

import pytest
import torch

from lollm_amd.qwen3_5.config import Qwen3_5Config, micro_config_dict
from oracle import qwen3_5_ref as R
from test_model_gpu import build, close_logits

pytestmark = pytest.mark.gpu
ATTN = 3   # micro_config_dict's attention layer


@pytest.fixture(scope="module")
def micro():
    return build(micro_config_dict())


@pytest.mark.parametrize("page", [16, 64])
def test_bf16_pages_against_the_oracle(micro, page):
    model, _, (W, W16), cfg = micro
    print(f"case model pages {page}", flush=True)
    ids = torch.randint(0, cfg.vocab_size, (2, 48), generator=torch.Generator().manual_seed(2))
    cache, slab, past, p16 = model.new_cache(2, 64, page=page), model.new_cache(2, 64), None, None
    for a, b in ((0, 41), (41, 42), (42, 46), (46, 48)):
        got, _ = model(ids[:, a:b].cuda(), cache)
        model(ids[:, a:b].cuda(), slab)
        ref, past = R.model_forward(W, cfg, ids[:, a:b], past)
        r16, p16 = R.model_forward(W16, cfg, ids[:, a:b], p16)
        close_logits(got, ref, r16)
    assert cache.seen_tokens == 48
    # the only attention layer's keys and values come of the same rows in both caches: v is copied;
    # k is rounded once in the pages, at four points in the slab (norm, cosine, products, sum)
    k, v = cache.read_kv(ATTN)
    ks, vs = slab.read_kv(ATTN)
    assert torch.equal(v, vs)
    assert ((k - ks).float().abs() <= 2.0 ** -6 * ks.float().abs().amax(-1, keepdim=True)).all()


def test_8_bit_pages_hold_the_bf16_pages_rows(micro):
    model = micro[0]
    g = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 512, (2, 50), generator=g).cuda()
    a, b = model.new_cache(2, 64, page=16), model.new_cache(2, 64, page=16, kv_dtype=torch.float8_e4m3fn)
    assert b.layers[ATTN]["k"].element_size() == 1
    x, _ = model(ids, a)
    y, _ = model(ids, b)
    for p, q, s in zip(a.read_kv(ATTN), b.read_kv(ATTN), ("ks", "vs")):
        p, q = p.float(), q.float()
        page, _ = b._rows(50)
        scale = b.layers[ATTN][s][page].transpose(1, 2)[..., None]          # of each row's page
        # half a step of e4m3 and, beside it, of the bf16 that it is compared with
        assert ((p - q).abs() <= torch.maximum((2.0 ** -4 + 2.0 ** -7) * p.abs(), 2.0 ** -10 * scale)).all()
    assert torch.isfinite(y.float()).all()


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn])
@pytest.mark.parametrize("temperature", [0.0, 0.8])
def test_speculative_decoder_eager_and_replayed(micro, kv, temperature):
    from lollm_amd.qwen3_5 import SpecDecoder
    model, mtp = micro[:2]
    print(f"case spec {kv} {temperature}", flush=True)
    prompts = torch.randint(0, 512, (3, 21), generator=torch.Generator().manual_seed(4)).cuda()

    def decoder():
        d = SpecDecoder(model, mtp, 3, 160, k=3, temperature=temperature, seed=5, page=16, kv_dtype=kv)
        d.prefill(prompts)
        d.step()
        return d

    a, b = decoder(), decoder()
    b.capture()
    for _ in range(12):
        a.step()
        b.replay()
        assert torch.equal(a.pending, b.pending) and torch.equal(a.cache.lengths, b.cache.lengths)
    assert a.tokens() == b.tokens()
    need = [-(-int(n) // 16) for n in a.cache.lengths]
    assert all(h >= n for h, n in zip(a.cache.held, need))


def test_decoder_out_of_pages_and_released(micro):
    from lollm_amd.qwen3_5 import SpecDecoder
    model, mtp = micro[:2]
    d = SpecDecoder(model, mtp, 2, 160, k=3, page=16, n_pages=6)
    d.prefill(torch.randint(0, 512, (2, 30), generator=torch.Generator().manual_seed(6)).cuda())
    with pytest.raises(RuntimeError, match="pool exhausted"):
        for _ in range(40):
            d.step()
    before = d.tokens()[0]
    lengths = d.cache.lengths.clone()
    d.cache.release(1)
    d.step()                                         # its pages go to the other one
    assert int(d.cache.lengths[0]) > int(lengths[0]) and d.tokens()[0][:len(before)] == before
    assert d.cache.held[1] == 0 and (d.cache.table[1] == -1).all()


def test_rollback_leaves_nothing_in_bf16_pages(micro):
    """4 tokens of which a + 1 are kept (a = 0 .. 3 over the batch, a page's end among them), then one
    more: bit for bit the logits of a cache that saw the kept ones only."""
    model, _, _, cfg = micro
    g = torch.Generator().manual_seed(7)
    prompts, blk, nxt = (torch.randint(0, cfg.vocab_size, (4, n), generator=g).cuda() for n in (46, 4, 1))
    acc = torch.arange(4, device="cuda").int()
    cache = model.new_cache(4, 80, page=16)
    model(prompts, cache, logits="last")
    short = cache.clone()
    model(blk, cache)
    cache.rollback(acc)
    got, _ = model(nxt, cache)
    for a in range(4):
        c = short.clone()
        model(blk[:, :a + 1], c)
        want, _ = model(nxt, c)
        assert torch.equal(got[a], want[a])


def test_generate_over_8_bit_pages(micro):
    from lollm_amd.generate import generate
    from lollm_amd.qwen3_5 import generate_mtp
    model, mtp = micro[:2]
    ids = list(range(5, 40))
    kw = dict(max_new_tokens=9, temperature=0.0, repetition_penalty=1.0, kv_dtype=torch.float8_e4m3fn)
    out = list(generate(model, ids, lambda t: "x" * len(t), [], page=32, **kw))
    assert len("".join(out)) == 9
    out = list(generate_mtp(model, mtp, ids, lambda t: "x" * len(t), [], k=2, **kw))
    assert len("".join(out)) == 9


@pytest.mark.parametrize("kv", [torch.bfloat16, torch.float8_e4m3fn])
def test_released_sequence_in_a_replayed_decoder(micro, kv):
    """Released between replays: its length stays a step's, its rows have no page, and the live one
    goes on to the end of the cache with pages that only it holds."""
    from lollm_amd.qwen3_5 import SpecDecoder
    model, mtp = micro[:2]
    print(f"case released {kv}", flush=True)
    d = SpecDecoder(model, mtp, 2, 96, k=3, page=16, kv_dtype=kv, n_pages=7)
    d.prefill(torch.randint(0, 512, (2, 30), generator=torch.Generator().manual_seed(8)).cuda())
    d.step()
    d.capture()
    d.cache.release(1)
    with pytest.raises(RuntimeError, match="capacity"):
        for _ in range(80):
            d.replay()
            assert int(d.cache.lengths[1]) <= 4 and (d.cache.table[1] == -1).all()
    assert int(d.cache.lengths[0]) > 92 and d.cache.held == [6, 0]


@pytest.mark.parametrize("page", [16, 64])
def test_logits_over_8_bit_pages(micro, page, monkeypatch):
    """A prompt, a token, a verify block and chunks over 8-bit pages, against the same forwards whose
    attention is the oracle's in 64 bits over what the cache's pages and scales hold: at the model's
    bf16 bar, which the same with K's scales and V's exchanged does not meet."""
    from lollm_amd import ops
    from paged_oracle import attention
    model, _, (W, W16), cfg = micro
    print(f"case logits over 8-bit pages of {page}", flush=True)
    ids = torch.randint(0, cfg.vocab_size, (2, 110), generator=torch.Generator().manual_seed(9))
    cache = model.new_cache(2, 128, page=page, kv_dtype=torch.float8_e4m3fn)
    past = p16 = None
    worst_exchanged = 0.0

    def oracle(c, first, second):
        def attn(q, k, v, table, kv_len, gate, **kw):
            s = {n: x.cpu() for n, x in c.layers[ATTN].items()}
            out, _ = attention(q.cpu(), s["k"], s["v"], c.table.cpu(), kv_len.cpu(), gate.cpu(), s[first], s[second])
            return out.bfloat16().cuda()
        return attn

    for a, b in ((0, 41), (41, 42), (42, 46), (46, 62), (62, 109), (109, 110)):
        x = ids[:, a:b].cuda()
        copies = cache.clone(), cache.clone()
        got, _ = model(x, cache)
        want = []
        for c, names in zip(copies, (("ks", "vs"), ("vs", "ks"))):
            with monkeypatch.context() as m:
                m.setattr(ops, "attn_paged", oracle(c, *names))
                want.append(model(x, c)[0].float())
        assert torch.equal(cache.layers[ATTN]["k"].view(torch.uint8), copies[0].layers[ATTN]["k"].view(torch.uint8))
        ref, past = R.model_forward(W, cfg, ids[:, a:b], past)
        r16, p16 = R.model_forward(W16, cfg, ids[:, a:b], p16)
        bar = 2 * float((r16.float() - ref).abs().max()) + 1e-3 * float(ref.abs().max())
        err = float((got.float() - want[0]).abs().max())
        assert err <= bar, f"tokens {a} .. {b}: off by {err}, bar {bar}"
        worst_exchanged = max(worst_exchanged, float((got.float() - want[1]).abs().max()) / bar)
    assert worst_exchanged > 1, worst_exchanged
