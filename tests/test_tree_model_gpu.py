"""A verify step over a tree of drafts, the model's and its caches': logits of every node against the
oracle along its path, the committed path, the walk that accepts it, and the loop of them, with bf16
and 4-bit weights, over slabs and pages."""

import pytest
import torch

from lollm_amd.qwen3_5.config import micro_config_dict
from oracle import qwen3_5_ref as R
from test_model_gpu import build, close_logits
from test_reference_gpu import _PLAIN_LINEAR, _dithered_linear


@pytest.fixture(scope="module")
def micro():
    return build(micro_config_dict())


# node 0 is the pending token; two sequences, one tree each
PARENTS = [[-1, 0, 0, 1, 1, 2, 3, 3, 4, 6, 5, 0, 11], [-1, 0, 1, 2, 3, 4, 5, 0, 7, 7, 0, 10, 1]]


def paths(parents):
    out = []
    for i in range(len(parents)):
        p, n = [], i
        while n >= 0:
            p.append(n)
            n = parents[n]
        out.append(p[::-1])
    return out


def oracle_nodes(W, cfg, past, ids, parents):
    """Logits (T, V) of one sequence's nodes, each from the oracle's pass over the node's whole path."""
    rows = []
    for p in paths(parents):
        lg, _ = R.model_forward(W, cfg, ids[p][None], past.clone())
        rows.append(lg[0, -1])
    return torch.stack(rows)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [None, 16, 64])
@pytest.mark.parametrize("context", [0, 1, 37])
def test_tree_forward_and_kept_path_against_the_oracle(micro, context, page):
    from lollm_amd import ops
    model, _, (W, W16), cfg = micro
    print("case tree forward", context, page, flush=True)
    g = torch.Generator().manual_seed(context)
    T = len(PARENTS[0])
    prompt = torch.randint(0, cfg.vocab_size, (2, context), generator=g)
    ids = torch.randint(0, cfg.vocab_size, (2, T), generator=g)
    cache = model.new_cache(2, 80, spec_slots=16, page=page)
    past, past16 = [[R.RefCache(cfg.num_hidden_layers) for _ in range(2)] for _ in range(2)]
    if context:
        model(prompt.cuda(), cache)
        for b in range(2):
            R.model_forward(W, cfg, prompt[b:b + 1], past[b])
            R.model_forward(W16, cfg, prompt[b:b + 1], past16[b])
    tree = ops.tree_masks(torch.tensor(PARENTS, dtype=torch.int32).cuda())
    got, _ = model(ids.cuda(), cache, tree=tree)
    want = torch.stack([oracle_nodes(W, cfg, past[b], ids[b], PARENTS[b]) for b in range(2)])
    want16 = torch.stack([oracle_nodes(W16, cfg, past16[b], ids[b], PARENTS[b]) for b in range(2)])
    close_logits(got, want, want16)
    # nothing is committed: the same call again gives the same bits
    assert cache.seen_tokens == context
    again, _ = model(ids.cuda(), cache, tree=tree)
    assert torch.equal(got, again)
    # a path of one sequence longer than the other's, then plain calls, a short and a long one
    keep = [paths(PARENTS[0])[9], paths(PARENTS[1])[8]]
    path = torch.full((2, T), -1, dtype=torch.int32)
    for b in range(2):
        path[b, :len(keep[b])] = torch.tensor(keep[b])
    count = torch.tensor([len(k) for k in keep], dtype=torch.int32)
    cache.keep_path(path.cuda(), count.cuda())
    assert cache.lengths.tolist() == [context + n for n in count.tolist()]
    for b in range(2):
        R.model_forward(W, cfg, ids[b, keep[b]][None], past[b])
        R.model_forward(W16, cfg, ids[b, keep[b]][None], past16[b])
    for n in (3, 1, 20):
        more = torch.randint(0, cfg.vocab_size, (2, n), generator=g)
        got, _ = model(more.cuda(), cache)
        want, want16 = ([R.model_forward(w, cfg, more[b:b + 1], p[b])[0] for b in range(2)]
                        for w, p in ((W, past), (W16, past16)))
        close_logits(got, torch.cat(want), torch.cat(want16))


@pytest.mark.gpu
def test_kept_paths_one_after_another(micro):
    """Trees on kept paths, some of a single node or of none; the halves change sides every time."""
    from lollm_amd import ops
    model, _, (W, W16), cfg = micro
    g = torch.Generator().manual_seed(5)
    cache = model.new_cache(2, 120, spec_slots=20)
    past, past16 = [[R.RefCache(cfg.num_hidden_layers) for _ in range(2)] for _ in range(2)]
    for turn, T in enumerate((5, 17, 1, 20, 9)):
        print("case kept path", turn, T, flush=True)
        parents = [[-1 if i == 0 else int(torch.randint(max(0, i - 4), i, (), generator=g)) for i in range(T)]
                   for _ in range(2)]
        ids = torch.randint(0, cfg.vocab_size, (2, T), generator=g)
        got, _ = model(ids.cuda(), cache, tree=ops.tree_masks(torch.tensor(parents, dtype=torch.int32).cuda()))
        close_logits(got, torch.stack([oracle_nodes(W, cfg, past[b], ids[b], parents[b]) for b in range(2)]),
                     torch.stack([oracle_nodes(W16, cfg, past16[b], ids[b], parents[b]) for b in range(2)]))
        keep = [paths(parents[0])[T - 1], [] if turn == 1 else paths(parents[1])[T // 2]]
        path = torch.full((2, T), -1, dtype=torch.int32)
        for b in range(2):
            path[b, :len(keep[b])] = torch.tensor(keep[b], dtype=torch.int32)
            if keep[b]:
                R.model_forward(W, cfg, ids[b, keep[b]][None], past[b])
                R.model_forward(W16, cfg, ids[b, keep[b]][None], past16[b])
        cache.keep_path(path.cuda(), torch.tensor([len(k) for k in keep], dtype=torch.int32).cuda())


def accept_by_hand(drawn, ids, parents):
    path = [0]
    while True:
        child = [i for i in range(len(ids)) if parents[i] == path[-1] and ids[i] == drawn[path[-1]]]
        if not child:
            return path, drawn[path[-1]]
        path.append(child[0])


@pytest.mark.gpu
@pytest.mark.parametrize("T", (1, 2, 7, 33, 64))
def test_tree_accept(T):
    from lollm_amd import ops
    print("case accept", T, flush=True)
    g = torch.Generator().manual_seed(T)
    B = 40
    parents = torch.tensor([[-1 if i == 0 else int(torch.randint(max(0, i - 5), i, (), generator=g)) for i in range(T)]
                            for _ in range(B)], dtype=torch.int32)
    parents[0, 1:] = torch.arange(T - 1, dtype=torch.int32)       # a chain, wholly accepted
    ids = torch.randint(0, 3, (B, T), generator=g, dtype=torch.int32)
    drawn = torch.randint(0, 3, (B, T), generator=g, dtype=torch.int32)
    drawn[0, :-1] = ids[0, 1:]
    mask, _ = ops.tree_masks(parents.cuda())
    path, count, nxt = (t.cpu() for t in ops.tree_accept(drawn.cuda(), ids.cuda(), mask))
    for b in range(B):
        want, token = accept_by_hand(drawn[b].tolist(), ids[b].tolist(), parents[b].tolist())
        assert int(count[b]) == len(want) and int(nxt[b]) == token
        assert path[b].tolist() == want + [-1] * (T - len(want))
    assert int(count[0]) == T


def drafts(truth, vocab, g):
    """A tree around a guess at the next tokens: the guess (wrong from some place on), siblings of each."""
    parents, ids, at = [-1], [truth[0]], 0
    cut = int(torch.randint(0, len(truth), (), generator=g))
    for i, t in enumerate(truth[1:]):
        for s in range(2):
            parents.append(at)
            ids.append(int(torch.randint(0, vocab, (), generator=g)))
        parents.append(at)
        ids.append(t if i < cut else (t + 1) % vocab)
        at = len(ids) - 1
    return parents, ids


@pytest.mark.gpu
@pytest.mark.parametrize("bits,page", [(16, None), (16, 16), (4, None), (4, 64)])
def test_greedy_tree_decoding(bits, page):
    """The whole step, again and again: a forward over the tree (4-bit weights among them), the argmax of
    every node, the walk, the commit.  Every emitted token is the argmax of a plain forward over the emitted
    text, up to a bf16 near-tie, and drafts are accepted."""
    from lollm_amd import ops
    model, _, _, cfg = build(micro_config_dict(), seed=3)
    if bits == 4:
        model.quantize(64, zeros=True)
    print("case tree decoding", bits, page, flush=True)
    g = torch.Generator().manual_seed(1)
    prompt = torch.randint(0, cfg.vocab_size, (2, 21), generator=g)
    plain = model.new_cache(2, 90)
    lg, _ = model(prompt.cuda(), plain, logits="last")
    first = lg[:, -1].float().argmax(-1)
    truth, tok = [first], first
    for _ in range(30):
        lg, _ = model(tok[:, None], plain)
        tok = lg[:, -1].float().argmax(-1)
        truth.append(tok)
    truth = torch.stack(truth, 1).tolist()
    cache = model.new_cache(2, 90, spec_slots=16, page=page)
    model(prompt.cuda(), cache)
    out, pending, accepted = [[int(first[0])], [int(first[1])]], first.int(), 0
    while min(map(len, out)) < 20:
        trees = [drafts([out[b][-1]] + truth[b][len(out[b]):len(out[b]) + 4], cfg.vocab_size, g) for b in range(2)]
        ids = torch.tensor([t[1] for t in trees], dtype=torch.int32).cuda()
        mask, depth = ops.tree_masks(torch.tensor([t[0] for t in trees], dtype=torch.int32).cuda())
        assert torch.equal(ids[:, 0], pending)
        lg, _ = model(ids, cache, tree=(mask, depth))
        B, T, V = lg.shape
        drawn = ops.sample_rows(lg.view(B * T, V), 0.0).view(B, T)
        path, count, pending = ops.tree_accept(drawn, ids, mask)
        cache.keep_path(path, count)
        for b in range(2):
            n = int(count[b])
            out[b] += ids[b, path[b, 1:n].long()].tolist() + [int(pending[b])]
            accepted += n - 1
    assert cache.lengths.tolist() == [21 + len(o) - 1 for o in out]
    assert accepted > 10
    for b in range(2):
        text = torch.cat([prompt[b], torch.tensor(out[b])])[None]
        lg, _ = model(text.cuda(), model.new_cache(1, 90))
        rows = lg[0, 20:-1].float()
        top = rows.max(-1).values
        mine = rows.gather(1, torch.tensor(out[b]).cuda()[:, None])[:, 0]
        assert (top - mine <= 2 ** -4 * rows.abs().max()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("group,zeros", [(32, False), (128, True)])
def test_4_bit_model_against_the_oracle(group, zeros):
    """The oracle over the values that the 4-bit weights hold, at the model tests' bar with the bf16 error
    measured over 17 flows of the oracle's own bf16 arithmetic, 16 of them with GEMM outputs that round
    differently (as for speculate in test_reference_gpu): the inputs of group 32 have a row (64) that amplifies
    roundings, on which those flows' 1 - cos alone is 0.0004 to 0.0020."""
    from lollm_amd import ops
    raw = micro_config_dict()
    model, mtp, (W, W16), cfg = build(raw, seed=2)
    model.quantize(group, zeros)
    mtp.quantize(group, zeros)
    print("case 4-bit model", group, zeros, flush=True)

    def held(w):
        codes, scales, zero = ops.q4_quantize(w.to(torch.bfloat16).cuda(), group, zeros)
        N, K = w.shape
        code = torch.stack([codes & 15, codes >> 4], -1).view(N, K // group, group).float()
        z = 8.0 if zero is None else zero.float()[..., None]
        return ((code - z) * scales.float()[..., None]).view(N, K).cpu()

    names = ("q_proj", "k_proj", "v_proj", "o_proj", "in_proj_qkv", "in_proj_z", "in_proj_b", "in_proj_a", "out_proj",
             "gate_proj", "up_proj", "down_proj", "mtp.fc")
    W, W16 = dict(W), dict(W16)
    for k in W:
        if any(f"{n}.weight" in k for n in names):
            W[k] = held_k = _held_rows(held, W[k])
            W16[k] = held_k.bfloat16()
    ids = torch.randint(0, cfg.vocab_size, (2, 70), generator=torch.Generator().manual_seed(2))
    ref, _ = R.model_forward(W, cfg, ids)
    flows = []
    try:
        for seed in range(-1, 16):
            R.linear = _PLAIN_LINEAR if seed < 0 else _dithered_linear(seed)
            flows.append(R.model_forward(W16, cfg, ids)[0].float())
    finally:
        R.linear = _PLAIN_LINEAR
    cache, got = model.new_cache(2, 96), []
    for a, b in ((0, 50), (50, 51), (51, 55), (55, 70)):
        got.append(model(ids[:, a:b].cuda(), cache)[0])
    got = torch.cat(got, 1).float().cpu()
    cs = torch.nn.functional.cosine_similarity
    spread, off = (max((1 - cs(f, ref, dim=-1)).max().item() for f in flows),
                   max((f - ref).abs().max().item() for f in flows))
    assert (1 - cs(got, ref, dim=-1)).max().item() <= max(2 * spread, 1e-3)
    assert (got - ref).abs().max().item() <= 2 * off + 1e-3 * ref.abs().max().item()
    from lollm_amd.qwen3_5 import speculate
    assert torch.isfinite(speculate(model, mtp, ids[:, :9]).float()).all()


def _held_rows(held, w):
    """Rows are quantised alone, so a matrix of a few rows is padded to the 64 that a call takes."""
    n = -w.shape[0] % 64
    return held(torch.cat([w, w.new_zeros(n, w.shape[1])]))[:w.shape[0]]


@pytest.mark.gpu
def test_4_bit_speculative_decoder_replayed(micro):
    """SpecDecoder over 4-bit weights, captured: its replays emit the eager decoder's tokens."""
    from lollm_amd.qwen3_5 import SpecDecoder
    out = []
    for graph in (False, True):
        model, mtp, _, cfg = build(micro_config_dict(), seed=4)
        model.quantize(64)
        mtp.quantize(64)
        dec = SpecDecoder(model, mtp, 2, 128, k=3, temperature=0.7, seed=5)
        prompt = torch.randint(0, cfg.vocab_size, (2, 30), generator=torch.Generator().manual_seed(2))
        dec.prefill(prompt.cuda())
        if graph:
            dec.capture()
        print("case 4-bit decoder", graph, flush=True)
        for _ in range(8):
            dec.replay() if graph else dec.step()
        torch.cuda.synchronize()
        out.append((dec.out_tokens.cpu().clone(), dec.out_count.cpu().clone()))
    n = int(min(out[0][1].min(), out[1][1].min()))
    assert n >= 8 and torch.equal(out[0][0][:, :8], out[1][0][:, :8])    # (a step emits one token at least)


@pytest.mark.gpu
def test_load_checkpoint_in_4_bits(tmp_path):
    """A checkpoint loaded with weight_bits=4 is the loaded model quantised: the same bits."""
    from lollm_amd.qwen3_5 import load, load_checkpoint
    from lollm_amd.qwen3_5.blocks import Projection4
    from test_checkpoint import micro_weights, write_checkpoint
    raw, W = micro_weights(seed=6)
    write_checkpoint(str(tmp_path), raw, W)
    model, mtp, unused = load_checkpoint(str(tmp_path), weight_bits=4, group=64)
    assert unused == [] and isinstance(model.model.layers[0].mlp.down, Projection4)
    assert isinstance(mtp.layers[0].mlp.down, Projection4) and model.model.layers[0].mlp.down.q4.group == 64
    ref = load(raw, dict(W), "hf", device="cuda").quantize(64)
    ids = torch.randint(0, raw["vocab_size"], (2, 7), generator=torch.Generator().manual_seed(1)).cuda()
    print("case checkpoint in 4 bits", flush=True)
    assert torch.equal(model(ids, model.new_cache(2, 32))[0], ref(ids, ref.new_cache(2, 32))[0])


@pytest.mark.gpu
def test_tree_beside_a_released_sequence(micro):
    """A released sequence's nodes mean nothing, take no pages and leave the others' tree as it is, over several
    trees; the others' numbers at the model tests' bar (keys are dealt out by all sequences' lengths)."""
    from lollm_amd import ops
    model, _, _, cfg = micro
    g = torch.Generator().manual_seed(12)
    prompt = torch.randint(0, cfg.vocab_size, (2, 20), generator=g).cuda()
    nodes = [torch.randint(0, cfg.vocab_size, (2, 13), generator=g).cuda() for _ in range(3)]
    mask, depth = ops.tree_masks(torch.tensor(PARENTS, dtype=torch.int32).cuda())
    path = torch.tensor([[0, 1, 3], [0, 1, 2]], dtype=torch.int32).cuda()
    count = torch.tensor([3, 2], dtype=torch.int32).cuda()
    out = []
    for released in (False, True):
        cache = model.new_cache(2, 96, spec_slots=13, page=16)
        model(prompt, cache)
        if released:
            cache.release(0)
        rows = []
        print("case tree beside a released sequence", released, flush=True)
        for ids in nodes:
            rows.append(model(ids, cache, tree=(mask, depth))[0][1].float())
            cache.keep_path(path, count)
        if released:
            assert cache.held[0] == 0
        assert int(cache.lengths[1]) == 20 + 3 * 2
        out.append(torch.cat(rows))
    cs = torch.nn.functional.cosine_similarity
    assert (1 - cs(out[0], out[1], dim=-1)).max().item() <= 1e-3


@pytest.mark.gpu
def test_tree_refusals(micro):
    from lollm_amd import ops
    model = micro[0]
    ids = torch.zeros(1, 5, dtype=torch.int64).cuda()
    tree = ops.tree_masks(torch.full((1, 5), -1, dtype=torch.int32).cuda())
    path, one = torch.zeros(1, 1, dtype=torch.int32).cuda(), torch.ones(1, dtype=torch.int32).cuda()
    with pytest.raises(ValueError):
        model(ids, model.new_cache(1, 32, spec_slots=4), tree=tree)
    with pytest.raises(ValueError):
        model(ids, model.new_cache(1, 32, spec_slots=8, kv_dtype=torch.float8_e4m3fn), tree=tree)
    cache = model.new_cache(1, 32, spec_slots=8)
    with pytest.raises(RuntimeError):
        cache.keep_path(path, one)
    with pytest.raises(RuntimeError):
        model(ids, model.new_cache(1, 4, spec_slots=8), tree=tree)
    model(ids[:, :3], cache)
    for after in (lambda: model(ids[:, :1], cache), lambda: cache.advance(0), cache.settle,
                  lambda: cache.rollback(one)):
        model(ids, cache, tree=tree)
        after()
        with pytest.raises(RuntimeError):
            cache.keep_path(path, one)
    model(ids, cache, tree=tree)
    cache.keep_path(path, one)
    with pytest.raises(RuntimeError):
        cache.rollback(one)
    with pytest.raises(RuntimeError):
        cache.keep_path(path, one)
    s = cache.layers[0]
    for bad in (lambda: ops.tree_keep_gdn(s["rep"], s["win"], cache.rec_half, cache.conv_off, path, one, 9, 4),
                lambda: ops.tree_keep_gdn(s["rep"], s["win"], cache.rec_half, cache.conv_off, path.long(), one, 5, 4),
                lambda: ops.tree_keep_kv(s["win"], s["win"], cache.lengths, path, one, 5),
                lambda: ops.tree_accept(path.long(), path, tree[0]), lambda: ops.tree_accept(path, path, tree[0])):
        with pytest.raises((ValueError, TypeError)):
            bad()
    with pytest.raises(ValueError):
        from lollm_amd.qwen3_5 import load
        load(micro_config_dict(), {}, "hf", weight_bits=8)


def test_tree_commit_entry_points_check_before_any_launch():
    from lollm_amd import _lib
    L = _lib.lib()
    p = 4096     # an address that no check reads
    assert L.lollm_tree_accept(p, p, None, p, p, p, 1, 4, None) == 1
    assert L.lollm_tree_accept(p, p, p, p, p, p, 1, 65, None) == 2
    assert L.lollm_tree_keep_kv(p, None, p, None, 0, 0, 0, 0, p, p, 4, 1, 4, 2, 256, 64, None) == 1
    assert L.lollm_tree_keep_kv(p, p, p, None, 0, 0, 0, 0, p, p, 4, 1, 4, 2, 128, 64, None) == 2
    assert L.lollm_tree_keep_kv(p, p, p, p, 1, 2, 4, 16, p, p, 4, 1, 4, 2, 256, 0, None) == 1
    assert L.lollm_tree_keep_kv(p, p, p, p, 2, 2, 4, 48, p, p, 4, 1, 4, 2, 256, 0, None) == 2
    assert L.lollm_tree_keep_kv(p, p, p, None, 0, 0, 0, 0, p, p, 4, 1, 4, 2, 256, 0, None) == 1
    assert L.lollm_tree_keep_gdn(p, p, p, p, p, p, 4, 1, 9, 4, 8, 12, 1024, 4, None) == 1
    assert L.lollm_tree_keep_gdn(p, p, p, p, p, p, 4, 1, 8, 4, 8, 10, 1024, 4, None) == 1
    assert L.lollm_tree_keep_gdn(p, p, p, p, p, p, 4, 1, 8, 4, 8, 11, 1020, 4, None) == 1
