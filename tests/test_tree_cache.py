"""A tree of drafts that a cache holds uncommitted ends with whatever writes over its rows."""

import pytest
import torch

from lollm_amd.qwen3_5 import Qwen3_5Cache, Qwen3_5Config, Qwen3_5PagedCache
from lollm_amd.qwen3_5.config import micro_config_dict

LAYER = 3     # full attention


def slab(batch=2, max_len=64, spec_slots=8):
    return Qwen3_5Cache(Qwen3_5Config.from_hf(micro_config_dict()), batch, max_len, spec_slots, "cpu")


def pages(batch=2, max_len=64, spec_slots=8, **kw):
    return Qwen3_5PagedCache(Qwen3_5Config.from_hf(micro_config_dict()), batch, max_len, spec_slots, "cpu", page=16, **kw)


def open_tree(c, T=5):
    c.tree_begins(T)
    c.reserve(T)
    c.tree_written(T)


def ended(c):
    with pytest.raises(RuntimeError, match="follows a forward over a tree"):
        c.keep_path(torch.zeros(2, 1, dtype=torch.int32), torch.ones(2, dtype=torch.int32))


@pytest.mark.parametrize("make", (slab, pages))
def test_appended_rows_end_the_tree(make):
    c = make()
    c.advance(9)
    open_tree(c)
    rows = torch.zeros(2, 2, 1, 256, dtype=torch.bfloat16)
    c.append_kv(LAYER, rows[:, :, :0], rows[:, :, :0])      # writes nothing
    assert c.tree_T == 5
    c.append_kv(LAYER, rows, rows)
    ended(c)


@pytest.mark.gpu
def test_a_forward_that_commits_nothing_ends_the_tree():
    """hidden_states writes its tokens' rows and records where the tree's are."""
    from lollm_amd import ops
    from test_model_gpu import build
    model = build(micro_config_dict())[0]
    c = model.new_cache(2, 32, spec_slots=8)
    ids = torch.zeros(2, 5, dtype=torch.int64).cuda()
    model(ids[:, :2], c)
    model(ids, c, tree=ops.tree_masks(torch.full((2, 5), -1, dtype=torch.int32).cuda()))
    assert c.tree_T == 5
    model.hidden_states(ids[:, :1], c)
    ended(c)
