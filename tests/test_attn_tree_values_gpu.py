"""Tree attention over cached values of any size: the result does not depend on how a call deals its keys
out (bars and 64-bit reference of test_attn_tree_gpu)."""

import pytest
import torch

from test_attn_tree_gpu import D, close, inputs, reference, run, tree

KINDS = ("slab", (16, 16), (64, 16), (64, 8))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS, ids=str)
@pytest.mark.parametrize("B,T,hq,hkv,lens", [(2, 24, 32, 4, [1500, 777]), (1, 64, 16, 2, [2900]), (2, 3, 8, 2, [700, 90])],
                         ids=str)
def test_attn_tree_columns_of_any_size(B, T, hq, hkv, lens, kind):
    """A head's value columns from 2^-30 to 1, each at its own bar, the keys of some calls in several parts."""
    print("case tree attention, sizes of columns", B, T, kind, flush=True)
    q, k, v, gate = inputs(B, T, hq, hkv, lens, 21)
    v = (v.float() * torch.exp2(-(torch.arange(D) * 37 % 31).float())).bfloat16()
    _, words = tree(B, T, 6, 5)
    got, kh, vh = run(kind, q, k, v, gate, lens, words)
    close(got, *reference(q, kh, vh, gate, lens, words))


@pytest.mark.gpu
@pytest.mark.parametrize("size", (-30, 0, 30))
@pytest.mark.parametrize("kind", KINDS[:3], ids=str)
def test_attn_tree_an_infinite_value_stays_in_its_column(kind, size):
    """A committed key's value that is infinite in one column: that column is not finite, the others are what
    they are without it."""
    B, T, hq, hkv, lens = 2, 24, 32, 4, [1500, 777]
    print("case tree attention, an infinite value", kind, size, flush=True)
    q, k, v, gate = inputs(B, T, hq, hkv, lens, 22)
    v = (v.float() * 2.0 ** size).bfloat16()
    _, words = tree(B, T, 6, 5)
    ref, mag = reference(q, k, v, gate, lens, words)
    v[:, :, 100, 5] = float("inf")
    got, _, _ = run(kind, q, k, v, gate, lens, words)
    got = got.cpu().view(ref.shape)
    others = torch.arange(D) != 5
    assert not torch.isfinite(got[..., 5]).any()
    close(got[..., others].contiguous(), ref[..., others], mag[..., others])
