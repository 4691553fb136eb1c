"""The Gated DeltaNet layer over a tree whose first nodes forget nearly everything and whose later ones nearly
nothing (inputs, 64-bit reference and bars of test_gdn_tree_gpu)."""

import pytest
import torch

from test_gdn_tree_gpu import D, check, layer, tree


@pytest.mark.gpu
@pytest.mark.parametrize("big", (30.0, 1e3, 1e4, 1e6, 3e38))
@pytest.mark.parametrize("T,spread", [(12, 1), (40, 1), (40, 4), (64, 1)])
def test_gdn_tree_strong_decays_above_weak_ones(T, spread, big):
    """Weights between later nodes are e^0 .. e^-9 whatever the sums above them are, infinite ones among them."""
    B, Hk, Hv, slots = 2, 2, 4, 64
    print("case gdn tree, decays", T, spread, big, flush=True)
    s = layer(B, T, Hk, Hv, slots, 31)
    C = 2 * Hk * D + Hv * D
    a = s["proj"][..., C + Hv * D + Hv:C + Hv * D + 2 * Hv]
    s["dt_bias"][:] = 0.0
    s["A_log"][:] = torch.tensor([0.0, 2.0, 4.0, 5.0])
    a[:, :3] = big
    a[:, 3:] = -7.0
    check(s, tree(B, T, spread, 1), B, T, Hk, Hv, slots)
