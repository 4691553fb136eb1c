"""The Gated DeltaNet layer over a tree whose queries and keys cancel nearly all of the committed state (64-bit
reference and bars of test_gdn_tree_gpu)."""

import pytest
import torch

from test_gdn_tree_gpu import D, K, check, layer, tree


@pytest.mark.gpu
@pytest.mark.parametrize("size", (1.0, 2.0 ** 12, 2.0 ** 14))
@pytest.mark.parametrize("T,spread", [(1, 1), (12, 3), (20, 1), (40, 8)])
def test_gdn_tree_states_that_cancel(T, spread, size):
    """S0 = size a b^T + 0.1 noise, a orthogonal to all queries and keys: what is left is the noise's, which the norm
    behind it scales to one.  Sums in fp32 are off by some 2^-24 size |b| / 11 of each of a few additions, at
    2^14 below 2^-10 of the result; 16 bits of the state by 2^-18 size |b| / 20, which passes the bar.  Queries and keys
    are single inputs from 20 on, whose SiLU is the input itself, so that no rounding of theirs spoils the angle."""
    B, Hk, Hv, slots = 2, 1, 2, 40
    print("case gdn tree, states", T, spread, size, flush=True)
    s = layer(B, T, Hk, Hv, slots, 17)
    g = torch.Generator().manual_seed(T)
    s["conv_w"][:] = 0
    s["conv_w"][:, K - 1] = 1
    s["proj"][..., :2 * D] = (20 + 20 * torch.rand(B, T, 2 * D, generator=g)).bfloat16()
    s["replay"][:] = 0
    for b in range(B):
        rows = s["proj"][b, :, :2 * D].double().reshape(2 * T, D)
        for h in range(Hv):
            a = torch.randn(D, generator=g).double()
            basis = torch.linalg.qr(rows.t())[0]
            for _ in range(2):
                a = a - basis @ (basis.t() @ a)
            a = a / a.norm()
            state = size * a[:, None] * torch.randn(D, generator=g).double()[None] + 0.1 * torch.randn(D, D, generator=g).double()
            s["rec"][b, int(s["rec_half"][b]), h] = state.float()
    check(s, tree(B, T, spread, T), B, T, Hk, Hv, slots)
