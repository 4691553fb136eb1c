"""Tree attention over slabs: a sequence's numbers come from its keys, not from what its slab could hold."""

import pytest
import torch

from test_attn_tree_gpu import D, close, inputs, reference, tree


@pytest.mark.gpu
@pytest.mark.parametrize("B,T,hq,hkv,lens", [(1, 16, 32, 4, [600]), (4, 16, 32, 4, [16, 900, 0, 333]), (1, 40, 2, 2, [1000]),
                                             (1, 7, 8, 2, [138]), (2, 9, 16, 2, [1023, 40])], ids=str)
def test_attn_tree_is_the_same_in_slabs_of_any_capacity(B, T, hq, hkv, lens):
    from lollm_amd import ops
    print("case tree attention, capacities", B, T, hq, hkv, lens, flush=True)
    q, k, v, gate = inputs(B, T, hq, hkv, lens, 4)
    _, words = tree(B, T, 4, 2)
    out = []
    for capacity in (1024, 8192, 8193, 20000):
        kc, vc = (torch.zeros(B, hkv, capacity, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        kc[:, :, :k.shape[2]], vc[:, :, :k.shape[2]] = k.cuda(), v.cuda()
        out.append(ops.attn_verify(q.cuda(), kc, vc, torch.tensor(lens, dtype=torch.int32).cuda(),
                                   gate.reshape(B, T, hq * D).cuda(), tree=words.cuda()))
    for got in out[1:]:
        assert torch.equal(got, out[0])
    close(out[0], *reference(q, k, v, gate, lens, words))
