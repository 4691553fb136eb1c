"""Rounding to 4 bits where a group's numbers are tiny."""

import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("zeros", (False, True))
@pytest.mark.parametrize("group", (32, 64, 128))
@pytest.mark.parametrize("size", (1e-30, 2e-37, 1e-37, 2e-38, 1e-38, 5e-39, 0.0))
def test_q4_quantize_groups_of_tiny_numbers(group, zeros, size):
    """Every value within half a step of its code's, the range's ends by what the scale's rounding (coarse where
    bf16 has few bits left) moves them, and with a zero that is rounded itself half a step more."""
    from lollm_amd import ops
    print("case quantise tiny", group, zeros, size, flush=True)
    g = torch.Generator().manual_seed(group)
    w = (torch.rand(64, 128, generator=g) * 2 - 1) * size
    w[:, ::3] = 0
    w = w.bfloat16()
    codes, scales, zero = ops.q4_quantize(w.cuda(), group, zeros)
    v, s = w.double().view(64, 128 // group, group), scales.double().cpu()[..., None]
    lo, hi = v.amin(-1, keepdim=True).clamp(max=0), v.amax(-1, keepdim=True).clamp(min=0)
    step = (hi - lo) / 15 if zeros else torch.maximum(hi, -lo) / 7.5
    code = torch.stack([codes & 15, codes >> 4], -1).view(v.shape).cpu().double()
    back = (code - (8.0 if zero is None else zero.cpu().double()[..., None])) * s
    room = s * (1.0 if zeros else 0.5) + 15 * (s - step).abs() + s * 2 ** -20   # (products with the reciprocal, fp32)
    assert ((back - v).abs() <= room).all()
    assert (back[v == 0] == 0).all() or zeros
