"""What gemm_q4 does on the host, without a device: a stand-in for the library sees each call's arguments."""

import gc

import pytest
import torch

from lollm_amd import _lib, ops
from lollm_amd.qwen3_5 import MTP, Qwen3_5Model, blocks, load
from lollm_amd.qwen3_5.config import micro_config_dict
from lollm_amd.qwen3_5.modeling_qwen3_5 import DecoderLayer


@pytest.fixture
def library(monkeypatch):
    """Host tensors as the current device's; the calls of lollm_gemm_q4 go to `calls`."""
    class Library:
        calls = []

        def lollm_gemm_q4(self, *args):
            ws = args[6]
            alive = [t for t in gc.get_objects() if issubclass(type(t), torch.Tensor) and t.data_ptr() == ws] if ws else []
            self.calls.append((args, sum(t.numel() * t.element_size() for t in alive)))
            return 0

    stand_in = Library()
    stand_in.calls = []
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: -1)      # (what a host tensor's get_device() says)
    monkeypatch.setattr(torch._C, "_cuda_getCurrentRawStream", lambda dev: 0)
    monkeypatch.setattr(_lib, "lib", lambda: stand_in)
    monkeypatch.setattr(ops, "_q4_workspace_bytes", lambda M, N, K, group, dev: 6 * M * 32)
    return stand_in


def test_gemm_q4_holds_its_workspace_until_the_call_has_returned(library):
    """The call releases the interpreter's lock: a block that went back to the allocator before it may be
    another thread's by the time its kernels are launched."""
    N, K, M = 64, 256, 200
    w = ops.Q4Weight(torch.empty(N * K // 2 + 4 * N, dtype=torch.uint8), N, K, 128, False, ops.GEMM_NONE)
    ops.gemm_q4(torch.zeros(M, K, dtype=torch.bfloat16), w)
    (args, alive), = library.calls
    assert args[7] == 6 * M * 32 and args[6] and alive >= args[7]


def test_gemm_q4_of_few_rows_takes_no_workspace(library):
    w = ops.Q4Weight(torch.empty(64 * 64 + 64 * 4, dtype=torch.uint8), 64, 128, 64, False, ops.GEMM_NONE)
    ops.gemm_q4(torch.zeros(64, 128, dtype=torch.bfloat16), w)
    (args, _), = library.calls
    assert args[6] is None and args[7] == 0


def linear(N=128, K=256):
    return blocks.Projection(torch.zeros(N, K))


def held(group=64, zeros=False, N=128, K=256):
    p = blocks.Projection4.__new__(blocks.Projection4)
    p.q4 = ops.Q4Weight(torch.empty(0, dtype=torch.uint8), N, K, group, zeros, ops.GEMM_NONE)
    p.N, p.K, p.epilogue = N, K, ops.GEMM_NONE
    return p


@pytest.mark.parametrize("group", (0, 16, 48, 100, 256))
def test_quantized_refuses_groups_that_no_weight_has(group):
    """(Instead of leaving everything in bf16.)"""
    with pytest.raises(ValueError, match="32, 64, 128"):
        blocks.quantized(linear(), group)
    with pytest.raises(ValueError, match="32, 64, 128"):
        load(micro_config_dict(), {}, "hf", weight_bits=4, group=group)


def test_quantized_refuses_another_group_or_zeros_for_what_is_in_4_bits():
    p = held(64, False)
    assert blocks.quantized(p, 64) is p and blocks.quantized(p, 64, zeros=False) is p
    for group, zeros in ((128, False), (64, True), (32, True)):
        with pytest.raises(ValueError, match="groups of 64 without zeros"):
            blocks.quantized(p, group, zeros)
    odd = linear(100, 256)
    assert blocks.quantized(odd, 64) is odd        # no 4-bit form: bf16 as it was


def test_a_refused_quantize_changes_nothing():
    """The projections are looked over before the first of them is rounded."""
    model = Qwen3_5Model.__new__(Qwen3_5Model)
    model.model = type("Inner", (), {})()
    layers = []
    for late in (linear(), held(64)):
        mlp = blocks.MLP.__new__(blocks.MLP)
        mlp.gate_up, mlp.down = linear(), late
        mixer = blocks.GatedDeltaNet.__new__(blocks.GatedDeltaNet)
        mixer.in_proj, mixer.out_proj = linear(), linear()
        layer = DecoderLayer.__new__(DecoderLayer)
        layer.layer_type, layer.linear_attn, layer.mlp = "linear_attention", mixer, mlp
        layers.append(layer)
    model.model.layers, model.lm_head = layers, linear()
    before = model.projections()
    with pytest.raises(ValueError, match="groups of 64"):
        model.quantize(128)
    assert all(a is b for a, b in zip(before, model.projections()))
    mtp = MTP.__new__(MTP)
    mtp.fc, mtp.layers = linear(), layers[1:]
    fc = mtp.fc
    with pytest.raises(ValueError, match="groups of 64"):
        mtp.quantize(32)
    assert mtp.fc is fc


def test_a_product_in_4_bits_refuses_what_would_have_to_follow_it(library):
    """A gradient that would silently be lost, a function transform, a trace."""
    p = held(64, False, 64, 128)
    p.q4.packed = torch.empty(64 * 64 + 64 * 4, dtype=torch.uint8)
    x = torch.zeros(3, 128, dtype=torch.bfloat16)
    p(x)
    leaf = x.clone().requires_grad_()
    with torch.no_grad():
        p(leaf)
    p(leaf.detach())
    assert len(library.calls) == 3

    def dual():
        with torch.autograd.forward_ad.dual_level():
            p(torch.autograd.forward_ad.make_dual(x, x))

    for call in (lambda: p(leaf), dual, lambda: torch.func.vmap(p)(x[None]), lambda: torch.func.jvp(p, (x,), (x,)),
                 lambda: torch.jit.trace(p.__call__, (x,))):
        with pytest.raises(RuntimeError, match="4-bit weight"):
            call()
    assert len(library.calls) == 3


def test_the_in_projections_weight_is_gone_in_4_bits():
    mixer = blocks.GatedDeltaNet.__new__(blocks.GatedDeltaNet)
    mixer.in_proj = linear()
    assert mixer.w_in is mixer.in_proj.weight
    mixer.in_proj = held()
    with pytest.raises(AttributeError, match="in 4 bits"):
        mixer.w_in
