"""What gemm_q4 does on the host, without a device: a stand-in for the library sees each call's arguments."""

import gc

import pytest
import torch

from lollm_amd import _lib, ops


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
