"""quantize() lets the bf16 weights go: not while a graph may replay over them."""

import pytest
import torch

from lollm_amd.qwen3_5 import SpecDecoder
from lollm_amd.qwen3_5.blocks import Projection
from lollm_amd.qwen3_5.config import micro_config_dict
from test_model_gpu import build


@pytest.mark.gpu
def test_quantize_after_a_decoders_capture_is_refused():
    """The replays emit the eager decoder's tokens afterwards, as the weights are where they were."""
    out = []
    for graph in (False, True):
        model, mtp, _, cfg = build(micro_config_dict(), seed=4)
        dec = SpecDecoder(model, mtp, 2, 128, k=3, temperature=0.7, seed=5)
        prompt = torch.randint(0, cfg.vocab_size, (2, 30), generator=torch.Generator().manual_seed(2))
        dec.prefill(prompt.cuda())
        if graph:
            dec.capture()
            for holder in (model, mtp):
                with pytest.raises(RuntimeError, match="graph"):
                    holder.quantize(64)
            assert all(type(p) is Projection for p in model.projections() + [mtp.fc] + mtp.layers[0].projections())
        print("case decoder", graph, flush=True)
        for _ in range(6):
            dec.replay() if graph else dec.step()
        torch.cuda.synchronize()
        out.append(dec.out_tokens.cpu()[:, :6])
    assert torch.equal(out[0], out[1])


@pytest.mark.gpu
def test_quantize_after_a_captured_forward_is_refused():
    model = build(micro_config_dict(), seed=4)[0]
    ids = torch.zeros(1, 4, dtype=torch.int64).cuda()
    cache = model.new_cache(1, 64)
    model(ids, cache)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        model(ids, cache)
    with pytest.raises(RuntimeError, match="graph"):
        model.quantize(64)


@pytest.mark.gpu
def test_quantize_after_eager_calls_and_then_a_capture():
    """Eager calls hold nothing, and what is in this form already may be asked for again."""
    model, mtp, _, cfg = build(micro_config_dict(), seed=4)
    dec = SpecDecoder(model, mtp, 2, 128, k=2)
    dec.prefill(torch.zeros(2, 9, dtype=torch.int64).cuda())
    dec.step()
    model.quantize(64)
    mtp.quantize(64)
    dec.capture()
    held = model.projections()
    model.quantize(64)
    mtp.quantize(64)
    assert all(a is b for a, b in zip(held, model.projections()))
