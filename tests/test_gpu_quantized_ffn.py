"""The encoder's 8-bit FFN after its weights changed: outputs of the weights that it has now."""

from __future__ import annotations

import pytest
import torch

from test_gpu_int8_encoder import encoder, packed

pytestmark = pytest.mark.gpu


def scale(model):
    with torch.no_grad():
        for layer in model.layers:
            layer.wi.mul_(-0.5)


def load(model):
    g = torch.Generator(device="cuda").manual_seed(11)
    model.load_state_dict({k: v + 0.02 * torch.randn(v.shape, device=v.device, generator=g).to(v.dtype)
                           for k, v in model.state_dict().items()})


def there_and_back(model):
    model.to("cpu")
    scale(model)
    model.to("cuda")


@pytest.mark.parametrize("change", [scale, load, there_and_back])
def test_changed_weights_are_served(cuda, change):
    model, store, ids = encoder(cuda)
    _, _, pb = packed(model, store, ids, [30, 7, 64])
    with torch.no_grad():
        model.quantize_ffn()
        before = model.encode_packed(pb, store)
        change(model)
        got = model.encode_packed(pb, store)
        model.quantize_ffn()
        assert torch.equal(got, model.encode_packed(pb, store)) and not torch.equal(got, before)


def test_a_capture_wants_them_quantised_before(cuda):
    model, store, ids = encoder(cuda)
    _, _, pb = packed(model, store, ids, [30, 7, 64])
    with torch.no_grad():
        model.quantize_ffn()
        model.encode_packed(pb, store)
        ao, h = torch.randn(2, 9, 256, device=cuda).bfloat16()
        want = model._ffn(1, ao, h)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model._ffn(1, ao, h)
        graph.replay()
        assert torch.equal(out, want)
        scale(model)
        with pytest.raises(RuntimeError, match="before the capture"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                model._ffn(1, ao + 1, h)
        got = model._ffn(1, ao, h)
        assert not torch.equal(got, want)
        graph.replay()  # the captured forward reads the same weights
        assert torch.equal(out, got)
