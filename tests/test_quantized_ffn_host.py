"""The encoder's 8-bit FFN weights and the weights that they were made from, on the host (the
quantisation and the operator replaced by records of their arguments)."""

from __future__ import annotations

import copy
from types import SimpleNamespace

import pytest
import torch
from torch import nn
from transformers import XLMRobertaConfig

import latefuse_b200 as lf
from latefuse_b200 import engine


@pytest.fixture
def model(monkeypatch):
    conf = XLMRobertaConfig(vocab_size=64, hidden_size=64, num_hidden_layers=2, num_attention_heads=1, intermediate_size=72,
                            max_position_embeddings=40, pad_token_id=1, type_vocab_size=1)
    cfg = lf.LoraServingConfig(model_name="synthetic", lora_rank=16, batch_size=4, max_seq_len=32,
                               target_modules=["query"], device="cpu", dtype=torch.float32, hf_config=conf)
    made = lambda cls, w: SimpleNamespace(q=w.detach().clone(), scale=torch.ones(w.shape[0]), shape=tuple(w.shape))
    monkeypatch.setattr(engine.Int8Weight, "from_float", classmethod(made))
    monkeypatch.setattr(engine, "ffn_int8", lambda a, r, g, b, eps, up, ub, down, db, *rest, **more: (a, (up.q, down.q)))
    monkeypatch.setattr(engine, "add_layernorm", lambda o, *rest, **more: o)
    return lf.EncoderWithLora.random_init(conf, cfg, seed=1)


def ffn(model, idx=1):
    return model._ffn(idx, torch.zeros(3, 64), torch.zeros(3, 64))


def test_unchanged_weights_are_served(model):
    model.quantize_ffn()
    for _ in range(2):
        up, down = ffn(model)
        assert torch.equal(up, model.layers[1].wi) and torch.equal(down, model.layers[1].wo2)


def load(model):
    model.load_state_dict({k: torch.randn_like(v) for k, v in model.state_dict().items()})


def edit(model):
    with torch.no_grad():
        model.layers[1].wo2.mul_(2.0)


def replace(model):
    model.layers[1].wi = nn.Parameter(torch.randn(72, 64))


@pytest.mark.parametrize("change", [load, edit, replace])
def test_weights_that_changed_are_quantised_again(model, change):
    model.quantize_ffn()
    change(model)
    up, down = ffn(model)
    assert torch.equal(up, model.layers[1].wi) and torch.equal(down, model.layers[1].wo2)


def test_a_copy_has_weights_of_its_own(model):
    model.quantize_ffn()
    other = copy.deepcopy(model)
    edit(other)
    assert torch.equal(ffn(other)[1], other.layers[1].wo2) and torch.equal(ffn(model)[1], model.layers[1].wo2)


def test_unchanged_layers_are_not_quantised_again(model):
    model.quantize_ffn()
    kept = ffn(model, 0)
    edit(model)
    assert ffn(model, 0)[0] is kept[0] and ffn(model, 0)[1] is kept[1]
    again = ffn(model)
    assert ffn(model)[1] is again[1]


def test_weights_made_in_inference_mode(model):
    with torch.inference_mode():
        model.layers[1].wi = nn.Parameter(torch.randn(72, 64), requires_grad=False)
        model.quantize_ffn()
    assert torch.equal(ffn(model)[0], model.layers[1].wi)
