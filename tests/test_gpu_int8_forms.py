"""The 8-bit feed-forward half in the forms that its other tests leave out: f32, without
biases, without a residual, without an activation, leading dimensions, other widths; and
the encoder's padded forward with it."""

from __future__ import annotations

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200 import ffn_int8, linear_int8
from latefuse_b200.encoder_ops import ACT_GELU, ACT_NONE, add_layernorm
from test_gpu_int8 import DTYPES, activations, check_projection, ref_rows, weight
from test_gpu_int8_encoder import encoder

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h,i", [(1, 8, 1), (2, 1024, 33), (19, 264, 1000), (70, 64, 2049), (300, 1032, 520),
                                   (2100, 128, 1024)])
@pytest.mark.parametrize("act", [ACT_GELU, ACT_NONE])
def test_ffn_int8_in_every_form(cuda, dtype, m, h, i, act):
    """h bit for bit add_layernorm's, and o within its roundings of the formula on the integers
    of the middle that the up projection gives, with and without residual and biases."""
    a, r = activations(cuda, m, h, dtype, 1), activations(cuda, m, h, dtype, 2)
    g, b = torch.rand(h, device=cuda).to(dtype) + 0.5, torch.randn(h, device=cuda).to(dtype)
    (up, ups), (down, downs) = weight(cuda, i, h, 3), weight(cuda, h, i, 4)
    u8, d8 = lf.Int8Weight(up, ups), lf.Int8Weight(down, downs)
    ub, db = torch.randn(i, device=cuda).to(dtype), torch.randn(h, device=cuda).to(dtype)
    for residual, up_bias, down_bias in ((r, ub, db), (None, ub, None), (r, None, db), (None, None, None)):
        x, o = ffn_int8(a, residual, g, b, 1e-5, u8, up_bias, d8, down_bias, act=act)
        assert torch.equal(x, add_layernorm(a, residual, g, b, 1e-5))
        mid = linear_int8(x, u8, up_bias, act=act)
        check_projection(mid, *ref_rows(x), up, ups, up_bias, act)
        check_projection(o, *ref_rows(mid), down, downs, down_bias, ACT_NONE)


def test_ffn_int8_leading_dimensions_and_no_rows(cuda):
    a, r = (activations(cuda, 24, 64, torch.bfloat16, s) for s in (1, 2))
    g, b = torch.ones(64, device=cuda).bfloat16(), torch.zeros(64, device=cuda).bfloat16()
    up, down = lf.Int8Weight(*weight(cuda, 200, 64, 3)), lf.Int8Weight(*weight(cuda, 64, 200, 4))
    want = ffn_int8(a, r, g, b, 1e-5, up, None, down, None)
    got = ffn_int8(a.view(2, 3, 4, 64), r.view(2, 3, 4, 64), g, b, 1e-5, up, None, down, None)
    for x, y in zip(got, want):
        assert x.shape == (2, 3, 4, 64) and torch.equal(x.reshape(24, 64), y)
    for x in ffn_int8(a[:0], r[:0], g, b, 1e-5, up, None, down, None):
        assert x.shape == (0, 64)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("lora", [True, False])
def test_padded_forward_with_8_bit_ffn(cuda, dtype, lora):
    """Every layer's feed-forward half of the padded forward is the operators' composition, bit
    for bit, and the forward without it comes back."""
    model, store, ids = encoder(cuda, dtype)
    tokens = torch.randint(5, 512, (3, 40), generator=torch.Generator().manual_seed(2)).to(cuda)
    mask = torch.arange(40, device=cuda) < torch.tensor([40, 7, 1], device=cuda)[:, None]
    tokens = torch.where(mask, tokens, torch.ones_like(tokens))
    weights = lf.BatchAssembler(store, model.config).batch_lora(list(ids[:3]), seq_len=40) if lora else None
    halves, ffn = [], model._ffn

    def kept(idx, ao, h):
        given = ao.clone(), h.clone()
        halves.append((idx, *given, ffn(idx, ao, h)))
        return halves[-1][3]

    with torch.no_grad():
        want = model.encode(tokens, mask, weights, apply_lora=lora)
        model.quantize_ffn()
        model._ffn = kept
        got = model.encode(tokens, mask, weights, apply_lora=lora)
        for idx, ao, h, out in halves:
            layer, (up, down) = model.layers[idx], model._ffn8[idx]
            x, o = ffn_int8(ao, h, layer.ln1.weight, layer.ln1.bias, model.eps, up, layer.bi, down, layer.bo2)
            assert torch.equal(out, add_layernorm(o, x, layer.ln2.weight, layer.ln2.bias, model.eps))
        assert len(halves) == 2 and got.shape == (3, 40, 256) and torch.equal(got.view(120, 256), halves[-1][3])
        model._ffn = ffn
        model.quantize_ffn(False)
        assert torch.equal(model.encode(tokens, mask, weights, apply_lora=lora), want) and not torch.equal(got, want)
