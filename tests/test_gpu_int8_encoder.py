"""The 8-bit operators and the cross attention as they are used together: the encoder
with its FFN in 8-bit integers, and a cross-attention block that reads its packed
states (8-bit projections around the attention), each step against its own formula."""

from __future__ import annotations

import pytest
import torch
from transformers import XLMRobertaConfig

import latefuse_b200 as lf
from latefuse_b200.encoder_ops import ACT_GELU, ACT_NONE, add_layernorm
from test_gpu_cross_attention import check_sequence
from test_gpu_int8 import check_projection, ref_rows

pytestmark = pytest.mark.gpu


def encoder(cuda, dtype=torch.bfloat16, act="gelu"):
    conf = XLMRobertaConfig(vocab_size=512, hidden_size=256, num_hidden_layers=2, num_attention_heads=4,
                            intermediate_size=520, max_position_embeddings=300, pad_token_id=1, type_vocab_size=1,
                            hidden_act=act)
    cfg = lf.LoraServingConfig(model_name="synthetic", lora_rank=16, batch_size=4, max_seq_len=256,
                               target_modules=["query", "key", "value", "dense"], device=cuda, dtype=dtype, hf_config=conf)
    store = lf.AdapterStore(cfg)
    ids = store.fill_random_(3, std=0.02, generator=torch.Generator(device=cuda).manual_seed(1))
    return lf.EncoderWithLora.random_init(conf, cfg, seed=3), store, ids


def packed(model, store, ids, lengths):
    g = torch.Generator().manual_seed(2)
    tokens = torch.randint(5, 512, (len(lengths), max(lengths)), generator=g)
    mask = torch.arange(max(lengths)) < torch.tensor(lengths)[:, None]
    tokens = torch.where(mask, tokens, torch.ones_like(tokens))
    return tokens, mask, model.pack(tokens, lengths, store.slots([ids[i % 3] for i in range(len(lengths))]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("act", ["gelu", "relu"])
def test_ffn_step_is_its_formula(cuda, dtype, act):
    """One layer's feed-forward half: the LayerNorms bit for bit, each projection within its
    roundings of the formula on the integers the definition gives."""
    model, _, _ = encoder(cuda, dtype, act)
    model.quantize_ffn()
    layer, (up, down) = model.layers[1], model._ffn8[1]
    wq, ws = ref_rows(layer.wi.detach())
    assert torch.equal(up.q.double(), wq) and torch.equal(up.scale, ws)
    ao, h = (torch.randn(77, 256, device=cuda).to(dtype) for _ in range(2))
    with torch.no_grad():
        got = model._ffn(1, ao, h)
        h1 = add_layernorm(ao, h, layer.ln1.weight, layer.ln1.bias, model.eps)
        q, xs = ref_rows(h1)
        mid = lf.linear_int8(h1, up, layer.bi, act=ACT_GELU if act == "gelu" else ACT_NONE)
        check_projection(mid, q, xs, up.q, up.scale, layer.bi, ACT_GELU if act == "gelu" else ACT_NONE)
        mid = mid if act == "gelu" else torch.relu(mid)
        o = lf.linear_int8(mid, down, layer.bo2)
        check_projection(o, *ref_rows(mid), down.q, down.scale, layer.bo2, ACT_NONE)
        assert torch.equal(got, add_layernorm(o, h1, layer.ln2.weight, layer.ln2.bias, model.eps))


def test_encoder_with_8_bit_ffn_stays_near_and_comes_back(cuda):
    """Rounding to steps of max / 127 is off by a step / sqrt 12 on average: with max / rms of
    about 4 by 0.9% of the rms, for activations and weights each, so 1.3% a projection, under
    2% after two, under 3% of the state after two layers (the LayerNorms keep its size).
    A row that is 14% off has a cosine of 0.99 with the other model's."""
    model, store, ids = encoder(cuda)
    lengths = [200, 37, 256, 1, 129]
    tokens, mask, pb = packed(model, store, ids, lengths)
    with torch.no_grad():
        want = model.encode_packed(pb, store)
        model.quantize_ffn()
        got = model.encode_packed(pb, store)
        again = model.encode_packed(pb, store)
        model.quantize_ffn(False)
        back = model.encode_packed(pb, store)
    assert model._runner.status.item() == 0
    assert torch.equal(got, again) and torch.equal(back, want) and not torch.equal(got, want)
    cos = torch.nn.functional.cosine_similarity(got.float(), want.float(), dim=1)
    assert cos.min() > 0.99, cos.min().item()


@pytest.mark.parametrize("steps", [1, 40, 150])
def test_cross_attention_block_reads_the_states(cuda, steps):
    """Queries of `steps` tokens a sequence over the packed states of an encoder batch: keys and
    values by one 8-bit projection of the states, queries and output by others."""
    model, store, ids = encoder(cuda)
    model.quantize_ffn()
    lengths = [200, 37, 256, 1, 129]
    _, _, pb = packed(model, store, ids, lengths)
    with torch.no_grad():
        states = model.encode_packed(pb, store)
    g = torch.Generator(device=cuda).manual_seed(5)
    w_q, w_o = (torch.randn(256, 256, device=cuda, generator=g).bfloat16() / 16 for _ in range(2))
    w_kv = torch.randn(256, 256, device=cuda, generator=g).bfloat16() / 16  # 4 query heads over 2 key heads of 64
    b_kv = torch.randn(256, device=cuda, generator=g).bfloat16()
    q8, kv8, o8 = (lf.Int8Weight.from_float(w) for w in (w_q, w_kv, w_o))
    kv = lf.linear_int8(states, kv8, b_kv)
    check_projection(kv, *ref_rows(states), kv8.q, kv8.scale, b_kv, ACT_NONE)
    kv_lengths = [lengths[b] for b in pb.order]  # packed order
    x = torch.randn(steps * len(lengths), 256, device=cuda, generator=g).bfloat16()
    q = lf.linear_int8(x, q8)
    batch = lf.cross_batch([steps] * len(lengths), kv_lengths, cuda)
    ctx = lf.cross_attention_varlen(q, kv[:, :128], kv[:, 128:], batch, 4, 2)
    k0 = 0
    for i, n in enumerate(kv_lengths):
        rows = slice(i * steps, (i + 1) * steps)
        check_sequence(ctx[rows], q[rows], kv[k0:k0 + n, :128], kv[k0:k0 + n, 128:], 4, 2, 0.125)
        k0 += n
    out = lf.linear_int8(ctx, o8)
    check_projection(out, *ref_rows(ctx), o8.q, o8.scale, None, ACT_NONE)
