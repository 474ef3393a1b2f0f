"""The 8-bit operators and the cross attention on tensors of more than 2^31 elements: the rows
behind that border are the bits that a call on those rows alone gives."""

from __future__ import annotations

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200.encoder_ops import ACT_GELU
from test_gpu_cross_attention import check_sequence
from test_gpu_int8 import activations, weight

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [4096, 4099])
def test_far_projection_rows(cuda, n):
    """Outputs stored by TMA and row by row."""
    m = (1 << 31) // n + 1000
    x = activations(cuda, m, 32, torch.bfloat16, n)
    wt = lf.Int8Weight(*weight(cuda, n, 32, 1))
    y = lf.linear_int8(x, wt, act=ACT_GELU)
    assert y.numel() > 1 << 31
    for rows in (slice(0, 300), slice(m - 1300, m)):
        assert torch.equal(y[rows], lf.linear_int8(x[rows], wt, act=ACT_GELU))


@pytest.mark.parametrize("k", [4096, 4095])
def test_far_quantised_rows(cuda, k):
    m = (1 << 31) // k + 500
    x = torch.zeros(m, k, device=cuda, dtype=torch.float16)
    x[-700:] = activations(cuda, 700, k, torch.float16, 3)
    got, want = lf.quantize_rows(x), lf.quantize_rows(x[-700:])
    assert torch.equal(got.q[-700:], want.q) and torch.equal(got.scale[-700:], want.scale)
    wt = lf.Int8Weight(*weight(cuda, 40, k, 1))
    assert torch.equal(lf.linear_int8(got, wt)[-700:], lf.linear_int8(want, wt))


def test_far_layernorm_rows(cuda):
    m, h = (1 << 31) // 4096 + 500, 4096
    a = torch.ones(m, h, device=cuda, dtype=torch.bfloat16)
    a[-700:] = activations(cuda, 700, h, torch.bfloat16, 3)
    g, b = torch.rand(h, device=cuda).bfloat16() + 0.5, torch.randn(h, device=cuda).bfloat16()
    (out, rows), (want, few) = lf.add_layernorm_int8(a, None, g, b, 1e-5), lf.add_layernorm_int8(a[-700:], None, g, b, 1e-5)
    assert torch.equal(out[-700:], want) and torch.equal(rows.q[-700:], few.q) and torch.equal(rows.scale[-700:], few.scale)


@pytest.mark.parametrize("q_len", [1, 40, 140])
def test_far_queries(cuda, q_len):
    """Queries and outputs of rows whose offsets pass 2^31 elements, and rows before them."""
    heads, d = 32, 128
    rows = (1 << 31) // (heads * d) + 1000
    q = torch.zeros(rows, heads * d, device=cuda, dtype=torch.bfloat16)
    q[:q_len], q[-q_len:] = torch.randn(2, q_len, heads * d, device=cuda).bfloat16()
    k, v = torch.randn(2, 400, heads * d, device=cuda).bfloat16()
    batch = lf.cross_batch([q_len] * 2, [300, 100], cuda, q_starts=[0, rows - q_len])
    out = torch.full_like(q, 7.0)
    lf.cross_attention_varlen(q, k, v, batch, heads, out=out)
    check_sequence(out[:q_len], q[:q_len], k[:300], v[:300], heads, heads, d ** -0.5)
    check_sequence(out[-q_len:], q[-q_len:], k[300:], v[300:], heads, heads, d ** -0.5)
    assert (out[q_len:-q_len] == 7).all()
