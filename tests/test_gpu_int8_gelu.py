"""The fused GELU of the 8-bit projection on chosen inputs, against 64 bits.

A row (a token) of one element x is the integer 127 with the scale x / 127, so with a weight
of 1 and no bias the activation's input is v = (127 scale) w_scale, two f32 products that are
known exactly here.  What is left is the activation's own error and the last rounding:
  * 16-bit results: for |v| up to 5, |v| Phi(-|v|) is taken from a polynomial that is off by
    2^-18.84 (bf16) or 2^-20.77 (f16), evaluated within 2^-19.71 (the sum of its terms'
    magnitudes, each rounded to 2^-24 at most thirteen times, over its value), times an
    exponential within 2^-22, whose exponent of at most 18.1 is rounded to 2.5 * 2^-24 of
    itself (31.3 * 2^-24 of the exponential).  Their sum, where it is largest: 2^-17.48 and
    2^-17.97.  Past 5 5 R(5) stands for z R(z), which rises from 0.3847 there to 0.3990: 3.7%
    off at most.  exp(-v^2 / 2) below 2^-126 counts as 0.  The sum with max(0, v) is rounded to
    2^-24.
  * f32 results: the formula with its erf off by 2^-23: |v| 2^-21.
A result lies between the rounded ends of that interval (rounding is monotonic; 2^-23 more
of the value covers the reference's own way to 16 bits through f32).
"""

from __future__ import annotations

import math

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200.encoder_ops import ACT_GELU, ACT_NONE

pytestmark = pytest.mark.gpu


def interval(v, dtype):
    v = v.double()
    tail = 0.5 * torch.erfc(v.abs() / math.sqrt(2.0)) * v.abs()  # |v| Phi(-|v|)
    exact = v.clamp(min=0) - tail
    if dtype == torch.float32:
        off = v.abs() * 2.0 ** -21
    else:
        near = 2.0 ** -17.48 if dtype == torch.bfloat16 else 2.0 ** -17.97
        off = tail * torch.where(v.abs() <= 5, near, 0.037) + 5 * 2.0 ** -126 + exact.abs() * (2.0 ** -24 + 2.0 ** -23)
    return exact, (exact - off).to(dtype), (exact + off).to(dtype)


def check(y, v):
    exact, low, high = interval(v, y.dtype)
    bad = (y < low) | (y > high) | y.isnan()
    assert not bad.any(), (int(bad.sum()), v[bad][:4], y[bad][:4], exact[bad][:4])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,n", [(1, 1 << 20), (3, 300000), (700, 2000)])
def test_gelu_is_the_rounded_formula(cuda, dtype, m, n):
    """Inputs evenly over +-9 and over the exponents, through the few-token kernel (one and three
    rows) and the other."""
    x = torch.tensor([1.0, -1.0, 0.015625], device=cuda)[torch.arange(m, device=cuda) % 3]
    x = (x * (1 + torch.arange(m, device=cuda) % 128 / 128)).to(dtype)[:, None]
    ws = torch.cat([torch.linspace(0, 9, n - n // 4, device=cuda),
                    torch.logspace(-30, 1, n // 4, base=2.0, device=cuda)])
    weight = lf.Int8Weight(torch.ones(n, 1, dtype=torch.int8, device=cuda), ws)
    rows = lf.quantize_rows(x)
    assert (rows.q.abs() == 127).all()
    v = (rows.q.float() * rows.scale[:, None]) * ws
    assert torch.equal(lf.linear_int8(x, weight, act=ACT_NONE), v.to(dtype))
    check(lf.linear_int8(x, weight, act=ACT_GELU), v)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_gelu_of_every_16_bit_value(cuda, dtype):
    """Every finite value of the type, as the bias of a row of zeros; NaN stays NaN."""
    v = torch.arange(-(1 << 15), 1 << 15, device=cuda).to(torch.int16).view(dtype)
    weight = lf.Int8Weight(torch.ones(v.numel(), 1, dtype=torch.int8, device=cuda), torch.ones(v.numel(), device=cuda))
    y = lf.linear_int8(torch.zeros(1, 1, device=cuda, dtype=dtype), weight, v, act=ACT_GELU)[0]
    finite = v.isfinite()
    check(y[finite], v[finite].float())
    assert y[v.isnan()].isnan().all() and y[v == float("inf")].item() == float("inf")
