"""Sizes past the native calls' 32-bit numbers are refused on the host, before any memory is
taken: tensors that stand for them are one element repeated."""

from __future__ import annotations

import ctypes

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200 import _native as nat
from latefuse_b200._build import build

INT32_MAX, UNSUPPORTED = 2**31 - 1, 2


def rows(*shape, dtype=torch.bfloat16):
    return torch.zeros(1, dtype=dtype).expand(*shape)


def test_quantize_rows_entry():
    build()
    lib = nat.lib()
    buf = ctypes.create_string_buffer(1 << 9)
    addr = (ctypes.addressof(buf) + 255) // 256 * 256
    for dtype in (0, 1, 2):
        for cols in (INT32_MAX - 4095, INT32_MAX - 2048, INT32_MAX - 255, INT32_MAX - 1, INT32_MAX):
            assert lib.lf_quantize_rows(None, dtype, addr, 1 << 32, 1, cols, addr, 1 << 32, addr) == UNSUPPORTED
            assert b"above" in lib.lf_last_error()
        assert lib.lf_quantize_rows(None, dtype, addr, 1 << 32, 0, INT32_MAX - 4096, addr, 1 << 32, addr) == 0


@pytest.mark.parametrize("cols", [INT32_MAX - 4095, 2**31, 2**32 + 64])
def test_quantize_rows(cols):
    with pytest.raises(ValueError, match="elements are needed"):
        lf.quantize_rows(rows(2, cols))
    with pytest.raises(ValueError, match="elements are needed"):
        lf.Int8Weight.from_float(rows(2, cols))


@pytest.mark.parametrize("n", [2**31 - 256, 2**32 + 8])
def test_weights(n):
    with pytest.raises(ValueError, match="N in"):
        lf.Int8Weight(rows(n, 1, dtype=torch.int8), rows(n, dtype=torch.float32))


def test_layernorm_rows_and_heads():
    wide = rows(2, 2**32 + 64)
    with pytest.raises(ValueError, match="elements"):
        lf.add_layernorm_int8(wide, None, wide[0], wide[0], 1e-5)
    batch = lf.cross_batch([2], [2], "cpu")
    for heads in (1, 2**26 + 1):  # of 64 columns
        with pytest.raises(ValueError, match="heads"):
            lf.cross_attention_varlen(wide, wide, wide, batch, heads)
