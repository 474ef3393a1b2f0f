"""An output over any of the projection's inputs is refused: other tiles still read them when
the first are written."""

from __future__ import annotations

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200 import _native as nat

M, N, K = 6, 32, 64


@pytest.fixture
def memory(monkeypatch):
    monkeypatch.setattr(nat, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(nat, "call", lambda *a: None)
    return torch.zeros(1 << 15, dtype=torch.uint8)


def test_every_input(memory):
    """Inputs 4 KB apart; an output whose last byte is an input's first, whose first is its last, and
    one between them."""
    at = lambda i, n, dtype: memory[4096 * i:4096 * i + n].view(dtype)
    bf = torch.bfloat16
    q = at(1, N * K, torch.int8).view(N, K)
    weight = lf.Int8Weight(q, at(2, 4 * N, torch.float32))
    assert weight.q.data_ptr() == q.data_ptr()
    x, bias = at(3, 2 * M * K, bf).view(M, K), at(4, 2 * N, bf)
    rows = lf.Int8Rows(at(5, M * K, torch.int8).view(M, K), at(6, 4 * M, torch.float32), (M, K), bf)
    size = 2 * M * N
    out = lambda first: memory[first:first + size].view(bf).view(M, N)
    lf.linear_int8(x, weight, bias, out=out(7 * 4096))
    lf.linear_int8(rows, weight, bias, out=out(7 * 4096))
    for given, used in ((x, {1: N * K, 2: 4 * N, 3: 2 * M * K, 4: 2 * N}), (rows, {1: N * K, 2: 4 * N, 4: 2 * N, 5: M * K, 6: 4 * M})):
        for i, n in used.items():
            for first in (4096 * i - size + 2, 4096 * i, 4096 * i + n - 2):
                with pytest.raises(ValueError, match="overlap"):
                    lf.linear_int8(given, weight, bias, out=out(first))
            if i < 4:
                lf.linear_int8(given, weight, bias, out=out(4096 * i - size))
    lf.linear_int8(rows, weight, out=out(4 * 4096))  # a bias that is not given
    lf.linear_int8(x, weight, bias.float(), out=out(4 * 4096))  # or that is read from a copy
