"""The 8-bit operators hand their status word to the native call, and the encoder's 8-bit FFN
the word that ``check_device_status`` reads (the native call replaced by a record of its
arguments: a timeout is not brought about)."""

from __future__ import annotations

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200 import _native as nat, engine
from test_quantized_ffn_host import model as quantized  # noqa: F401  (a fixture)


@pytest.fixture
def calls(monkeypatch):
    seen = []
    monkeypatch.setattr(nat, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(nat, "call", lambda fn, what, dev, *args: seen.append((what, args[-1])))
    return seen


def test_the_word_reaches_the_call(calls):
    status = torch.zeros(1, dtype=torch.int32)
    x, v = torch.zeros(3, 32, dtype=torch.bfloat16), torch.ones(32, dtype=torch.bfloat16)
    w = lf.Int8Weight(torch.zeros(32, 32, dtype=torch.int8), torch.ones(32))
    rows = lf.Int8Rows(torch.zeros(3, 32, dtype=torch.int8), torch.ones(3), (3, 32), torch.bfloat16)
    for given, word in ((status, status.data_ptr()), (None, None)):
        lf.linear_int8(x, w, status=given)
        lf.linear_int8(rows, w, status=given)
        lf.linear_int8(torch.zeros(100, 32), w, status=given)
        lf.ffn_int8(x, None, v, v, 1e-5, w, None, w, None, status=given)
        assert [what for what, _ in calls] == ["lf_linear_rows_int8", "lf_linear_int8", "lf_linear_rows_int8", "lf_ffn_int8"]
        assert all(got == word for _, got in calls)
        calls.clear()


@pytest.mark.parametrize("fused", [True, False])
def test_the_encoder_hands_its_own(quantized, monkeypatch, fused):  # noqa: F811
    words = []

    def ffn(a, *rest, status=None):
        words.append(status)
        return a, a

    def linear(x, *rest, status=None):
        words.append(status)
        return x

    monkeypatch.setattr(engine, "ffn_int8", ffn)
    monkeypatch.setattr(engine, "linear_int8", linear)
    monkeypatch.setattr(engine, "add_layernorm_int8", lambda a, *rest: (a, a))
    quantized._native_gelu = fused
    quantized.quantize_ffn()
    quantized._ffn(0, torch.zeros(3, 64), torch.zeros(3, 64))
    assert len(words) == (1 if fused else 2) and all(w is quantized._runner.status for w in words)
    assert words[0].dtype == torch.int32 and words[0].item() == 0
