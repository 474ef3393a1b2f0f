"""The cross attention's work list is checked before the native call reads it as records."""

from __future__ import annotations

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200 import _native as nat


@pytest.mark.parametrize("spoil", [lambda i: i[:, :4].contiguous(), lambda i: i.long(), lambda i: i.flatten(),
                                   lambda i: i.t().contiguous().t(), lambda i: i[::2], lambda i: i.float(),
                                   lambda i: torch.cat([i, i], 1)[:, :8]])
def test_other_layouts_are_refused(monkeypatch, spoil):
    monkeypatch.setattr(nat, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(nat, "call", lambda *a: pytest.fail("the native call was made"))
    q = torch.zeros(8, 64, dtype=torch.bfloat16)
    batch = lf.cross_batch([2] * 4, [2] * 4, "cpu")
    batch.items = spoil(batch.items)
    with pytest.raises(ValueError, match="items"):
        lf.cross_attention_varlen(q, q, q, batch, 1)
