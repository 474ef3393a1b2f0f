"""Cross attention: records that promise less than they hold, for both kernels (the tolerances
are those of the comparison with the formula, derived beside it)."""

from __future__ import annotations

import pytest
import torch

from latefuse_b200 import cross_attention_varlen, cross_batch
from latefuse_b200 import _native as nat
from test_gpu_cross_attention import check_sequence

pytestmark = pytest.mark.gpu


# few rows; many rows of short texts; more than a tile of rows
@pytest.mark.parametrize("seqs,q_len,kv_len,heads", [(3, 1, 200, 2), (3, 20, 200, 2), (200, 33, 100, 16), (3, 127, 200, 16),
                                                     (64, 128, 100, 16), (3, 140, 200, 2), (3, 300, 200, 2)])
def test_a_record_past_max_q_stores_nothing(cuda, seqs, q_len, kv_len, heads):
    """One sequence holds a query more than max_q says: it is reported and its rows stay as they
    were, whichever kernel runs; the other sequences are as ever."""
    lengths = [q_len] * seqs
    lengths[1] += 1
    g = torch.Generator(device=cuda).manual_seed(seqs + q_len)
    q = torch.randn(sum(lengths), heads * 64, device=cuda, generator=g).bfloat16()
    kv = torch.randn(seqs * kv_len, 2 * heads * 64, device=cuda, generator=g).bfloat16()
    k, v = kv[:, :heads * 64], kv[:, heads * 64:]
    batch = cross_batch(lengths, [kv_len] * seqs, cuda)
    batch.max_q = q_len
    out = torch.full_like(q, 7.0)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    cross_attention_varlen(q, k, v, batch, heads, out=out, status=status)
    assert status.item() == nat.LF_STATUS_BAD_SEGMENT
    assert (out[q_len:2 * q_len + 1] == 7).all()
    for s in (0, 2, seqs - 1):
        q0 = s * q_len + (s > 1)
        rows, keys = slice(q0, q0 + q_len), slice(s * kv_len, (s + 1) * kv_len)
        check_sequence(out[rows], q[rows], k[keys], v[keys], heads, heads, 0.125)


@pytest.mark.parametrize("d", [64, 80])
@pytest.mark.parametrize("seqs,q_len,kv_len,heads", [(3, 1, 200, 2), (3, 20, 2000, 2), (64, 128, 100, 16), (3, 140, 300, 2)])
def test_scores_that_are_all_minus_infinity_give_zeros(cuda, seqs, q_len, kv_len, heads, d):
    g = torch.Generator(device=cuda).manual_seed(seqs + d)
    q = torch.randn(seqs * q_len, heads * d, device=cuda, generator=g).abs().add(0.5).bfloat16()
    k, v = torch.randn(2, seqs * kv_len, heads * d, device=cuda, generator=g).bfloat16()
    k[kv_len:2 * kv_len] = float("-inf")
    out = cross_attention_varlen(q, k, v, cross_batch([q_len] * seqs, [kv_len] * seqs, cuda), heads)
    assert (out[q_len:2 * q_len] == 0).all()
    for s in (0, seqs - 1):
        rows, keys = slice(s * q_len, (s + 1) * q_len), slice(s * kv_len, (s + 1) * kv_len)
        check_sequence(out[rows], q[rows], k[keys], v[keys], heads, heads, d ** -0.5)
