"""The cross attention's work list over the states of a packed batch: each sequence reads the
rows of its own text, wherever the packing by tenant put them."""

from __future__ import annotations

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200.packing import pack_rows
from test_gpu_cross_attention import check_sequence
from test_gpu_int8_encoder import encoder

LENGTHS, SLOTS = [5, 3, 8, 1, 4, 6], [2, 0, 1, 0, 2, 1]


def tokens(lengths):
    ids = torch.zeros(len(lengths), max(lengths), dtype=torch.long)
    for row, n in enumerate(lengths):
        ids[row, :n] = 100 * (row + 1) + torch.arange(n)
    return ids


def test_records_name_the_rows_of_their_text():
    ids = tokens(LENGTHS)
    pb = pack_rows(ids, LENGTHS, SLOTS, None, None, torch.device("cpu"))
    assert pb.order != sorted(pb.order)
    b = lf.cross_batch([2, 1, 130, 0, 7, 3], pb, "cpu")
    q0 = {0: 0, 2: 1, 3: 2, 133: 4, 140: 5}  # first query row -> text
    for start, _, k0, n, *_ in b.items.tolist():
        text = q0[start]
        assert pb.ids[k0:k0 + n].tolist() == ids[text, :LENGTHS[text]].tolist()
    assert {r[0] for r in b.items.tolist()} == set(q0) and b.n_kv == sum(LENGTHS) and b.max_kv == 8


def test_refusals():
    pb = pack_rows(tokens(LENGTHS), LENGTHS, SLOTS, None, None, torch.device("cpu"))
    with pytest.raises(ValueError, match="kv_starts"):
        lf.cross_batch([1] * 6, pb, "cpu", kv_starts=[0] * 6)
    with pytest.raises(ValueError, match="one query and one key length"):
        lf.cross_batch([1] * 5, pb, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("steps", [1, 60, 140])
def test_queries_read_their_own_text(cuda, steps):
    """Texts of several tenants, queries in the texts' own order, as the states are used."""
    model, store, ids = encoder(cuda)
    lengths = [40, 7, 256, 1, 129]
    text = torch.randint(5, 512, (5, 256), generator=torch.Generator().manual_seed(2))
    slots = store.slots([ids[i] for i in (2, 0, 1, 0, 2)])
    with torch.no_grad():
        packed = model.pack(text, lengths, slots)
        states = model.encode_packed(packed, store)
    assert packed.order != sorted(packed.order)
    q = torch.randn(5 * steps, 256, device=cuda, generator=torch.Generator(device=cuda).manual_seed(3)).bfloat16()
    out = lf.cross_attention_varlen(q, states, states, lf.cross_batch([steps] * 5, packed, cuda), 4)
    for i, n in enumerate(lengths):
        first = int(packed.first_token[i])
        rows, mine = slice(i * steps, (i + 1) * steps), states[first:first + n]
        check_sequence(out[rows], q[rows], mine, mine, 4, 4, 0.125)
        assert packed.ids[first:first + n].tolist() == text[i, :n].tolist()
