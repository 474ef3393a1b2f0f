"""Cross attention's choice of kernel and split goes by the keys of its records, not by the rows
of the key tensor: beams that share a text, and buffers with spare rows."""

from __future__ import annotations

import ctypes

import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200 import _native as nat, encoder_ops
from latefuse_b200._build import build
from test_gpu_cross_attention import check_sequence


def test_total_of_the_records():
    assert lf.cross_batch([3, 0, 300, 128], [5, 7, 0, 900], "cpu").total_kv == 905
    assert lf.cross_batch([1] * 64, [4096] * 64, "cpu", kv_starts=[0] * 64).total_kv == 64 * 4096
    assert lf.cross_batch([300, 1], [10, 7], "cpu").total_kv == 3 * 10 + 7  # three records of the first
    assert lf.cross_batch([], [], "cpu").total_kv == 0


def test_the_call_gets_the_total_and_not_the_tensor_rows(monkeypatch):
    calls = []
    monkeypatch.setattr(nat, "require_cuda", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(nat, "call", lambda fn, what, dev, *args: calls.append(args))
    q, k = torch.zeros(8, 64, dtype=torch.bfloat16), torch.zeros(5000, 64, dtype=torch.bfloat16)
    batch = lf.cross_batch([1] * 8, [100] * 8, "cpu", kv_starts=[0] * 8)
    encoder_ops.cross_attention_varlen(q, k, k, batch, 1)
    batch.total_kv = None
    encoder_ops.cross_attention_varlen(q, k, k, batch, 1)
    # ..., n_kv, n_heads, n_kv_heads, d, items, n_items, max_q, max_kv, total_kv, scale, out, ld_out, status
    assert [(c[-14 + 1], c[-6], c[-5]) for c in calls] == [(5000, 100, 800), (5000, 100, 100)]


def test_refusals():
    build()
    lib = nat.lib()
    buf = ctypes.create_string_buffer(1 << 12)
    addr = (ctypes.addressof(buf) + 255) // 256 * 256
    f = lambda total=9, scale=0.1: lib.lf_cross_attention_varlen_total(
        None, 1, addr, 128, 4, addr, 128, addr, 128, 9, 2, 2, 64, addr, 1, 4, 9, total, scale, addr, 128, None)
    for call, text in ((lambda: f(total=-1), b"sizes"), (lambda: f(scale=0.0), b"scale")):
        assert call() == 1 and text in lib.lf_last_error()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,d", [(16, 16, 64), (32, 8, 128), (4, 4, 80)])
@pytest.mark.parametrize("q_len,kv", [(1, [64] * 31 + [8192]), (1, [1000] * 8), (1, [300] * 64), (5, [2000, 40]), (40, [500] * 6)])
def test_spare_rows_change_no_bit(cuda, heads, kv_heads, d, q_len, kv):
    g = torch.Generator(device=cuda).manual_seed(heads + q_len)
    q = torch.randn(len(kv) * q_len, heads * d, device=cuda, generator=g).bfloat16()
    states = torch.full((1 << 17, 2 * kv_heads * d), float("nan"), device=cuda, dtype=torch.bfloat16)
    n = sum(kv)
    states[:n] = torch.randn(n, 2 * kv_heads * d, device=cuda, generator=g).bfloat16()
    k, v = states.split(kv_heads * d, dim=1)
    batch = lf.cross_batch([q_len] * len(kv), kv, cuda)
    want = lf.cross_attention_varlen(q, k[:n], v[:n], batch, heads, kv_heads)
    for rows in (n + 1, 3 * n, 1 << 17):
        assert torch.equal(lf.cross_attention_varlen(q, k[:rows], v[:rows], batch, heads, kv_heads), want)


@pytest.mark.gpu
@pytest.mark.parametrize("beams,q_len,keys,heads,kv_heads,d", [(64, 1, 4096, 16, 16, 64), (64, 16, 4096, 32, 8, 128),
                                                               (4, 1, 8192, 2, 2, 64), (200, 2, 130, 4, 2, 80)])
def test_beams_of_one_text(cuda, beams, q_len, keys, heads, kv_heads, d):
    g = torch.Generator(device=cuda).manual_seed(beams)
    q = torch.randn(beams * q_len, heads * d, device=cuda, generator=g).bfloat16()
    k, v = torch.randn(keys + 5, 2 * kv_heads * d, device=cuda, generator=g).bfloat16().split(kv_heads * d, dim=1)
    batch = lf.cross_batch([q_len] * beams, [keys] * beams, cuda, kv_starts=[3] * beams)
    out = lf.cross_attention_varlen(q, k, v, batch, heads, kv_heads)
    check_sequence(out, q, k[3:3 + keys], v[3:3 + keys], heads, kv_heads, d ** -0.5)
