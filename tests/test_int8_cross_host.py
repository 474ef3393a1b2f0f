"""The 8-bit and cross-attention entries on the host: refusals of the C ABI before any
device work, of the Python functions, and the cross attention's work list."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

import latefuse_b200 as lf
from latefuse_b200 import _native as nat, encoder_ops, int8_ops
from latefuse_b200._build import build

INVALID, UNSUPPORTED, WORKSPACE = 1, 2, 4


@pytest.fixture(scope="module")
def lib():
    build()
    return nat.lib()


@pytest.fixture(scope="module")
def addr():
    buf = ctypes.create_string_buffer(1 << 12)
    base = (ctypes.addressof(buf) + 255) // 256 * 256
    yield base
    del buf


def refused(lib, rc, code, text):
    assert rc == code and text.encode() in lib.lf_last_error(), (rc, lib.lf_last_error())


def test_quantize_rows_refusals(lib, addr):
    q = lambda dtype=1, x=addr, ldx=64, rows=4, cols=64, out=addr, ldq=64, scale=addr: \
        lib.lf_quantize_rows(None, dtype, x, ldx, rows, cols, out, ldq, scale)
    refused(lib, q(dtype=9), INVALID, "dtype")
    refused(lib, q(cols=0), INVALID, "rows")
    refused(lib, q(rows=-1), INVALID, "rows")
    refused(lib, q(x=None), INVALID, "null")
    refused(lib, q(scale=None), INVALID, "null")
    refused(lib, q(ldx=63), INVALID, "stride")
    refused(lib, q(ldq=63), INVALID, "stride")
    assert q(rows=0, x=None) == 0


def test_linear_int8_refusals(lib, addr):
    def f(dtype=1, x=addr, ldx=64, xs=addr, w=addr, ldw=64, ws=addr, bias=None, y=addr, ldy=32, m=4, n=32, k=64, act=0):
        return lib.lf_linear_int8(None, dtype, x, ldx, xs, w, ldw, ws, bias, y, ldy, m, n, k, act, None)
    refused(lib, f(dtype=3), INVALID, "dtype")
    refused(lib, f(act=2), INVALID, "act")
    refused(lib, f(n=0), INVALID, "n 0")
    refused(lib, f(m=-1), INVALID, "m -1")
    refused(lib, f(k=131073, ldx=131088, ldw=131088), UNSUPPORTED, "32 bits")
    refused(lib, f(x=None), INVALID, "null")
    refused(lib, f(ws=None), INVALID, "null")
    refused(lib, f(ldx=48), INVALID, "stride")
    refused(lib, f(ldy=31), INVALID, "stride")
    refused(lib, f(x=addr + 8), INVALID, "16-byte")
    refused(lib, f(ldw=72), INVALID, "16-byte")
    assert f(m=0, x=None) == 0


def test_workspace_entries(lib, addr):
    need = lib.lf_linear_rows_int8_workspace_bytes(17, 100)
    assert need == 2048 + 256  # 17 rows of 112 bytes, 17 scales, each to 256 bytes
    assert lib.lf_linear_rows_int8_workspace_bytes(4, 131073) == 0
    assert lib.lf_linear_rows_int8_workspace_bytes(4, 4096) == 0  # one launch, no workspace
    for m in (0, 1, 4, 5, 16, 17, 100, 70001):
        for k in (1, 16, 100, 1024, 1025, 4096, 4097, 131072):
            assert int8_ops._rows_bytes(m, k) == lib.lf_linear_rows_int8_workspace_bytes(m, k)
            for code, size in ((0, 4), (1, 2), (2, 2)):
                assert int8_ops._ffn_bytes(size, m, 264, k) == lib.lf_ffn_int8_workspace_bytes(code, m, 264, k)
    g = lambda ws, size, dtype=1, k=100: lib.lf_linear_rows_int8(None, dtype, addr, 100, addr, 112, addr, None, addr, 32, 17, 32,
                                                                 k, 0, ws, size, None)
    one = lambda dtype=1, x=addr, ldx=100, w=addr, ldw=112, scale=addr, act=0, n=32: lib.lf_linear_rows_int8(
        None, dtype, x, ldx, w, ldw, scale, None, addr, 32, 4, n, 100, act, None, 0, None)
    refused(lib, one(dtype=7), INVALID, "dtype")
    refused(lib, one(x=None), INVALID, "null")
    refused(lib, one(scale=None), INVALID, "null")
    refused(lib, one(ldx=99), INVALID, "stride")
    refused(lib, one(w=addr + 8), INVALID, "16-byte")
    refused(lib, one(act=9), INVALID, "act")
    refused(lib, one(n=0), INVALID, "n 0")
    refused(lib, g(addr, need - 1), WORKSPACE, "workspace")
    refused(lib, g(None, need), WORKSPACE, "workspace")
    refused(lib, g(addr + 16, need), WORKSPACE, "aligned")
    refused(lib, g(addr, need, dtype=7), INVALID, "dtype")
    assert lib.lf_ffn_int8_workspace_bytes(1, 3, 64, 100) == 256 + 256 + 512 + 256 + 768
    assert lib.lf_ffn_int8_workspace_bytes(1, 3, 0, 100) == 0
    h = lambda size, hidden=64, m=3: lib.lf_ffn_int8(
        None, 1, addr, 64, None, 0, addr, addr, 1e-5, addr, 64, addr, None, addr, 112, addr, None, m, hidden, 100, 1,
        addr, 64, addr, 64, addr, size, None)
    refused(lib, h(100), WORKSPACE, "workspace")
    refused(lib, h(1 << 20, hidden=-1), INVALID, "hidden")
    refused(lib, h(1 << 20, hidden=60), INVALID, "multiple of 8")
    assert h(0, m=0) == 0


def test_add_layernorm_int8_refusals(lib, addr):
    f = lambda hidden=64, q=addr, ldq=64, scale=addr: lib.lf_add_layernorm_int8(
        None, 1, addr, 64, None, 0, addr, addr, 1e-5, 3, hidden, addr, 64, q, ldq, scale)
    refused(lib, f(q=None), INVALID, "null q")
    refused(lib, f(scale=None), INVALID, "null q")
    refused(lib, f(ldq=56), INVALID, "8-byte")
    refused(lib, f(ldq=68), INVALID, "8-byte")
    refused(lib, f(q=addr + 4), INVALID, "8-byte")
    refused(lib, f(hidden=60), INVALID, "multiple of 8")


def test_cross_attention_refusals(lib, addr):
    def f(dtype=1, q=addr, ldq=128, n_q=4, k=addr, ldk=128, v=addr, ldv=128, n_kv=9, heads=2, kv_heads=2, d=64, items=addr,
          n_items=1, max_q=4, max_kv=9, scale=0.1, out=addr, ldo=128):
        return lib.lf_cross_attention_varlen(None, dtype, q, ldq, n_q, k, ldk, v, ldv, n_kv, heads, kv_heads, d, items, n_items,
                                             max_q, max_kv, scale, out, ldo, None)
    refused(lib, f(dtype=0), UNSUPPORTED, "bf16 or f16")
    for d in (0, 4, 60, 136):
        refused(lib, f(d=d), UNSUPPORTED, "head_dim")
    refused(lib, f(heads=3), INVALID, "heads")
    refused(lib, f(kv_heads=0), INVALID, "heads")
    refused(lib, f(n_kv=-1), INVALID, "sizes")
    for scale in (0.0, -1.0, float("nan"), float("inf")):
        refused(lib, f(scale=scale), INVALID, "scale")
    refused(lib, f(k=None), INVALID, "null")
    refused(lib, f(items=None), INVALID, "null")
    refused(lib, f(ldq=120), INVALID, "stride")
    refused(lib, f(ldv=64), INVALID, "stride")
    refused(lib, f(ldk=132), INVALID, "16-byte")
    refused(lib, f(v=addr + 8), INVALID, "16-byte")
    assert f(n_items=0, items=None) == 0 and f(n_q=0, q=None) == 0 and f(max_q=0) == 0


def test_cross_batch_records():
    b = lf.cross_batch([3, 0, 300, 128], [5, 7, 0, 900], "cpu")
    assert (b.n_seqs, b.n_q, b.n_kv, b.max_q, b.max_kv) == (4, 431, 912, 300, 900)
    want = [[303, 128, 12, 900, 0], [0, 3, 0, 5, 0]] + [[3, 300, 12, 0, t] for t in range(3)]
    assert b.items.dtype == torch.int32 and b.items[:, :5].tolist() == want and (b.items[:, 5:] == 0).all()
    b = lf.cross_batch([2, 2], [10, 10], "cpu", q_starts=[5, 1], kv_starts=[0, 0])
    assert (b.n_q, b.n_kv) == (7, 10) and b.items[:, :4].tolist() == [[5, 2, 0, 10], [1, 2, 0, 10]]
    e = lf.cross_batch([], [], "cpu")
    assert e.items.shape == (0, 8) and e.n_q == e.max_kv == 0
    assert lf.cross_batch(np.array([1, 1]), torch.tensor([3, 4]), "cpu").n_kv == 7


def test_cross_batch_refusals():
    with pytest.raises(ValueError, match="one query and one key length"):
        lf.cross_batch([1, 2], [3], "cpu")
    with pytest.raises(ValueError, match="negative"):
        lf.cross_batch([1, -2], [3, 3], "cpu")
    with pytest.raises(ValueError, match="negative"):
        lf.cross_batch([1], [3], "cpu", kv_starts=[-1])
    with pytest.raises(ValueError, match="starts"):
        lf.cross_batch([1, 1], [3, 3], "cpu", q_starts=[0])
    with pytest.raises(ValueError, match="overlap"):
        lf.cross_batch([3, 2], [3, 3], "cpu", q_starts=[0, 2])
    with pytest.raises(ValueError, match="32 bits"):
        lf.cross_batch([1], [3], "cpu", kv_starts=[2**31 - 50])
    lf.cross_batch([3, 0, 2], [3, 3, 3], "cpu", q_starts=[0, 1, 3])  # an empty range overlaps nothing


def test_int8_weight_layout_and_refusals():
    q = torch.randint(-127, 128, (5, 37), dtype=torch.int8)
    w = lf.Int8Weight(q, torch.ones(5))
    assert w.shape == (5, 37) and w.ld == 48 and torch.equal(w.q, q) and w.q.data_ptr() % 16 == 0
    with pytest.raises(ValueError, match="int8"):
        lf.Int8Weight(q.float(), torch.ones(5))
    with pytest.raises(ValueError, match="int8"):
        lf.Int8Weight(q[0], torch.ones(5))
    with pytest.raises(ValueError, match="scale"):
        lf.Int8Weight(q, torch.ones(4))
    with pytest.raises(ValueError, match="scale"):
        lf.Int8Weight(q, torch.ones(5).double())
    with pytest.raises(ValueError, match="K must be"):
        lf.Int8Weight(torch.empty(2, 131073, dtype=torch.int8), torch.ones(2))
    with pytest.raises(nat.NativeLibraryError, match="CUDA tensors"):
        lf.quantize_rows(torch.ones(2, 3))
    with pytest.raises(nat.NativeLibraryError, match="CUDA tensors"):
        lf.linear_int8(torch.ones(2, 37), w)
    with pytest.raises(nat.NativeLibraryError, match="CUDA tensors"):
        lf.cross_attention_varlen(torch.ones(2, 64), torch.ones(2, 64), torch.ones(2, 64), lf.cross_batch([2], [2], "cpu"), 1)


def test_int8_rows_refusals():
    q, s = torch.zeros(6, 32, dtype=torch.int8), torch.zeros(6)
    rows = lf.Int8Rows(q, s, (2, 3, 32), torch.bfloat16)
    assert rows.ld == 32 and rows.dequantize().shape == (2, 3, 32)
    assert lf.Int8Rows(q[:1, :20], s[:1], (20,), torch.float16).ld == 32  # a single row's stride is its own, padded
    for bad in ((q.float(), s, (6, 32)), (q[0], s, (6, 32)), (q.t(), torch.zeros(32), (32, 6)), (q, s[:5], (6, 32)),
                (q, torch.zeros(12)[::2], (6, 32)), (q, s.double(), (6, 32)), (q, s, (5, 32)), (q, s, (6, 31)), (q, s, ())):
        with pytest.raises(ValueError):
            lf.Int8Rows(*bad, torch.bfloat16)


def test_shared_memory_is_found():
    """Every pair of column and row ranges of one buffer, against the sets of their elements;
    ranges of other row strides count as shared when they lie within each other."""
    buf = torch.arange(7 * 12, dtype=torch.int16).reshape(7, 12)
    views = [buf[a:b, c:d] for a, b in ((0, 7), (0, 3), (3, 7), (2, 3)) for c, d in ((0, 12), (0, 4), (4, 12), (3, 5), (2, 2))]
    for x in views:
        for y in views:
            shared = bool(set(x.flatten().tolist()) & set(y.flatten().tolist()))
            assert encoder_ops._share_memory(x, y) == shared, (x.shape, y.shape)
    flat = buf.flatten()
    assert encoder_ops._share_memory(flat[:20].view(2, 10), flat[10:34].view(3, 8))
    assert not encoder_ops._share_memory(flat[:20].view(2, 10), flat[20:44].view(3, 8))
    assert not encoder_ops._share_memory(buf, buf.clone())
