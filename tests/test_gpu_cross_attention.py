"""Cross attention of packed sequences against its formula in 64 bits.

Both kernels (few query rows: split over the keys; many: tcgen05 tiles) hold statistics
and sums in f32 and round the probabilities to the 16-bit type before the second
product.  With u half a step of that type (``eps / 2``), d the head's width, n the keys:
  * a score is a sum of d exact products in f32, at most (d + 8) 2^-24 sum |q k| off, then
    scaled and shifted (2^-23 of its size); 2^x adds 2^-21: together delta, relative, on p;
  * each p is rounded to the type: u (f16: or 2^-25 of the row's largest, below 2^-14);
  * the second product is an f32 sum of n terms: (n + 16) 2^-23;
  * the result is rounded once: u.
So |out - exact| <= A (u + 2 delta + (n + 16) 2^-23) + 2^-25 B + u |exact|, A the
probability-weighted mean of |v| and B the sum of |v| (over the largest p, which is 1).
"""

from __future__ import annotations

import pytest
import torch

from latefuse_b200 import cross_attention_varlen, cross_batch
from latefuse_b200 import _native as nat

pytestmark = pytest.mark.gpu


def check_sequence(out, q, k, v, heads, kv_heads, scale):
    """One sequence's rows of out against the formula, within the bound above."""
    nq, nk = q.shape[0], k.shape[0]
    d = q.shape[1] // heads
    if nq == 0:
        return
    if nk == 0:
        assert (out == 0).all()
        return
    u = torch.finfo(q.dtype).eps / 2
    q, k, v = (t.double().reshape(t.shape[0], -1, d) for t in (q, k, v))
    out = out.double().reshape(nq, heads, d)
    for h in range(heads):
        g = h // (heads // kv_heads)
        s = q[:, h] @ k[:, g].t() * scale
        size = q[:, h].abs() @ k[:, g].abs().t() * scale
        delta = ((d + 8) * 2.0 ** -24 * size + 2.0 ** -23 * s.abs()).amax(1, keepdim=True) + 2.0 ** -21
        p = (s - s.amax(1, keepdim=True)).exp()
        total = p.sum(1, keepdim=True)
        exact, mean = p @ v[:, g] / total, p @ v[:, g].abs() / total
        tol = mean * (u + 2 * delta + (nk + 16) * 2.0 ** -23) + u * exact.abs() + \
            2.0 ** -25 * v[:, g].abs().sum(0, keepdim=True) / total
        err = (out[:, h] - exact).abs()
        assert (err <= tol).all(), (h, (err / tol).max().item())


def run(cuda, q_lengths, kv_lengths, heads, kv_heads, d, dtype, seed=1, gap=0, growth=0.0, scale=None):
    """Sequences `gap` rows apart; rows outside them hold NaN (q, k, v) and 7 (out)."""
    g = torch.Generator(device=cuda).manual_seed(seed)
    qs = [sum(q_lengths[:i]) + gap * (i + 1) for i in range(len(q_lengths))]
    ks = [sum(kv_lengths[:i]) + gap * (i + 1) for i in range(len(kv_lengths))]
    tq, tk = sum(q_lengths) + gap * (len(q_lengths) + 1), sum(kv_lengths) + gap * (len(kv_lengths) + 1)
    q = torch.full((tq, heads * d + (8 if gap else 0)), float("nan"), device=cuda, dtype=dtype)
    kv = torch.full((tk, 2 * kv_heads * d + (16 if gap else 0)), float("nan"), device=cuda, dtype=dtype)
    for s, n in zip(qs, q_lengths):
        q[s:s + n, :heads * d] = torch.randn(n, heads * d, device=cuda, generator=g).to(dtype)
    for s, n in zip(ks, kv_lengths):
        rows = torch.randn(n, 2 * kv_heads * d, device=cuda, generator=g)
        if growth:  # later keys score higher: the running max moves
            rows[:, :kv_heads * d] *= (1 + growth * torch.arange(n, device=cuda) / 128).unsqueeze(1)
        kv[s:s + n, :2 * kv_heads * d] = rows.to(dtype)
    q, k, v = q[:, :heads * d], kv[:, :kv_heads * d], kv[:, kv_heads * d:2 * kv_heads * d]
    out = torch.full((tq, heads * d + (24 if gap else 0)), 7.0, device=cuda, dtype=dtype)
    view = out[:, :heads * d]
    batch = cross_batch(q_lengths, kv_lengths, cuda, q_starts=qs, kv_starts=ks)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    assert cross_attention_varlen(q, k, v, batch, heads, kv_heads, scale=scale, out=view, status=status) is view
    torch.cuda.synchronize()
    assert status.item() == 0
    scale = d ** -0.5 if scale is None else scale
    outside = torch.ones(tq, dtype=torch.bool, device=cuda)
    for s, n, t, m in zip(qs, q_lengths, ks, kv_lengths):
        check_sequence(view[s:s + n], q[s:s + n], k[t:t + m], v[t:t + m], heads, kv_heads, scale)
        outside[s:s + n] = False
    assert (out[outside] == 7).all() and (out[:, heads * d:] == 7).all()
    return q, k, v, batch, view


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (2, 1, 128), (16, 2, 64), (3, 3, 80), (2, 2, 8), (4, 2, 40),
                                              (5, 1, 104), (8, 8, 128), (1, 1, 72), (1, 1, 16)])
def test_single_tokens(cuda, dtype, heads, kv_heads, d):
    lengths = [1, 15, 16, 17, 63, 64, 65, 0, 77, 300, 513]
    run(cuda, [1] * len(lengths), lengths, heads, kv_heads, d, dtype, gap=3)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (2, 1, 128), (6, 2, 64), (3, 3, 80), (2, 2, 8), (2, 2, 48),
                                              (4, 2, 40), (2, 1, 104), (2, 2, 112), (1, 1, 72), (1, 1, 24)])
def test_prompts(cuda, dtype, heads, kv_heads, d):
    q = [1, 33, 128, 129, 200, 7, 0, 256, 31, 97, 64]
    kv = [5, 128, 64, 65, 300, 0, 9, 513, 1, 16, 127]
    run(cuda, q, kv, heads, kv_heads, d, dtype, gap=5)


@pytest.mark.parametrize("heads,kv_heads,d", [(4, 4, 64), (4, 2, 128), (2, 2, 80)])
@pytest.mark.parametrize("q", [[1, 1, 1], [3, 1, 5], [9, 16, 2], [17, 32, 8], [100, 128, 1], [40, 3, 150]])
def test_long_keys_and_a_moving_max(cuda, heads, kv_heads, d, q):
    """Up to 8,192 keys: every split of the few-row kernel, many tiles of the other, with
    scores that grow along the keys."""
    run(cuda, q, [8192, 1000, 4097], heads, kv_heads, d, torch.bfloat16, growth=1.0)
    run(cuda, q, [2048, 2047, 130], heads, kv_heads, d, torch.float16, gap=1)


@pytest.mark.parametrize("heads,d", [(16, 64), (8, 128)])
@pytest.mark.parametrize("seqs", [1, 5, 8, 12, 20])
def test_single_tokens_of_many_sequences(cuda, seqs, heads, d):
    """As many sequences and heads as it takes for the keys to be split in eight, four, two or
    not at all (few against many CTAs), of ragged lengths around 900."""
    kv = [900 - 37 * (i % 7) for i in range(seqs)]
    run(cuda, [1] * seqs, kv, heads, heads // 2, d, torch.bfloat16)
    run(cuda, [2, 1] * (seqs // 2) + [1] * (seqs % 2), kv, heads, heads, d, torch.float16, growth=1.0)


def test_many_units(cuda):
    """More units than SMs: every CTA walks several, with other group's tiles in between."""
    gen = torch.Generator().manual_seed(3)
    q = torch.randint(1, 300, (40,), generator=gen).tolist()
    kv = torch.randint(0, 700, (40,), generator=gen).tolist()
    run(cuda, q, kv, 16, 16, 64, torch.bfloat16)
    run(cuda, q, kv, 8, 4, 128, torch.float16)
    run(cuda, [1] * 40, kv, 16, 16, 64, torch.bfloat16)


def test_scale_and_one_hot_scores(cuda):
    """A large scale leaves one key per row; a small one the mean of the values."""
    run(cuda, [1, 4], [100, 50], 2, 2, 64, torch.bfloat16, scale=3.0)
    run(cuda, [140, 60], [100, 50], 2, 2, 64, torch.bfloat16, scale=3.0)
    run(cuda, [140, 1], [100, 500], 2, 1, 128, torch.float16, scale=1e-6)


@pytest.mark.parametrize("q_len", [1, 70, 150])
def test_no_keys_at_all(cuda, q_len):
    q = torch.randn(2 * q_len, 128, device=cuda, dtype=torch.bfloat16)
    k = torch.empty(0, 128, device=cuda, dtype=torch.bfloat16)
    out = cross_attention_varlen(q, k, k, cross_batch([q_len] * 2, [0, 0], cuda), 2)
    assert out.shape == q.shape and (out == 0).all()
    none = cross_attention_varlen(q[:0], k, k, cross_batch([], [], cuda), 2)
    assert none.shape == (0, 128)


@pytest.mark.parametrize("q_len", [2, 90, 150])
def test_infinities_stay_in_their_sequence_and_scores(cuda, q_len):
    """A key of -inf scores (its probability is 0) changes nothing but its own weight; a NaN
    value makes its sequence NaN and no other."""
    q = torch.randn(3 * q_len, 64, device=cuda, dtype=torch.bfloat16).abs()
    k, v = torch.randn(60, 64, device=cuda, dtype=torch.bfloat16), torch.randn(60, 64, device=cuda, dtype=torch.bfloat16)
    batch = cross_batch([q_len] * 3, [20, 20, 20], cuda)
    want = cross_attention_varlen(q, k, v, batch, 1)
    k2 = k.clone()
    k2[20:24] = float("-inf")  # the first keys of sequence 1
    got = cross_attention_varlen(q, k2, v, batch, 1)
    check_sequence(got[q_len:2 * q_len], q[q_len:2 * q_len], k[24:40], v[24:40], 1, 1, 0.125)
    assert torch.equal(got[:q_len], want[:q_len]) and torch.equal(got[2 * q_len:], want[2 * q_len:])
    v2 = v.clone()
    v2[30] = float("nan")
    got = cross_attention_varlen(q, k, v2, batch, 1)
    assert got[q_len:2 * q_len].isnan().all()
    assert torch.equal(got[:q_len], want[:q_len]) and torch.equal(got[2 * q_len:], want[2 * q_len:])


@pytest.mark.parametrize("q_len", [1, 50, 140])
def test_shared_states(cuda, q_len):
    """Beams: sequences whose key ranges coincide or overlap read the same states."""
    q = torch.randn(4 * q_len, 256, device=cuda, dtype=torch.float16)
    k, v = (torch.randn(200, 256, device=cuda, dtype=torch.float16) for _ in range(2))
    starts, lengths = [0, 0, 50, 120], [100, 100, 150, 80]
    batch = cross_batch([q_len] * 4, lengths, cuda, kv_starts=starts)
    out = cross_attention_varlen(q, k, v, batch, 4)
    for i, (s, n) in enumerate(zip(starts, lengths)):
        check_sequence(out[i * q_len:(i + 1) * q_len], q[i * q_len:(i + 1) * q_len], k[s:s + n], v[s:s + n], 4, 4, 0.125)


def test_far_rows(cuda):
    """Rows whose element offset passes 2^31."""
    rows = (1 << 31) // 4096 + 3000
    kv = torch.zeros(rows, 4096, device=cuda, dtype=torch.bfloat16)
    tail = torch.randn(2100, 256, device=cuda, dtype=torch.bfloat16)
    kv[rows - 2100:, 3840:] = tail
    k, v = kv[:, 3840:3968], kv[:, 3968:]
    for q_len in (1, 100, 140):
        q = torch.randn(2 * q_len, 128, device=cuda, dtype=torch.bfloat16)
        batch = cross_batch([q_len] * 2, [2100, 70], cuda, kv_starts=[rows - 2100, rows - 70])
        out = cross_attention_varlen(q, k, v, batch, 2)
        check_sequence(out[:q_len], q[:q_len], tail[:, :128], tail[:, 128:], 2, 2, 0.125)
        check_sequence(out[q_len:], q[q_len:], tail[-70:, :128], tail[-70:, 128:], 2, 2, 0.125)
    del kv, k, v


@pytest.mark.parametrize("q_len", [1, 100, 140])
def test_capture_replay_and_streams(cuda, q_len):
    kv = torch.randn(1500, 512, device=cuda, dtype=torch.bfloat16)
    k, v = kv[:, :256], kv[:, 256:]
    batch = cross_batch([q_len] * 3, [1000, 100, 400], cuda)
    qs = [torch.randn(3 * q_len, 256, device=cuda, dtype=torch.bfloat16) for _ in range(4)]
    want = [cross_attention_varlen(q, k, v, batch, 4) for q in qs]
    static = qs[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cross_attention_varlen(static, k, v, batch, 4)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cross_attention_varlen(static, k, v, batch, 4)
    for q, w in zip(qs, want):
        static.copy_(q)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, q in zip(streams, qs):
            with torch.cuda.stream(s):
                got.append(cross_attention_varlen(q, k, v, batch, 4))
    torch.cuda.synchronize()
    for n, o in enumerate(got):
        assert torch.equal(o, want[n % 4])


@pytest.mark.parametrize("q_len", [2, 80, 140])
def test_records_outside_the_tensors_store_nothing(cuda, q_len):
    """Records past the queries or the keys, with a negative start or a tile past their
    queries, are reported and write no row; the others are as without them."""
    q = torch.randn(2 * q_len, 128, device=cuda, dtype=torch.bfloat16)
    k, v = (torch.randn(300, 128, device=cuda, dtype=torch.bfloat16) for _ in range(2))
    batch = cross_batch([q_len] * 2, [200, 100], cuda)
    want = cross_attention_varlen(q, k, v, batch, 2)
    tq = 2 * q_len
    bad = torch.tensor([[tq - 1, q_len, 0, 50, 0, 0, 0, 0], [0, q_len, 290, 20, 0, 0, 0, 0], [-1, q_len, 0, 9, 0, 0, 0, 0],
                        [0, q_len, -2, 9, 0, 0, 0, 0], [0, q_len, 0, 9, 3, 0, 0, 0], [0, -4, 0, 9, 0, 0, 0, 0],
                        [0, q_len, 0, -9, 0, 0, 0, 0], [2**31 - 1, q_len, 2**31 - 1, 9, 0, 0, 0, 0]],
                       dtype=torch.int32, device=cuda)
    big = torch.full((tq + 200, 128), 7.0, device=cuda, dtype=torch.bfloat16)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    batch.items = bad
    cross_attention_varlen(q, k, v, batch, 2, out=big[:tq], status=status)
    assert status.item() == nat.LF_STATUS_BAD_SEGMENT and (big == 7).all()
    batch.items = torch.cat([bad, cross_batch([q_len] * 2, [200, 100], cuda).items, bad])
    cross_attention_varlen(q, k, v, batch, 2, out=big[:tq], status=status)
    check_sequence(big[:q_len], q[:q_len], k[:200], v[:200], 2, 2, 0.125)
    check_sequence(big[q_len:tq], q[q_len:], k[200:], v[200:], 2, 2, 0.125)
    assert (big[tq:] == 7).all() and want.shape == q.shape


def test_refusals(cuda):
    q = torch.randn(4, 128, device=cuda, dtype=torch.bfloat16)
    batch = cross_batch([2, 2], [2, 2], cuda)
    with pytest.raises(ValueError, match="heads"):
        cross_attention_varlen(q, q, q, batch, 3)
    with pytest.raises(ValueError, match="k and v"):
        cross_attention_varlen(q, q[:, :64], q[:, :64], batch, 2)
    with pytest.raises(ValueError, match="key rows"):
        cross_attention_varlen(q, q[:3], q[:3], batch, 2)
    with pytest.raises(ValueError, match="key rows"):
        cross_attention_varlen(q[:3], q, q, batch, 2)
    with pytest.raises(ValueError, match="out must"):
        cross_attention_varlen(q, q, q, batch, 2, out=torch.empty(4, 128, device=cuda))
    with pytest.raises(ValueError, match="contiguous"):
        cross_attention_varlen(q, q[:, :64].t().contiguous().t()[:, :64].repeat(1, 1), q[:, ::2], batch, 2, 1)
    with pytest.raises(nat.NativeLibraryError, match="head_dim"):
        cross_attention_varlen(q[:, :60], q[:, :60], q[:, :60], batch, 5)
    with pytest.raises(nat.NativeLibraryError, match="head_dim"):
        big = torch.randn(4, 136, device=cuda, dtype=torch.bfloat16)
        cross_attention_varlen(big, big, big, batch, 1)
    with pytest.raises(nat.NativeLibraryError, match="bf16 or f16"):
        cross_attention_varlen(q.float(), q.float(), q.float(), batch, 2)
    with pytest.raises(nat.NativeLibraryError, match="scale"):
        cross_attention_varlen(q, q, q, batch, 2, scale=-1.0)
    with pytest.raises(nat.NativeLibraryError, match="aligned"):
        odd = torch.randn(4, 130, device=cuda, dtype=torch.bfloat16)[:, 1:129]
        cross_attention_varlen(odd, q, q, batch, 2)
    with pytest.raises(nat.NativeLibraryError, match="CUDA tensors"):
        cross_attention_varlen(q.cpu(), q, q, batch, 2)


def test_outputs_over_their_inputs_are_refused(cuda):
    fused = torch.randn(6, 512, device=cuda, dtype=torch.bfloat16)
    q, k, v, free = fused.split(128, dim=1)
    batch = cross_batch([2, 4], [3, 3], cuda)
    for taken in (q, k, v, fused[:, 64:192]):
        with pytest.raises(ValueError, match="overlap"):
            cross_attention_varlen(q, k, v, batch, 2, out=taken)
    want = cross_attention_varlen(q, k, v, batch, 2)
    assert torch.equal(cross_attention_varlen(q, k, v, batch, 2, out=free), want)
