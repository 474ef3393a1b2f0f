"""The 8-bit projections against their formulas in 64 bits.

Quantisation is decided exactly, so its integers and scales are compared for equality.
The projection's integer sum is exact; what is left is f32: the sum becomes f32 (2^-24),
times the token's scale (2^-24), times the channel's scale plus the bias (one FMA,
2^-24 of the result), then one rounding to the output type (half a step, ``eps / 2``).
The fused GELU passes its input's error on by at most 1.13 (the largest slope of GELU)
and adds its own:
  * f32 results: a fit of erfc within 1.2e-7 (2^-23) with the formula's own f32
    roundings, within |v| 2^-21 of the formula;
  * 16-bit results: max(0, v) - |v| Phi(-|v|) with Phi(-z) = exp(-z^2 / 2) R(z), R a
    polynomial within 2^-13.0 (bf16, degree 8) or 2^-16.8 (f16, degree 10) of its value on
    [0, 5].  The exponent -z^2 / 2 log2 e, at most 18.1, is rounded twice and the
    exponential once (18.1 * 2^-23 + 2^-21 < 2^-18): 2^-12.9 or 2^-16.3 of |v| Phi(-|v|) in
    all.  Past 5 R(5) stands for R(z) and 5 for |v|, which together are off by less than
    their value there, |v| Phi(-|v|) <= 5 * 2.9e-7: by at most 1.5e-6 * exp((25 - v^2) / 2),
    and since both err towards each other by under 2% of it (R falls as 1 / z while the
    factor |v| grows as z): 3e-8.
"""

from __future__ import annotations

import pytest
import torch

from latefuse_b200 import (Int8Rows, Int8Weight, add_layernorm_int8, ffn_int8, linear_int8, quantize_rows)
from latefuse_b200 import _native as nat
from latefuse_b200.encoder_ops import ACT_GELU, ACT_NONE, add_layernorm

pytestmark = pytest.mark.gpu

DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def ref_rows(x):
    """Integers (as f64) and scales of the rows of x, from the definition."""
    top = x.abs().amax(1, keepdim=True)
    q = torch.round(127.0 * x.double() / torch.where(top > 0, top, torch.ones_like(top)).double())
    # through f64: torch divides f32 by a number on the GPU as a product with its reciprocal;
    # top / 127 is never within 2^-33 of a point half way between two f32 unless it is one
    return q, (top.double()[:, 0] / 127.0).float()


def weight(cuda, n, k, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randint(-127, 128, (n, k), device=cuda, generator=g, dtype=torch.int8),
            torch.rand(n, device=cuda, generator=g) * 0.02 + 1e-3)


def activations(cuda, m, k, dtype, seed):
    g = torch.Generator(device=cuda).manual_seed(seed)
    return (torch.randn(m, k, device=cuda, generator=g) * (torch.rand(m, 1, device=cuda, generator=g) * 4 + 0.1)).to(dtype)


def check_projection(y, q, xs, w, ws, bias, act):
    """y against act(q w^T xs ws + bias) in 64 bits, within the roundings counted above."""
    prod = (q.double() @ w.double().t()) * xs.double()[:, None] * ws.double()
    v = prod + (0.0 if bias is None else bias.double())
    tol = 2.0 ** -24 * (3 * prod.abs() + v.abs())
    if act == ACT_GELU:
        if y.dtype == torch.float32:
            own = v.abs() * 2.0 ** -21
        else:
            own = v.abs() * torch.special.ndtr(-v.abs()) * 2.0 ** (-12.9 if y.dtype == torch.bfloat16 else -16.3) + \
                torch.where(v.abs() > 5, 3e-8, 0.0) + v.abs() * 2.0 ** -23
        tol = 1.13 * tol + own
        v = v * torch.special.ndtr(v)
    fi = torch.finfo(y.dtype)
    tol = tol + (v.abs() + tol) * fi.eps / 2 + fi.smallest_normal * fi.eps  # the last: subnormal results
    bad = (y.double() - v).abs() > tol
    assert not bad.any(), (int(bad.sum()), (y.double() - v).abs()[bad].max().item(), tol[bad].min().item())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 1), (3, 7), (5, 8), (17, 1000), (9, 1024), (33, 1032), (4, 2048), (7, 4097),
                                 (6, 8192), (3, 8200), (2, 20001), (1000, 64)])
def test_quantize_rows_is_the_definition(cuda, dtype, m, k):
    x = activations(cuda, m, k, dtype, m * 31 + k)
    r = quantize_rows(x)
    q, scale = ref_rows(x)
    assert torch.equal(r.q.double(), q) and torch.equal(r.scale, scale)
    assert r.q.stride(0) % 16 == 0 and r.dequantize().shape == x.shape


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("k", [1, 9, 256, 1023, 9001])
def test_quantize_rows_of_any_stride_and_alignment(cuda, dtype, k):
    """x from even and odd columns of a wider buffer; q with rows of any stride and alignment,
    whose bytes around them stay as they were."""
    wide = activations(cuda, 21, k + 5, dtype, 3)
    for first in (0, 1, 2, 3):
        x = wide[:, first:first + k]
        want = quantize_rows(x.contiguous())
        rows = quantize_rows(x)
        assert torch.equal(rows.q, want.q) and torch.equal(rows.scale, want.scale)
        q = torch.full((21, k + 6), 99, dtype=torch.int8, device=cuda)
        scale = torch.empty(21, device=cuda)
        part = q[:, 3:3 + k]
        nat.call(nat.lib().lf_quantize_rows, "lf_quantize_rows", x.device, nat.dtype_code(dtype), x.data_ptr(),
                 x.stride(0), 21, k, part.data_ptr(), q.stride(0), scale.data_ptr())
        assert torch.equal(part, want.q) and torch.equal(scale, want.scale)
        assert (q[:, :3] == 99).all() and (q[:, 3 + k:] == 99).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_quantize_rows_ties_and_ends(cuda, dtype):
    """Rows whose largest value is 254 steps make every second integer a tie (to even);
    magnitudes at both ends of the type; strided and misaligned rows."""
    x = torch.arange(-254, 255, device=cuda, dtype=torch.float32).repeat(8, 1)
    x *= torch.tensor([1.0, 2.0, 0.5, 2.0 ** -10, 2.0 ** 7, 1.0, 2.0 ** -20, 1.0], device=cuda)[:, None]
    x = x.to(dtype)  # f16 rounds the row at 2^-20: still a row like any other
    r = quantize_rows(x)
    q, scale = ref_rows(x)
    assert torch.equal(r.q.double(), q) and torch.equal(r.scale, scale)
    fi = torch.finfo(dtype)
    ends = torch.stack([torch.linspace(-1, 1, 64) * fi.max, torch.linspace(-1, 1, 64) * fi.smallest_normal,
                        torch.linspace(-1, 1, 64) * fi.smallest_normal * 3.7 * fi.eps]).to(cuda).to(dtype)
    r = quantize_rows(ends)
    q, scale = ref_rows(ends)
    assert torch.equal(r.q.double(), q) and torch.equal(r.scale, scale)
    for view in (x[:, 1:], x[:, ::2], x.t(), x[2:3], x[0].expand(5, -1), x.view(2, 4, -1)):
        r = quantize_rows(view)
        q, scale = ref_rows(view.reshape(-1, view.shape[-1]))
        assert torch.equal(r.q.double(), q) and torch.equal(r.scale, scale)


@pytest.mark.parametrize("dtype,digits", [(torch.bfloat16, 8), (torch.float16, 11)])
def test_quantize_rows_every_quotient(cuda, dtype, digits):
    """Every pair of significands of the type (f16: every seventh of the largest's), at every
    distance of exponents that leaves a quotient of 1/2 or more: the halves among them,
    and the quotients next to halves, are rounded as the definition says."""
    lo, hi = 2 ** (digits - 1), 2 ** digits
    tops = torch.arange(lo, hi, 1 if digits == 8 else 7, device=cuda)
    sig = torch.arange(lo, hi, device=cuda)
    x = torch.cat([sig * 2.0 ** -k for k in range(9)] + [torch.zeros(1, device=cuda)])
    rows = x.repeat(tops.numel(), 1)
    rows[rows > tops[:, None]] = 1.0
    rows[:, -1] = tops
    rows[:, ::2] *= -1
    rows = (rows * 2.0 ** -6).to(dtype)
    r = quantize_rows(rows)
    q, scale = ref_rows(rows)
    assert torch.equal(r.q.double(), q) and torch.equal(r.scale, scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_rows_of_zeros_infinities_and_nan(cuda, dtype):
    x = torch.randn(6, 72, device=cuda).to(dtype)
    x[1] = 0
    x[2, 5] = float("inf")
    x[3, 70] = float("nan")
    x[4, 0] = float("-inf")
    r = quantize_rows(x)
    assert (r.q[1:5] == 0).all() and r.scale[1] == 0 and r.scale[2:5].isnan().all()
    w, ws = weight(cuda, 40, 72, 3)
    b = torch.randn(40, device=cuda).to(dtype)
    y = linear_int8(x, Int8Weight(w, ws), b)
    assert y[2:5].isnan().all() and torch.equal(y[1], b) and not y[[0, 1, 5]].isnan().any()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 8, 16), (2, 130, 100), (16, 128, 128), (17, 257, 129), (33, 96, 1040),
                                   (65, 1024, 512), (129, 200, 300), (300, 512, 2048), (333, 771, 1000),
                                   (5, 40, 5000), (2500, 1024, 192), (4111, 771, 130), (2300, 1032, 1000)])
def test_linear_int8_matches_the_formula(cuda, dtype, m, n, k):
    x = activations(cuda, m, k, dtype, m + n + k)
    w, ws = weight(cuda, n, k, 5)
    b = torch.randn(n, device=cuda, generator=torch.Generator(device=cuda).manual_seed(7)).to(dtype)
    wt = Int8Weight(w, ws)
    q, xs = ref_rows(x)
    for act in (ACT_NONE, ACT_GELU):
        for bias in (b, None):
            y = linear_int8(x, wt, bias, act=act)
            assert y.dtype == dtype and y.shape == (m, n)
            check_projection(y, q, xs, w, ws, bias, act)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 1024, 1024), (2, 130, 100), (3, 257, 4095), (4, 128, 129), (5, 3000, 2568),
                                   (8, 96, 1040), (9, 12000, 264), (15, 64, 1023), (16, 512, 1024), (4, 40, 4096), (16, 1, 255)])
def test_few_float_rows_are_their_quantised_rows(cuda, dtype, m, n, k):
    """Up to 16 float rows of up to 16,384 elements in all, quantised inside the projection's launch, give
    what quantize_rows and the projection of its rows give, bit for bit: the same integers,
    scales and f32 operations.  Contiguous rows, and rows of a wider buffer from an odd column
    on (an element a load)."""
    g = torch.Generator(cuda).manual_seed(m * n + k)
    wide = torch.randn(m, k + 7, device=cuda, generator=g).to(dtype)
    w = Int8Weight.from_float(torch.randn(n, k, device=cuda, generator=g))
    bias = torch.randn(n, device=cuda, generator=g).to(dtype)
    for x in (wide[:, 3:3 + k].contiguous(), wide[:, 3:3 + k], wide[:, :k]):
        for act in (0, 1):
            before = nat.launch_count()
            y = linear_int8(x, w, bias, act=act)
            assert nat.launch_count() == before + 1
            assert torch.equal(y, linear_int8(quantize_rows(x), w, bias, act=act))


@pytest.mark.parametrize("dtype", DTYPES)
def test_few_float_rows_that_are_not_finite(cuda, dtype):
    x = torch.randn(6, 520, device=cuda).to(dtype)
    x[1] = 0
    x[2, 519] = float("inf")
    x[4, 0] = float("nan")
    w = Int8Weight.from_float(torch.randn(300, 520, device=cuda))
    y = linear_int8(x, w)
    assert y[[2, 4]].isnan().all() and (y[1] == 0).all() and y[[0, 3, 5]].isfinite().all()
    keep = [0, 3, 5]
    assert torch.equal(y[keep], linear_int8(x[keep], w))


def test_rows_do_not_depend_on_their_batch(cuda):
    """The integer sum is exact, so a row's result is the same bits alone, in a small batch
    (the split kernel) and in a large one (the CTA-pair kernel)."""
    x = activations(cuda, 4096, 1024, torch.bfloat16, 1)
    wt = Int8Weight(*weight(cuda, 1024, 1024, 2))
    y = linear_int8(x, wt, act=ACT_GELU)
    for m in (1, 16, 31, 64, 100, 300):
        assert torch.equal(linear_int8(x[:m], wt, act=ACT_GELU), y[:m]), m
    rows = quantize_rows(x)
    assert torch.equal(linear_int8(rows, wt, act=ACT_GELU), y)


def test_largest_sum(cuda):
    """K = 131,072 of 127 * 127: the sum 2,114,060,288 stays inside 32 bits."""
    k = 131072
    x = torch.ones(3, k, device=cuda)
    x[1] = -1
    wt = Int8Weight(torch.full((5, k), 127, dtype=torch.int8, device=cuda), torch.ones(5, device=cuda))
    y = linear_int8(x, wt)
    want = torch.tensor([1.0, -1.0, 1.0], device=cuda)[:, None] * float(127 * k)
    assert ((y - want).abs() <= 4 * 2.0 ** -24 * want.abs()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [3, 50, 2600])
def test_strided_outputs_leave_their_surroundings(cuda, dtype, m):
    x = activations(cuda, m, 520, dtype, m)
    wt = Int8Weight(*weight(cuda, 1000, 520, 4))
    want = linear_int8(x, wt)
    for lead, ld in ((0, 1008), (3, 1005), (8, 1016), (1, 1001)):
        big = torch.full((m + 2, ld + 8), 7.0, device=cuda, dtype=dtype)
        out = big[1:m + 1, lead:lead + 1000]
        assert linear_int8(x, wt, out=out) is out
        assert torch.equal(out, want)
        assert (big[0] == 7).all() and (big[-1] == 7).all() and (big[:, :lead] == 7).all() and \
            (big[:, lead + 1000:] == 7).all()


def test_views_and_shapes(cuda):
    x = activations(cuda, 6 * 7, 2048, torch.bfloat16, 1)
    wt = Int8Weight(*weight(cuda, 264, 1024, 2))
    y = linear_int8(x[:, :1024], wt)
    assert torch.equal(linear_int8(x[:, :1024].reshape(6, 7, 1024), wt), y.view(6, 7, 264))
    assert torch.equal(linear_int8(x[:1, :1024].t().contiguous().t(), wt), y[:1])
    assert linear_int8(x[:0, :1024], wt).shape == (0, 264)
    # a bias of another dtype is taken in x's
    b = torch.randn(264, device=cuda)
    assert torch.equal(linear_int8(x[:, :1024], wt, b), linear_int8(x[:, :1024], wt, b.bfloat16()))
    # int8 weights whose rows are not 16-byte aligned are laid out once
    w, ws = weight(cuda, 9, 37, 3)
    q, xs = ref_rows(x[:, :37])
    check_projection(linear_int8(x[:, :37], Int8Weight(w, ws)), q, xs, w, ws, None, ACT_NONE)


@pytest.mark.parametrize("dtype", DTYPES)
def test_from_float_stays_within_the_quantisation(cuda, dtype):
    """Against the unquantised product: each activation is off by at most half its token's
    step (and a weight by half its channel's), so the sum by at most
    s_w |x|_1 / 2 + s_x |w|_1 / 2 + K s_x s_w / 4."""
    x = activations(cuda, 70, 640, dtype, 1)
    w = torch.randn(300, 640, device=cuda, generator=torch.Generator(device=cuda).manual_seed(9)).to(dtype)
    wt = Int8Weight.from_float(w)
    y = linear_int8(x, wt).double()
    xd, wd = x.double(), w.double()
    sx, sw = (xd.abs().amax(1) / 127)[:, None], (wd.abs().amax(1) / 127)[None]
    tol = sw * xd.abs().sum(1, keepdim=True) / 2 + sx * wd.abs().sum(1)[None] / 2 + 640 * sx * sw / 4
    want = xd @ wd.t()
    tol = tol * (1 + 1e-5) + (want.abs() + tol) * torch.finfo(dtype).eps
    assert ((y - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,h", [(1, 8), (37, 264), (300, 1024), (65, 2560), (9, 4096)])
def test_add_layernorm_int8_is_both_passes(cuda, dtype, m, h):
    a, b = activations(cuda, m, h, dtype, 1), activations(cuda, m, h, dtype, 2)
    w = torch.rand(h, device=cuda).to(dtype) + 0.5
    beta = torch.randn(h, device=cuda).to(dtype)
    for second in (b, None):
        out, rows = add_layernorm_int8(a, second, w, beta, 1e-5)
        want = add_layernorm(a, second, w, beta, 1e-5)
        again = quantize_rows(want)
        assert torch.equal(out, want)
        assert torch.equal(rows.q, again.q) and torch.equal(rows.scale, again.scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m", [1, 40, 1500])
def test_ffn_int8_is_its_parts(cuda, dtype, m):
    h, i = 256, 1032
    a, r = activations(cuda, m, h, dtype, 1), activations(cuda, m, h, dtype, 2)
    w, beta = torch.rand(h, device=cuda).to(dtype) + 0.5, torch.randn(h, device=cuda).to(dtype)
    up, down = weight(cuda, i, h, 3), weight(cuda, h, i, 4)
    ub, db = torch.randn(i, device=cuda).to(dtype), torch.randn(h, device=cuda).to(dtype)
    x, o = ffn_int8(a, r, w, beta, 1e-5, Int8Weight(*up), ub, Int8Weight(*down), db)
    assert torch.equal(x, add_layernorm(a, r, w, beta, 1e-5))
    mid = linear_int8(x, Int8Weight(*up), ub, act=ACT_GELU)
    q, xs = ref_rows(mid)
    check_projection(o, q, xs, *down, db, ACT_NONE)


def test_capture_replay_and_streams(cuda):
    """Captured calls replay on new inputs; two streams run their calls at once."""
    wt = Int8Weight(*weight(cuda, 520, 264, 1))
    for m in (5, 40, 3000):
        xs = [activations(cuda, m, 264, torch.bfloat16, s) for s in range(4)]
        want = [linear_int8(x, wt, act=ACT_GELU) for x in xs]
        static = xs[0].clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            linear_int8(static, wt, act=ACT_GELU)
        torch.cuda.current_stream().wait_stream(side)
        graphs, outs = [], []
        for _ in range(2):  # two graphs of the same call share nothing but their input
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(linear_int8(static, wt, act=ACT_GELU))
            graphs.append(g)
        for x, y in zip(xs, want):
            static.copy_(x)
            for g in graphs:
                g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[0], y) and torch.equal(outs[1], y)
        streams = [torch.cuda.Stream() for _ in range(4)]
        got = []
        torch.cuda.synchronize()
        for _ in range(5):
            for s, x in zip(streams, xs):
                with torch.cuda.stream(s):
                    got.append(linear_int8(x, wt, act=ACT_GELU))
        torch.cuda.synchronize()
        for n, y in enumerate(got):
            assert torch.equal(y, want[n % 4])


def test_refusals(cuda):
    x = torch.randn(4, 64, device=cuda, dtype=torch.bfloat16)
    w, ws = weight(cuda, 32, 64, 1)
    wt = Int8Weight(w, ws)
    with pytest.raises(ValueError, match="columns"):
        linear_int8(x[:, :63], wt)
    with pytest.raises(ValueError, match="bias"):
        linear_int8(x, wt, torch.zeros(31, device=cuda))
    with pytest.raises(ValueError, match="out must be"):
        linear_int8(x, wt, out=torch.empty(32, 4, device=cuda, dtype=torch.bfloat16).t())
    with pytest.raises(ValueError, match="out must be"):
        linear_int8(x, wt, out=torch.empty(4, 32, device=cuda))
    with pytest.raises(nat.NativeLibraryError, match="act"):
        linear_int8(x, wt, act=5)
    with pytest.raises(nat.NativeLibraryError, match="dtype"):
        quantize_rows(x.double())
    with pytest.raises(nat.NativeLibraryError, match="CUDA tensors"):
        linear_int8(x.cpu(), wt)
    with pytest.raises(ValueError, match="up must be"):
        ffn_int8(x, x, x[0], x[0], 1e-5, wt, None, Int8Weight(*weight(cuda, 64, 33, 1)), None)
    rows = quantize_rows(x)
    assert isinstance(rows, Int8Rows)
    with pytest.raises(ValueError, match="columns"):
        linear_int8(rows, Int8Weight(*weight(cuda, 32, 48, 1)))


@pytest.mark.parametrize("m", [4, 40])
def test_outputs_over_their_inputs_are_refused(cuda, m):
    fused = torch.randn(m, 96, device=cuda, dtype=torch.bfloat16)
    wt = Int8Weight(*weight(cuda, 32, 64, 1))
    x = fused[:, :64]
    with pytest.raises(ValueError, match="overlap"):
        linear_int8(x, wt, out=fused[:, 40:72])
    want = linear_int8(x, wt)
    assert torch.equal(linear_int8(x, wt, out=fused[:, 64:]), want)  # its own columns of the same rows
    rows = quantize_rows(torch.randn(m, 64, device=cuda, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="overlap"):
        linear_int8(rows, wt, out=rows.q.view(torch.bfloat16))
