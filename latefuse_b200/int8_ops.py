"""Projections in 8-bit integers (W8A8), for the parts of the encoder that carry no LoRA delta.

A row of activations (a token) or of a weight (an output channel) is held as int8 steps
of its own scale: ``scale = max|row| / 127``, ``q = round(127 row / max|row|)`` (ties to
even, decided exactly).  A projection multiplies the integers exactly on the tensor
cores and scales the sum by the token's and the channel's scale:

    ``y = act((q_x q_w^T) * scale_x * scale_w + bias)``

``quantize_rows`` quantises a tensor's rows, ``linear_int8`` is the projection (on a
float tensor, which it quantises first, or on rows that already are),
``add_layernorm_int8`` is ``encoder_ops.add_layernorm`` whose output is quantised in the
same pass, and ``ffn_int8`` is the encoder layer's feed-forward half made of them (see
the ``lf_*`` declarations in ``include/latefuse_b200.h``).
"""

from __future__ import annotations

import math

import torch
from torch import Tensor

from latefuse_b200 import _native as nat
from latefuse_b200.encoder_ops import ACT_GELU, ACT_NONE, _share_memory

_MAX_K = 131072
_MAX_N = 2**31 - 257
_MAX_COLS = 2**31 - 1 - 4096  # lf_quantize_rows'


def _padded(n: int) -> int:
    return (n + 15) // 16 * 16


def _up256(n: int) -> int:
    return (n + 255) // 256 * 256


def _rows(t: Tensor) -> tuple[Tensor, int]:
    """``t`` as rows of its last dimension, each contiguous and at least a row apart, and
    their stride."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    m, k = t.shape
    s0, s1 = t.stride()
    if (k > 1 and s1 != 1) or (m > 1 and s0 < k):
        t = t.contiguous()
        s0 = k
    return t, (s0 if m > 1 else k)


class Int8Rows:
    """Rows held in 8-bit integers: ``q`` is the ``(M, K)`` int8 view (rows 16-byte aligned),
    ``scale`` the ``(M,)`` f32 scales, ``shape`` and ``dtype`` those of the tensor it came
    from (``shape[:-1]`` has M elements)."""

    __slots__ = ("q", "scale", "shape", "dtype", "ld")

    def __init__(self, q: Tensor, scale: Tensor, shape: tuple, dtype: torch.dtype):
        if q.dim() != 2 or q.dtype != torch.int8 or (q.shape[1] > 1 and q.stride(1) != 1):
            raise ValueError(f"int8 rows (M, K) are needed, got {q.dtype} {tuple(q.shape)}, strides {q.stride()}")
        m, k = q.shape
        if scale.shape != (m,) or scale.dtype != torch.float32 or scale.device != q.device or not scale.is_contiguous():
            raise ValueError(f"scale must be a contiguous ({m},) float32 tensor on {q.device}")
        if not shape or shape[-1] != k or math.prod(shape[:-1]) != m:
            raise ValueError(f"shape {tuple(shape)} is not {m} rows of {k}")
        self._set(q, scale, tuple(shape), dtype, q.stride(0) if m > 1 else _padded(k))

    def _set(self, q: Tensor, scale: Tensor, shape: tuple, dtype: torch.dtype, ld: int) -> Int8Rows:
        self.q, self.scale, self.shape, self.dtype, self.ld = q, scale, shape, dtype, ld
        return self

    def dequantize(self) -> Tensor:
        """The values the integers stand for, in ``shape`` and ``dtype``."""
        return (self.q.float() * self.scale.unsqueeze(1)).to(self.dtype).view(self.shape)


class Int8Weight:
    """An ``nn.Linear`` weight ``(N, K)`` in 8-bit integers with a scale per output channel.

    ``Int8Weight(q, scale)`` takes int8 ``(N, K)`` in [-127, 127] and f32 ``(N,)`` (rows that
    are not 16-byte aligned are laid out so once, here); ``Int8Weight.from_float(weight)``
    quantises a float weight on its GPU."""

    __slots__ = ("q", "scale", "shape", "ld")

    def __init__(self, q: Tensor, scale: Tensor):
        if q.dim() != 2 or q.dtype != torch.int8:
            raise ValueError(f"an int8 (N, K) weight is needed, got {q.dtype} {tuple(q.shape)}")
        if scale.shape != q.shape[:1] or scale.dtype != torch.float32 or scale.device != q.device:
            raise ValueError(f"scale must be a ({q.shape[0]},) float32 tensor on {q.device}")
        n, k = q.shape
        if not 1 <= k <= _MAX_K or not 1 <= n <= _MAX_N:
            raise ValueError(f"weight of {n} x {k}: K must be in 1..{_MAX_K}, N in 1..{_MAX_N}")
        if (k > 1 and q.stride(1) != 1) or q.data_ptr() % 16 or q.stride(0) % 16 or q.stride(0) < k:
            q = torch.empty(n, _padded(k), dtype=torch.int8, device=q.device)[:, :k].copy_(q)
        self.q, self.scale, self.shape, self.ld = q, scale.contiguous(), (n, k), q.stride(0)

    @classmethod
    def from_float(cls, weight: Tensor) -> Int8Weight:
        if weight.dim() != 2:
            raise ValueError(f"an (N, K) weight is needed, got {tuple(weight.shape)}")
        rows = quantize_rows(weight)
        return cls(rows.q, rows.scale)


def quantize_rows(x: Tensor) -> Int8Rows:
    """The rows (last dimension) of an f32, bf16 or f16 tensor in 8-bit integers with a scale
    each.  A row of zeros has scale 0; a row holding an infinity or NaN has scale NaN."""
    if x.dim() < 1 or not 1 <= x.shape[-1] <= _MAX_COLS:
        raise ValueError(f"rows of 1 to {_MAX_COLS} elements are needed, got {tuple(x.shape)}")
    dev = nat.require_cuda(x)
    x2, ldx = _rows(x)
    m, k = x2.shape
    kp = _padded(k)
    q = torch.empty(m, kp, dtype=torch.int8, device=dev)
    scale = torch.empty(m, dtype=torch.float32, device=dev)
    nat.call(nat.lib().lf_quantize_rows, "lf_quantize_rows", dev, nat.dtype_code(x.dtype), x2.data_ptr(), ldx, m, k,
             q.data_ptr(), kp, scale.data_ptr())
    return Int8Rows.__new__(Int8Rows)._set(q if kp == k else q[:, :k], scale, x.shape, x.dtype, kp)


def _bias(bias: Tensor | None, n: int, dtype: torch.dtype) -> Tensor | None:
    if bias is None:
        return None
    if bias.dim() != 1 or bias.numel() != n:
        raise ValueError(f"bias must have {n} entries, got {tuple(bias.shape)}")
    if bias.dtype is not dtype:
        bias = bias.to(dtype)
    return bias if bias.is_contiguous() else bias.contiguous()


def linear_int8(x: Tensor | Int8Rows, weight: Int8Weight, bias: Tensor | None = None, act: int = ACT_NONE,
                out: Tensor | None = None, status: Tensor | None = None) -> Tensor:
    """``act(x @ weight.T + bias)`` in 8-bit integers: ``x (..., K)`` f32, bf16 or f16, quantised
    per row first, or :class:`Int8Rows`; ``act`` is ``ACT_NONE`` or ``ACT_GELU`` (the erf GELU;
    bf16 and f16 results take it within 2^-17 of ``|v| Phi(-|v|)``, so that 0.02% and 0.03% of
    them round to the neighbouring value).  The result has x's dtype and is rounded to it
    once.  Any M, N and K up to 131,072;
    ``out`` must be viewable as rows without a copy and must overlap none of the inputs.  A wait that
    runs out sets ``LF_STATUS_TIMEOUT`` in ``status`` (an int32 on the GPU), where one is given,
    and leaves the result undefined."""
    rows = type(x) is Int8Rows
    dev = nat.require_cuda(x.q if rows else x, weight.q, bias, out, status)
    n, k = weight.shape
    shape, dtype = x.shape, x.dtype
    if shape[-1] != k:
        raise ValueError(f"x has {shape[-1]} columns, weight expects {k}")
    bias = _bias(bias, n, dtype)
    if rows:
        m = x.q.shape[0]
    else:
        x2, ldx = _rows(x)
        m = x2.shape[0]
    if out is None:
        out = torch.empty(m, n, dtype=dtype, device=dev) if rows else x.new_empty((m, n))
        ldo, ret = n, out if len(shape) == 2 else out.view(*shape[:-1], n)
    else:
        o2 = out.reshape(-1, n)
        ldo = o2.stride(0) if m > 1 else n
        if out.dtype != dtype or o2.shape[0] != m or o2.data_ptr() != out.data_ptr() or ldo < n or \
                (n > 1 and o2.stride(1) != 1) or (out.dim() > 2 and not out.is_contiguous()):
            raise ValueError(f"out must be ({m}, {n}) {dtype} rows viewable without a copy")
        inputs = [x.q, x.scale] if rows else [x2]
        for t in (*inputs, weight.q, weight.scale, *([] if bias is None else [bias])):
            if _share_memory(o2, t if t.dim() == 2 else t.view(1, -1)):
                raise ValueError("out must not overlap x, the weight, the scales or the bias")
        ret = out
    code, b = nat.dtype_code(dtype), nat.ptr(bias)
    if rows:
        nat.call(nat.lib().lf_linear_int8, "lf_linear_int8", dev, code, x.q.data_ptr(), x.ld, x.scale.data_ptr(),
                 weight.q.data_ptr(), weight.ld, weight.scale.data_ptr(), b, out.data_ptr(), ldo, m, n, k, int(act),
                 nat.ptr(status))
    else:
        size = _rows_bytes(m, k)
        ws = torch.empty(size, dtype=torch.uint8, device=dev) if size else None
        nat.call(nat.lib().lf_linear_rows_int8, "lf_linear_rows_int8", dev, code, x2.data_ptr(), ldx, weight.q.data_ptr(),
                 weight.ld, weight.scale.data_ptr(), b, out.data_ptr(), ldo, m, n, k, int(act), nat.ptr(ws), size,
                 nat.ptr(status))
    return ret


def _rows_bytes(m: int, k: int) -> int:
    """``lf_linear_rows_int8_workspace_bytes``, without the call."""
    return 0 if m <= 16 and k <= 4096 and m * k <= 16384 else _up256(m * _padded(k)) + _up256(4 * m)


def _ffn_bytes(size: int, m: int, hidden: int, inner: int) -> int:
    """``lf_ffn_int8_workspace_bytes``, without the call, for elements of ``size`` bytes."""
    return _up256(m * _padded(hidden)) + _up256(m * _padded(inner)) + 2 * _up256(4 * m) + _up256(m * _padded(inner) * size)


def add_layernorm_int8(a: Tensor, b: Tensor | None, weight: Tensor, bias: Tensor, eps: float) -> tuple[Tensor, Int8Rows]:
    """``add_layernorm(a, b, weight, bias, eps)`` and its rows in 8-bit integers, in one pass."""
    H, dtype = a.shape[-1], a.dtype
    if H >= 2**31:
        raise ValueError(f"rows of {H} elements")
    dev = nat.require_cuda(a, b, weight, bias)
    _same_rows(a, b)
    a2, lda = _rows(a)
    b2, ldb = _rows(b) if b is not None else (None, 0)
    m, hp = a2.shape[0], _padded(H)
    w, bb = _bias(weight, H, dtype), _bias(bias, H, dtype)
    out = torch.empty(a.shape, dtype=dtype, device=dev)
    q = torch.empty(m, hp, dtype=torch.int8, device=dev)
    scale = torch.empty(m, dtype=torch.float32, device=dev)
    nat.call(nat.lib().lf_add_layernorm_int8, "lf_add_layernorm_int8", dev, nat.dtype_code(dtype), a2.data_ptr(), lda,
             nat.ptr(b2), ldb, w.data_ptr(), bb.data_ptr(), float(eps), m, H, out.data_ptr(), H, q.data_ptr(), hp,
             scale.data_ptr())
    return out, Int8Rows.__new__(Int8Rows)._set(q if hp == H else q[:, :H], scale, a.shape, dtype, hp)


def _same_rows(a: Tensor, b: Tensor | None) -> None:
    if b is not None and (b.shape != a.shape or b.dtype != a.dtype):
        raise ValueError(f"a is {a.dtype} {tuple(a.shape)}, the residual {b.dtype} {tuple(b.shape)}")


def ffn_int8(a: Tensor, residual: Tensor | None, ln_weight: Tensor, ln_bias: Tensor, eps: float, up: Int8Weight,
             up_bias: Tensor | None, down: Int8Weight, down_bias: Tensor | None,
             act: int = ACT_GELU, status: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """The encoder layer's feed-forward half with both projections in 8-bit integers:
    ``h = layer_norm(a + residual)`` and ``o = down(act(up(h)))``, the middle activations
    rounded to a's dtype and then quantised per token.  Returns ``(h, o)``: the layer's
    output is ``add_layernorm(o, h, ...)``.  ``status`` as for :func:`linear_int8`."""
    dev = nat.require_cuda(a, residual, ln_weight, ln_bias, up.q, up_bias, down.q, down_bias, status)
    inner, hidden = up.shape
    dtype = a.dtype
    if a.shape[-1] != hidden or down.shape != (hidden, inner):
        raise ValueError(f"a has {a.shape[-1]} columns, up is {up.shape}, down {down.shape}: "
                         "up must be (inner, hidden), down (hidden, inner)")
    _same_rows(a, residual)
    a2, lda = _rows(a)
    r2, ldr = _rows(residual) if residual is not None else (None, 0)
    m = a2.shape[0]
    w, bb = _bias(ln_weight, hidden, dtype), _bias(ln_bias, hidden, dtype)
    ub, db = _bias(up_bias, inner, dtype), _bias(down_bias, hidden, dtype)
    h, o = a2.new_empty((m, hidden)), a2.new_empty((m, hidden))
    lib, code = nat.lib(), nat.dtype_code(dtype)
    size = _ffn_bytes(dtype.itemsize, m, hidden, inner)
    ws = torch.empty(size, dtype=torch.uint8, device=dev)
    nat.call(lib.lf_ffn_int8, "lf_ffn_int8", dev, code, a2.data_ptr(), lda, nat.ptr(r2), ldr, w.data_ptr(), bb.data_ptr(),
             float(eps), up.q.data_ptr(), up.ld, up.scale.data_ptr(), nat.ptr(ub), down.q.data_ptr(), down.ld,
             down.scale.data_ptr(), nat.ptr(db), m, hidden, inner, int(act), h.data_ptr(), hidden, o.data_ptr(), hidden,
             ws.data_ptr(), size, nat.ptr(status))
    return (h, o) if a.dim() == 2 else (h.view(a.shape), o.view(a.shape))
