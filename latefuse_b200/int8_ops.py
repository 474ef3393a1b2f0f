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

import torch
from torch import Tensor

from latefuse_b200 import _native as nat
from latefuse_b200.encoder_ops import ACT_GELU, ACT_NONE

_MAX_K = 131072


def _padded(n: int) -> int:
    return (n + 15) // 16 * 16


def _rows(t: Tensor) -> tuple[Tensor, int]:
    """``t`` as rows of its last dimension, each contiguous and at least a row apart."""
    k = t.shape[-1]
    t2 = t.reshape(-1, k)
    if (k > 1 and t2.stride(1) != 1) or (t2.shape[0] > 1 and t2.stride(0) < k):
        t2 = t2.contiguous()
    return t2, max(t2.stride(0), k)


class Int8Rows:
    """Rows held in 8-bit integers: ``q`` is the ``(M, K)`` int8 view (rows 16-byte aligned),
    ``scale`` the ``(M,)`` f32 scales, ``shape`` and ``dtype`` those of the tensor it came
    from (``shape[:-1]`` has M elements)."""

    __slots__ = ("q", "scale", "shape", "dtype")

    def __init__(self, q: Tensor, scale: Tensor, shape: tuple, dtype: torch.dtype):
        self.q, self.scale, self.shape, self.dtype = q, scale, tuple(shape), dtype

    def dequantize(self) -> Tensor:
        """The values the integers stand for, in ``shape`` and ``dtype``."""
        return (self.q.float() * self.scale.unsqueeze(1)).to(self.dtype).view(self.shape)


class Int8Weight:
    """An ``nn.Linear`` weight ``(N, K)`` in 8-bit integers with a scale per output channel.

    ``Int8Weight(q, scale)`` takes int8 ``(N, K)`` in [-127, 127] and f32 ``(N,)`` (rows are
    laid out 16-byte aligned once, here); ``Int8Weight.from_float(weight)`` quantises a
    float weight on its GPU."""

    __slots__ = ("q", "scale")

    def __init__(self, q: Tensor, scale: Tensor):
        if q.dim() != 2 or q.dtype != torch.int8:
            raise ValueError(f"an int8 (N, K) weight is needed, got {q.dtype} {tuple(q.shape)}")
        if scale.shape != q.shape[:1] or scale.dtype != torch.float32 or scale.device != q.device:
            raise ValueError(f"scale must be a ({q.shape[0]},) float32 tensor on {q.device}")
        n, k = q.shape
        if not 1 <= k <= _MAX_K or n < 1:
            raise ValueError(f"weight of {n} x {k}: K must be in 1..{_MAX_K}")
        if q.stride(1) != 1 or q.stride(0) % 16 or q.stride(0) < k or q.data_ptr() % 16:
            laid = torch.empty(n, _padded(k), dtype=torch.int8, device=q.device)[:, :k]
            q = laid.copy_(q)
        self.q, self.scale = q, scale.contiguous()

    @classmethod
    def from_float(cls, weight: Tensor) -> Int8Weight:
        if weight.dim() != 2:
            raise ValueError(f"an (N, K) weight is needed, got {tuple(weight.shape)}")
        rows = quantize_rows(weight)
        return cls(rows.q, rows.scale)

    @property
    def shape(self) -> torch.Size:
        return self.q.shape


def _quantize(x2: Tensor, ldx: int, dev: torch.device) -> tuple[Tensor, Tensor]:
    m, k = x2.shape
    q = torch.empty(m, _padded(k), dtype=torch.int8, device=dev)
    scale = torch.empty(m, dtype=torch.float32, device=dev)
    rc = nat.lib().lf_quantize_rows(nat.stream_ptr(dev), nat.dtype_code(x2.dtype), x2.data_ptr(), ldx, m, k,
                                    q.data_ptr(), q.stride(0), scale.data_ptr())
    nat.check(rc, "lf_quantize_rows")
    return (q if q.shape[1] == k else q[:, :k]), scale


def quantize_rows(x: Tensor) -> Int8Rows:
    """The rows (last dimension) of an f32, bf16 or f16 tensor in 8-bit integers with a scale
    each.  A row of zeros has scale 0; a row holding an infinity or NaN has scale NaN."""
    dev = nat.require_cuda(x)
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"rows of at least one element are needed, got {tuple(x.shape)}")
    with nat.on_device(dev):
        x2, ldx = _rows(x)
        q, scale = _quantize(x2, ldx, dev)
    return Int8Rows(q, scale, x.shape, x.dtype)


def linear_int8(x: Tensor | Int8Rows, weight: Int8Weight, bias: Tensor | None = None, act: int = ACT_NONE,
                out: Tensor | None = None) -> Tensor:
    """``act(x @ weight.T + bias)`` in 8-bit integers: ``x (..., K)`` f32, bf16 or f16, quantised
    per row first, or :class:`Int8Rows`; ``act`` is ``ACT_NONE`` or ``ACT_GELU`` (the exact erf
    GELU).  The result has x's dtype and is rounded to it once.  Any M, N and K up to 131,072;
    ``out`` must be viewable as rows without a copy and must not overlap ``x``."""
    rows = isinstance(x, Int8Rows)
    dev = nat.require_cuda(x.q if rows else x, weight.q, bias, out)
    n, k = weight.q.shape
    if x.shape[-1] != k:
        raise ValueError(f"x has {x.shape[-1]} columns, weight expects {k}")
    dtype = x.dtype
    with nat.on_device(dev):
        if rows:
            q, scale = x.q, x.scale
        else:
            x2, ldx = _rows(x)
            q, scale = _quantize(x2, ldx, dev)
        m = q.shape[0]
        if out is None:
            out = torch.empty(*x.shape[:-1], n, dtype=dtype, device=dev)
            o2 = out if out.dim() == 2 else out.view(m, n)
        else:
            o2 = out.reshape(-1, n)
            if out.dtype != dtype or o2.shape[0] != m or o2.data_ptr() != out.data_ptr() or \
                    (n > 1 and o2.stride(-1) != 1) or (out.dim() > 2 and not out.is_contiguous()):
                raise ValueError(f"out must be ({m}, {n}) {dtype} rows viewable without a copy")
        b = None
        if bias is not None:
            if bias.shape != (n,):
                raise ValueError(f"bias must have {n} entries, got {tuple(bias.shape)}")
            b = (bias if bias.dtype == dtype else bias.to(dtype)).contiguous()
        rc = nat.lib().lf_linear_int8(nat.stream_ptr(dev), nat.dtype_code(dtype), q.data_ptr(), q.stride(0),
                                      scale.data_ptr(), weight.q.data_ptr(), weight.q.stride(0),
                                      weight.scale.data_ptr(), nat.ptr(b), o2.data_ptr(), max(o2.stride(0), n), m, n, k,
                                      int(act), None)
        nat.check(rc, "lf_linear_int8")
    return out


def add_layernorm_int8(a: Tensor, b: Tensor | None, weight: Tensor, bias: Tensor, eps: float) -> tuple[Tensor, Int8Rows]:
    """``add_layernorm(a, b, weight, bias, eps)`` and its rows in 8-bit integers, in one pass."""
    dev = nat.require_cuda(a, b, weight, bias)
    H = a.shape[-1]
    if b is not None and (b.shape != a.shape or b.dtype != a.dtype):
        raise ValueError(f"a is {a.dtype} {tuple(a.shape)}, b {b.dtype} {tuple(b.shape)}")
    if weight.shape != (H,) or bias.shape != (H,):
        raise ValueError(f"weight and bias must have {H} entries")
    with nat.on_device(dev):
        a2, lda = _rows(a)
        b2, ldb = _rows(b) if b is not None else (None, 0)
        out = torch.empty(a.shape, dtype=a.dtype, device=dev)
        m = a2.shape[0]
        q = torch.empty(m, _padded(H), dtype=torch.int8, device=dev)
        scale = torch.empty(m, dtype=torch.float32, device=dev)
        w = (weight if weight.dtype == a.dtype else weight.to(a.dtype)).contiguous()
        bb = (bias if bias.dtype == a.dtype else bias.to(a.dtype)).contiguous()
        rc = nat.lib().lf_add_layernorm_int8(nat.stream_ptr(dev), nat.dtype_code(a.dtype), a2.data_ptr(), lda,
                                             nat.ptr(b2), ldb, w.data_ptr(), bb.data_ptr(), float(eps), m, H,
                                             out.data_ptr(), H, q.data_ptr(), q.stride(0), scale.data_ptr())
        nat.check(rc, "lf_add_layernorm_int8")
    return out, Int8Rows(q[:, :H], scale, a.shape, a.dtype)


def ffn_int8(a: Tensor, residual: Tensor | None, ln_weight: Tensor, ln_bias: Tensor, eps: float, up: Int8Weight,
             up_bias: Tensor | None, down: Int8Weight, down_bias: Tensor | None,
             act: int = ACT_GELU) -> tuple[Tensor, Tensor]:
    """The encoder layer's feed-forward half with both projections in 8-bit integers:
    ``h = layer_norm(a + residual)`` and ``o = down(act(up(h)))``, the middle activations
    rounded to a's dtype and then quantised per token.  Returns ``(h, o)``: the layer's
    output is ``add_layernorm(o, h, ...)``."""
    if down.shape[1] != up.shape[0]:
        raise ValueError(f"up gives {up.shape[0]} columns, down expects {down.shape[1]}")
    h, rows = add_layernorm_int8(a, residual, ln_weight, ln_bias, eps)
    mid = linear_int8(rows, up, up_bias, act=act)
    return h, linear_int8(mid, down, down_bias)
