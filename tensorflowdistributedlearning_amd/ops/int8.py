"""Linear layers and 1×1 convolutions in 8-bit integers, for inference.

    s_m = max_k |x_mk| / 127,   q_mk = rint(127 x_mk / max)          one scale per row (token, pixel)
    y_mn = act(s_m · w_n · Σ_k q_mk W_nk + bias_n [+ residual_mn])    one scale per output channel

``Int8Weight`` holds a layer's weight, laid out once; ``int8_linear(x, weight)`` quantises the rows
of x on the fly and multiplies (``csrc/kernels/int8.hip``: the sum is exact in 32-bit integers, the
epilogue is fused).  Layers that read the same activations share ``quantize_rows(x)``.
"""
from __future__ import annotations

import torch
from torch.autograd import forward_ad

from .common import on_gpu, ext

TINY = 2.0 ** -40   # smallest row maximum a scale is made from (csrc/kernels/int8.hip)
MAX_K = 131071      # longest sum that 32-bit integers hold for sure


def _check_k(k):
    if not 1 <= k <= MAX_K:
        raise ValueError(f"int8: 1 <= K <= {MAX_K}, got {k}")


def _kp(k):
    return (k + 127) // 128 * 128


def to_blocks(q):
    """[R, K] int8 → the kernels' order (csrc/kernels/int8.h): zero-padded to 16 rows and 128 k,
    blocks of 16 rows × 64 k as [4][16 rows][16 bytes]."""
    r, k = q.shape
    rp, kp = (r + 15) // 16 * 16, _kp(k)
    p = torch.zeros(rp, kp, dtype=torch.int8, device=q.device)
    p[:r, :k] = q
    return p.view(rp // 16, 16, kp // 64, 4, 16).permute(0, 2, 3, 1, 4).contiguous().view(rp, kp)


def from_blocks(p, rows, k):
    """The inverse of :func:`to_blocks`."""
    rp, kp = p.shape
    q = p.view(rp // 16, kp // 64, 4, 16, 16).permute(0, 3, 1, 2, 4).reshape(rp, kp)
    return q[:rows, :k]


def ref_quantize_rows(x):
    """(q int8 [M, K], scale fp32 [M]); the quotient in 64 bits, ties to even.  A row with a NaN or
    an infinity has the scale NaN and zeros."""
    xf = x.float()
    bad = ~torch.isfinite(xf).all(1)
    top = xf.abs().nan_to_num(0.0, 0.0).amax(1).clamp_min(TINY)
    q = torch.round(xf.double() * 127 / top.double()[:, None])
    q = torch.where(bad[:, None], torch.zeros_like(q), q).to(torch.int8)
    return q, torch.where(bad, torch.full_like(top, float("nan")), top / 127)


class Int8Weight:
    """A [N, K] weight in 8 bits with one scale per output channel, in the kernels' layout.

    ``Int8Weight(wq, scale)`` takes int8 values and fp32 scales; ``Int8Weight.quantize(w)`` makes
    them from a floating-point weight with the rule of the rows (scale = max / 127)."""

    def __init__(self, wq, scale):
        if wq.dim() != 2 or wq.dtype != torch.int8 or wq.shape[0] < 1:
            raise ValueError(f"Int8Weight: int8 [N, K], got {wq.dtype} {tuple(wq.shape)}")
        if scale.dtype != torch.float32 or tuple(scale.shape) != (wq.shape[0],):
            raise ValueError(f"Int8Weight: scale fp32 [{wq.shape[0]}], got {scale.dtype} {tuple(scale.shape)}")
        if scale.device != wq.device:
            raise ValueError(f"Int8Weight: scale on {scale.device}, weight on {wq.device}")
        _check_k(wq.shape[1])
        self.n, self.k = wq.shape
        self.blocks = to_blocks(wq)
        self.scale = scale.detach().clone()

    @classmethod
    def quantize(cls, w):
        if w.dim() != 2 or w.shape[0] < 1:
            raise ValueError(f"Int8Weight.quantize: [N, K], got {tuple(w.shape)}")
        _check_k(w.shape[1])
        return cls(*ref_quantize_rows(w.detach()))

    @property
    def device(self):
        return self.blocks.device

    def dequantize(self):
        return from_blocks(self.blocks, self.n, self.k).float() * self.scale[:, None]


class Int8Rows:
    """Quantised activations: rows of ``shape[:-1]`` over K = ``shape[-1]`` (see
    :func:`quantize_rows`); ``dtype`` is the type they came in and outputs go back to."""

    def __init__(self, blocks, scale, shape, dtype):
        self.blocks, self.scale, self.shape, self.dtype = blocks, scale, tuple(shape), dtype

    def dequantize(self):
        q = from_blocks(self.blocks, self.scale.numel(), self.shape[-1])
        return (q.float() * self.scale[:, None]).view(self.shape)


def _no_tangent(who, *tensors):
    if forward_ad._current_level >= 0 and any(
            t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{who}: inference only, no forward-mode derivative")


def _check_rows(x, who):
    if x.dim() < 1:
        raise ValueError(f"{who}: x [..., K], got a scalar")
    if x.dtype != torch.bfloat16 and x.dtype != torch.float32:
        raise TypeError(f"{who}: bf16 / fp32 activations, got {x.dtype}")
    if x.requires_grad and torch.is_grad_enabled():
        raise RuntimeError(f"{who}: inference only (torch.no_grad(), or a tensor without gradient)")
    _no_tangent(who, x)
    _check_k(x.shape[-1])


def quantize_rows(x):
    """Rows of ``x`` [..., K] (bf16 / fp32) in 8 bits with one scale each: :class:`Int8Rows`, for
    :func:`int8_linear` calls that share them."""
    _check_rows(x, "quantize_rows")
    m = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    if on_gpu(m):
        if (m.shape[1] > 1 and m.stride(1) != 1) or (m.shape[0] > 1 and m.stride(0) < m.shape[1]):
            m = m.contiguous()
        blocks, scale = ext().int8_quantize(m)
    else:
        q, scale = ref_quantize_rows(m)
        blocks = to_blocks(q)
    return Int8Rows(blocks, scale, x.shape, x.dtype)


def int8_linear(x, weight, bias=None, residual=None, relu=False):
    """act(x · Wᵀ + bias [+ residual]) with 8-bit operands, in x's type.

    ``x``: [..., K] bf16 / fp32 (rows are quantised here) or :class:`Int8Rows`; ``weight``:
    :class:`Int8Weight` [N, K]; ``bias``: fp32 [N]; ``residual``: [..., N] of x's type.  A row of x
    that holds a NaN or an infinity comes out as NaN.  Inference only."""
    if not isinstance(weight, Int8Weight):
        raise TypeError(f"int8_linear: weight is an Int8Weight, got {type(weight).__name__}")
    rows = x if isinstance(x, Int8Rows) else None
    if rows is None:
        _check_rows(x, "int8_linear")
    if x.shape[-1] != weight.k:
        raise ValueError(f"int8_linear: x has K = {x.shape[-1]}, the weight {weight.k}")
    device = (x if rows is None else rows.scale).device
    if device != weight.device:
        raise ValueError(f"int8_linear: x on {device}, weight on {weight.device}")
    _no_tangent("int8_linear", bias, residual)
    if bias is not None:
        if bias.dtype != torch.float32 or bias.shape != (weight.n,) or bias.device != device:
            raise ValueError(f"int8_linear: bias fp32 [{weight.n}] on {device}, got {bias.dtype} "
                             f"{tuple(bias.shape)} on {bias.device}")
        bias = bias.detach().contiguous()
    if residual is not None:
        out_shape = (*x.shape[:-1], weight.n)
        if residual.shape != out_shape or residual.dtype != x.dtype or residual.device != device:
            raise ValueError(f"int8_linear: residual {x.dtype} {out_shape} on {device}, got "
                             f"{residual.dtype} {tuple(residual.shape)} on {residual.device}")
        if residual.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("int8_linear: inference only")
    if rows is None and device.type == "cuda":
        return ext().int8_linear(x, weight.blocks, weight.scale, weight.n, bias, residual, relu)
    out_shape = (*x.shape[:-1], weight.n)
    if residual is not None:
        residual = residual.reshape(-1, weight.n).contiguous()
    if rows is None:
        rows = quantize_rows(x)
    m = rows.scale.numel()
    if device.type == "cuda":
        y = torch.empty(m, weight.n, dtype=x.dtype, device=device)
        ext().int8_gemm(rows.blocks, rows.scale, weight.blocks, weight.scale, weight.k, bias,
                        residual, relu, y)
        return y.view(out_shape)
    q = from_blocks(rows.blocks, m, weight.k).double()
    acc = (q @ from_blocks(weight.blocks, weight.n, weight.k).double().t()).float()
    y = acc * (rows.scale[:, None] * weight.scale)
    if bias is not None:
        y = y + bias
    if residual is not None:
        y = y + residual.float()
    return (torch.relu(y) if relu else y).to(x.dtype).view(out_shape)
