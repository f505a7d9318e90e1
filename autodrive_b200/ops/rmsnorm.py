"""Root-mean-square norm with the residual's addition on fused sm_100a kernels
(``csrc/rmsnorm.cu``): one read and one write of each element, fp32 sums.

``rms_norm(x, weight, residual=None, eps)`` normalises the last dimension of
`x` (fp32, bf16 or fp16; at most 32768 wide), with autograd. With a residual
it returns ``(y, h)``: h = x + residual, rounded to x's dtype, is the new
residual stream, and y its norm.

``rms_norm_fp8`` is the same with an 8-bit result: ``(q, scale)`` or
``(q, scale, h)``, q in e4m3 with one fp32 scale for each row and 128 columns,
as ``ops.fp8.fp8_matmul`` takes its first operand. It has no gradient.

``FusedRMSNorm`` is a drop-in ``nn.RMSNorm`` over one dimension whose forward
also takes a residual. On CPU all of them are plain PyTorch.
"""
from __future__ import annotations

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from ..utils import launches
from .ext import require_extension

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_WIDTH = 32768


def _check(x: Tensor, weight: Tensor, residual: Tensor | None) -> None:
    if x.dim() < 1 or x.dtype not in DTYPES:
        raise ValueError("rms_norm takes fp32, bf16 or fp16 rows")
    if not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"rms_norm rows are 1 to {MAX_WIDTH} wide, not {x.shape[-1]}")
    if weight.shape != x.shape[-1:] or weight.dtype not in DTYPES or weight.device != x.device:
        raise ValueError(f"rms_norm needs an fp32, bf16 or fp16 weight [{x.shape[-1]}] on {x.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("rms_norm needs a residual of x's shape, dtype and device")


def _rows(x: Tensor) -> Tensor:
    """`x` as [rows, D] with contiguous columns and rows that do not overlap."""
    y = x.reshape(-1, x.shape[-1])
    return y if y.stride(1) == 1 and y.stride(0) >= y.shape[1] else y.contiguous()


def from_rows(y: Tensor, lead) -> Tensor:
    """[rows, n] with the leading dimensions `lead` in place of its rows (a view)."""
    return y[0] if len(lead) == 0 else (y if len(lead) == 1 else y.unflatten(0, lead))


def reference_rms_norm(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-6):
    """The same operation in plain PyTorch, in fp32 (CPU path and test oracle)."""
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    y = (hf * (hf.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.float()).to(x.dtype)
    return y if residual is None else (y, h)


def reference_rms_norm_grad(dy: Tensor, dh: Tensor | None, h: Tensor, weight: Tensor, rstd: Tensor):
    """(dx, dweight) of rows in plain PyTorch, in fp32."""
    g, n = dy.float() * weight.float(), h.float() * rstd[:, None]
    dx = rstd[:, None] * (g - n * (g * n).mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.float()
    return dx.to(h.dtype), (dy.float() * n).sum(0).to(weight.dtype)


class _RmsNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        x2 = _rows(x)
        r2 = None if residual is None else _rows(residual)
        if x.is_cuda:
            launches.add(1)
            y, h, rstd, _ = require_extension().rms_norm_fwd(x2, r2, weight.contiguous(), eps, False, True)
        else:
            y, h = (reference_rms_norm(x2, weight, None, eps), None) if r2 is None else \
                reference_rms_norm(x2, weight, r2, eps)
            rstd = ((x2 if h is None else h).float().square().mean(-1) + eps).rsqrt()
        ctx.save_for_backward(x2 if h is None else h, weight, rstd)
        ctx.has_residual = residual is not None
        ctx.set_materialize_grads(False)
        return y.view(x.shape) if h is None else (y.view(x.shape), h.view(x.shape))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        shape = (dy if dy is not None else dh).shape if (dy is not None or dh is not None) else None
        if shape is None:
            return None, None, None, None
        if dy is None:    # only the residual stream was used
            return dh, None, dh if ctx.has_residual else None, None
        dy = dy.reshape(h.shape).to(h.dtype).contiguous()
        dh = None if dh is None else dh.reshape(h.shape).to(h.dtype).contiguous()
        if h.is_cuda:
            launches.add(2)
            dx, dw = require_extension().rms_norm_bwd(dy, dh, h, weight.contiguous(), rstd)
        else:
            dx, dw = reference_rms_norm_grad(dy, dh, h, weight, rstd)
        dx = dx.view(shape)
        return dx, dw, dx if ctx.has_residual else None, None


def rms_norm(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-6):
    """RMS norm of the last dimension of `x`; with a residual, ``(y, h)`` (see
    the module docstring)."""
    _check(x, weight, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return _RmsNormFn.apply(x, weight, residual, float(eps))
    if not x.is_cuda:
        return reference_rms_norm(x, weight, residual, eps)
    launches.add(1)
    y, h, _, _ = require_extension().rms_norm_fwd(_rows(x), None if residual is None else _rows(residual),
                                                  weight.contiguous(), float(eps), False, False)
    return y.view(x.shape) if h is None else (y.view(x.shape), h.view(x.shape))


def rms_norm_fp8(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-6):
    """RMS norm with an 8-bit result: ``(q, scale)``, or ``(q, scale, h)`` with
    a residual. q [..., D] is e4m3 (its rows start 16 bytes apart), scale
    [..., ceil(D / 128)] fp32; ``ops.fp8.dequantize_rows`` gives the values."""
    _check(x, weight, residual)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (x, weight, residual)):
        raise ValueError("rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    lead = x.shape[:-1]
    if not x.is_cuda:
        from .fp8 import reference_quantize_rows
        h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
        hf = h.float()
        y = hf * (hf.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.float()
        q, scale = reference_quantize_rows(y.reshape(-1, x.shape[-1]))
    else:
        launches.add(1)
        q, h, _, scale = require_extension().rms_norm_fwd(_rows(x), None if residual is None else _rows(residual),
                                                          weight.contiguous(), float(eps), True, False)
    q, scale = from_rows(q, lead), from_rows(scale, lead)
    return (q, scale) if residual is None else (q, scale, h.view(x.shape))


class FusedRMSNorm(nn.RMSNorm):
    """``nn.RMSNorm`` over one dimension on the fused kernels (same parameter
    and state-dict key). ``forward(x, residual)`` returns ``(norm(x + residual),
    x + residual)``."""

    def __init__(self, dim: int, eps: float = 1e-6, device=None, dtype=None):
        super().__init__(dim, eps=eps, elementwise_affine=True, device=device, dtype=dtype)

    def forward(self, x: Tensor, residual: Tensor | None = None):
        return rms_norm(x, self.weight, residual, self.eps)
