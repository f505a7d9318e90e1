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
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from .ext import require_extension

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_WIDTH = 32768


def wants_derivative(*tensors: Tensor | None) -> bool:
    """Whether a derivative of what is computed from `tensors` would be expected, in reverse or forward mode."""
    return any(t is not None and (torch.is_grad_enabled() and t.requires_grad or
                                  forward_ad.unpack_dual(t).tangent is not None) for t in tensors)


def _check(x: Tensor, weight: Tensor, residual: Tensor | None) -> None:
    if x.dim() < 1 or x.dtype not in DTYPES:
        raise ValueError("rms_norm takes fp32, bf16 or fp16 rows")
    if not 1 <= x.shape[-1] <= MAX_WIDTH:
        raise ValueError(f"rms_norm rows are 1 to {MAX_WIDTH} wide, not {x.shape[-1]}")
    if weight.shape != x.shape[-1:] or weight.dtype not in DTYPES or weight.device != x.device:
        raise ValueError(f"rms_norm needs an fp32, bf16 or fp16 weight [{x.shape[-1]}] on {x.device}")
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError("rms_norm needs a residual of x's shape, dtype and device")


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


class _RmsNormCpuFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, residual, eps):
        x2, r2 = (None if t is None else t.reshape(-1, t.shape[-1]) for t in (x, residual))
        y, h = (reference_rms_norm(x2, weight, None, eps), None) if r2 is None else \
            reference_rms_norm(x2, weight, r2, eps)
        n = x2 if h is None else h
        ctx.save_for_backward(n, weight, (n.float().square().mean(-1) + eps).rsqrt())
        ctx.set_materialize_grads(False)
        return y.view(x.shape) if h is None else (y.view(x.shape), h.view(x.shape))

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, *dh):
        h, weight, rstd = ctx.saved_tensors
        dx, dw = dh[0] if dh else None, None
        if dy is not None:
            dx, dw = reference_rms_norm_grad(dy.reshape(h.shape), None if dx is None else dx.reshape(h.shape), h, weight,
                                             rstd)
            dx = dx.view(dy.shape)
        return dx, dw, dx if dh else None, None


def rms_norm(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-6):
    """RMS norm of the last dimension of `x`; with a residual, ``(y, h)`` (see
    the module docstring)."""
    if x.is_cuda:
        return require_extension().rms_norm(x, weight, residual, eps)
    _check(x, weight, residual)
    return _RmsNormCpuFn.apply(x, weight, residual, eps)


def rms_norm_fp8(x: Tensor, weight: Tensor, residual: Tensor | None = None, eps: float = 1e-6):
    """RMS norm with an 8-bit result: ``(q, scale)``, or ``(q, scale, h)`` with
    a residual. q [..., D] is e4m3 (its rows start 16 bytes apart), scale
    [..., ceil(D / 128)] fp32; ``ops.fp8.dequantize_rows`` gives the values."""
    if x.is_cuda:
        return require_extension().rms_norm_fp8(x, weight, residual, eps)
    _check(x, weight, residual)
    if wants_derivative(x, weight, residual):
        raise ValueError("rms_norm_fp8 has no gradient: call it under torch.no_grad()")
    from .fp8 import reference_quantize_rows
    h = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    hf = h.float()
    y = hf * (hf.square().mean(-1, keepdim=True) + eps).rsqrt() * weight.float()
    q, scale = (from_rows(t, x.shape[:-1]) for t in reference_quantize_rows(y.reshape(-1, x.shape[-1])))
    return (q, scale) if residual is None else (q, scale, h)


class FusedRMSNorm(nn.RMSNorm):
    """``nn.RMSNorm`` over one dimension on the fused kernels (same parameter
    and state-dict key). ``forward(x, residual)`` returns ``(norm(x + residual),
    x + residual)``."""

    def __init__(self, dim: int, eps: float = 1e-6, device=None, dtype=None):
        super().__init__(dim, eps=eps, elementwise_affine=True, device=device, dtype=dtype)

    def forward(self, x: Tensor, residual: Tensor | None = None):
        return rms_norm(x, self.weight, residual, self.eps)
