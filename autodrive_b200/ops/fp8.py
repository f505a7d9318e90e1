"""8-bit floating-point products with a scale for each block of 128 on the
sm_100a tensor cores (``csrc/fp8_gemm.cu``, ``csrc/fp8_quant.cu``).

Operands are e4m3 with fp32 scales, a value being its 8-bit number times its
scale:

* rows (activations, gradients): one scale for each row and 128 columns,
  ``quantize_rows(x) -> (q [..., K], scale [..., ceil(K / 128)])``;
* matrices (weights): one scale for each 128 x 128 block,
  ``quantize_blocks(w) -> (q [N, K], scale [ceil(N / 128), ceil(K / 128)])``.

A scale is the largest magnitude of its group divided by 448, rounded to fp32,
and the 8-bit number is the one nearest to the exact quotient. A group that
holds a NaN or an infinity becomes NaN.

``fp8_matmul(a, a_scale, b, b_scale, bias, out_dtype)`` is the product of rows
with a weight matrix, a b^T, with fp32 sums. It has no gradient.

``fp8_linear(x, weight, bias)`` is a linear layer for training: both operands
are quantised on the way in; the backward takes the quantised gradient through
the same quantised weight (rounding counts as the identity), and the weight's
gradient as a product of the unquantised gradient and input with fp32 sums: as
they are where both are bf16 or both fp16, otherwise rounded to bf16 (2^-8 of
each term at most for each of the two).
``Fp8Linear`` is the module (a drop-in ``nn.Linear``, beside ``TcLinear``), and
``FrozenFp8Linear`` the one for acting and serving, which holds 8-bit weights
only. ``freeze_fp8(module)`` swaps a module's linear layers for frozen ones.

On CPU all of them compute the same in plain PyTorch, with fp32 sums in another
order and the weight's gradient from operands of any type as they are. The
product's kernel reports timed-out waits through the status word of the bf16 GEMM
(``ops.tc_linear.check_gemm_status``).
"""
from __future__ import annotations

import torch
from torch import Tensor, nn
from torch.autograd.function import once_differentiable

from .ext import require_extension
from .rmsnorm import from_rows, wants_derivative
from .tc_linear import _result_dtype, _Status

GROUP = 128
E4M3 = torch.float8_e4m3fn
E4M3_MAX = 448.
_MIN_AMAX = E4M3_MAX * 2. ** -126
_INPUTS = (torch.float32, torch.bfloat16, torch.float16)


def _groups(k: int) -> int:
    return (k + GROUP - 1) // GROUP


def _padded_q(values: Tensor) -> Tensor:
    """`values` in storage whose rows start 16 bytes apart."""
    m, k = values.shape
    buf = torch.zeros((m, (k + 15) // 16 * 16), dtype=torch.uint8, device=values.device)
    buf[:, :k] = values.view(torch.uint8)
    return buf.view(E4M3)[:, :k]


def _rows_with_padding(q: Tensor) -> Tensor:
    """The bytes of `q` [M, K] with its rows' padding, as ``_padded_q`` lays them out: a view, or a copy where `q` lies
    otherwise."""
    m, k = q.shape
    ld = (k + 15) // 16 * 16
    if q.stride() != (ld, 1) or q.untyped_storage().nbytes() < q.storage_offset() + m * ld:
        q = _padded_q(q)
    return q.view(torch.uint8).as_strided((m, ld), (ld, 1))


def _round_e4m3(t: Tensor) -> Tensor:
    """The nearest e4m3 number of each fp64 value (ties to even), in fp64."""
    _, exponent = torch.frexp(t)
    step = torch.ldexp(torch.ones_like(t), exponent.clamp_min(-5) - 4)
    return torch.round(t / step) * step


def _scales(amax: Tensor) -> Tensor:
    return (amax.double().clamp_min(_MIN_AMAX) / E4M3_MAX).float()


def reference_quantize_rows(x: Tensor) -> tuple[Tensor, Tensor]:
    """``quantize_rows`` of a matrix in plain PyTorch."""
    m, k = x.shape
    g = _groups(k)
    padded = torch.zeros((m, g * GROUP), dtype=torch.float32, device=x.device)
    padded[:, :k] = x
    padded = padded.view(m, g, GROUP)
    scale = _scales(padded.abs().amax(-1)) if g else padded.new_zeros((m, 0))
    q = _round_e4m3(padded.double() / scale[..., None].double())
    return _padded_q(q.view(m, -1)[:, :k].to(torch.float32).to(E4M3)), scale


def reference_quantize_blocks(w: Tensor) -> tuple[Tensor, Tensor]:
    """``quantize_blocks`` in plain PyTorch."""
    n, k = w.shape
    bn, bk = _groups(n), _groups(k)
    padded = torch.zeros((bn * GROUP, bk * GROUP), dtype=torch.float32, device=w.device)
    padded[:n, :k] = w
    padded = padded.view(bn, GROUP, bk, GROUP)
    scale = _scales(padded.abs().amax((1, 3))) if bn and bk else padded.new_zeros((bn, bk))
    q = _round_e4m3(padded.double() / scale[:, None, :, None].double())
    return _padded_q(q.view(bn * GROUP, bk * GROUP)[:n, :k].to(torch.float32).to(E4M3)), scale


def dequantize_rows(q: Tensor, scale: Tensor) -> Tensor:
    """The fp32 values of quantised rows."""
    return q.float() * scale.repeat_interleave(GROUP, -1)[..., :q.shape[-1]]


def dequantize_blocks(q: Tensor, scale: Tensor) -> Tensor:
    """The fp32 values of a matrix quantised in blocks."""
    n, k = q.shape
    return q.float() * scale.repeat_interleave(GROUP, 0)[:n].repeat_interleave(GROUP, 1)[:, :k]


def _check_input(x: Tensor, dims: int, what: str) -> None:
    if x.dtype not in _INPUTS or x.dim() < dims:
        raise ValueError(f"{what} takes fp32, bf16 or fp16 tensors of at least {dims} dimension(s)")


def quantize_rows(x: Tensor) -> tuple[Tensor, Tensor]:
    """`x` [..., K] as e4m3 with one fp32 scale for each row and 128 columns
    (see the module docstring). No gradient."""
    if x.is_cuda:
        return require_extension().quantize_rows(x)
    _check_input(x, 1, "quantize_rows")
    q, scale = reference_quantize_rows(x.detach().reshape(x.shape[:-1].numel(), x.shape[-1]))
    return from_rows(q, x.shape[:-1]), from_rows(scale, x.shape[:-1])


def quantize_blocks(w: Tensor, transposed: bool = False):
    """`w` [N, K] as e4m3 with one fp32 scale for each 128 x 128 block: (q,
    scale), with `transposed` (q, scale, q^T, scale^T), the transposes being
    matrices of their own. No gradient."""
    if w.is_cuda:
        return require_extension().quantize_blocks(w, transposed)
    _check_input(w, 2, "quantize_blocks")
    if w.dim() != 2:
        raise ValueError("quantize_blocks takes a matrix")
    q, scale = reference_quantize_blocks(w.detach())
    return (q, scale, _padded_q(q.view(torch.uint8).t().view(E4M3)), scale.t().contiguous()) if transposed \
        else (q, scale)


def reference_fp8_matmul(a: Tensor, a_scale: Tensor, b: Tensor, b_scale: Tensor, bias: Tensor | None = None,
                         out_dtype: torch.dtype = torch.bfloat16) -> Tensor:
    """``fp8_matmul`` of matrices in plain fp32 PyTorch."""
    y = dequantize_rows(a, a_scale) @ dequantize_blocks(b, b_scale).t()
    return (y if bias is None else y + bias.float()).to(out_dtype)


def fp8_matmul(a: Tensor, a_scale: Tensor, b: Tensor, b_scale: Tensor, bias: Tensor | None = None,
               out_dtype: torch.dtype = torch.bfloat16, wait_ns: int = 2_000_000_000) -> Tensor:
    """a b^T of quantised rows `a` [..., K] and a quantised matrix `b` [N, K]
    with their scales, plus `bias` [N]: [..., N] in `out_dtype` (fp32, bf16 or
    fp16). The product of a row's scale and a block's is taken in fp32: below
    its normal range, 2^-126, it counts as zero, beyond its end as infinite.
    `wait_ns` bounds every pipeline wait inside the kernel."""
    if a.is_cuda:
        y = require_extension().fp8_matmul(a, a_scale, b, b_scale, bias, out_dtype, _Status.get(a.device), wait_ns)
        _Status.after_launch(a.device)
        return y
    if a.dtype != E4M3 or b.dtype != E4M3 or a.dim() < 1 or b.dim() != 2:
        raise ValueError("fp8_matmul takes e4m3 rows [..., K] and an e4m3 matrix [N, K]")
    k, n, lead = a.shape[-1], b.shape[0], a.shape[:-1]
    if b.shape[1] != k:
        raise ValueError(f"fp8_matmul: a has {k} columns and b {b.shape[1]}")
    if a_scale.shape != (*lead, _groups(k)) or b_scale.shape != (_groups(n), _groups(k)):
        raise ValueError(f"fp8_matmul needs scales {(*lead, _groups(k))} and {(_groups(n), _groups(k))}, "
                         f"not {tuple(a_scale.shape)} and {tuple(b_scale.shape)}")
    if a_scale.dtype != torch.float32 or b_scale.dtype != torch.float32:
        raise ValueError("fp8_matmul needs fp32 scales")
    if bias is not None and bias.shape != (n,):
        raise ValueError(f"fp8_matmul needs a bias [{n}]")
    if out_dtype not in _INPUTS:
        raise ValueError("fp8_matmul gives fp32, bf16 or fp16")
    if any(t is not None and t.device != a.device for t in (a_scale, b, b_scale, bias)):
        raise ValueError("fp8_matmul needs all of its tensors on one device")
    if wants_derivative(a, a_scale, b, b_scale, bias):
        raise ValueError("fp8_matmul has no gradient: use fp8_linear, or call it under torch.no_grad()")
    rows = lead.numel()
    return reference_fp8_matmul(a.reshape(rows, k), a_scale.reshape(rows, _groups(k)), b, b_scale, bias,
                                out_dtype).view(*lead, n)


class _Fp8LinearCpuFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias):
        x2 = x.reshape(x.shape[:-1].numel(), x.shape[-1])
        wq, ws = reference_quantize_blocks(weight)
        y = reference_fp8_matmul(*reference_quantize_rows(x2), wq, ws, bias, x.dtype)
        ctx.save_for_backward(x, wq, ws)
        ctx.meta = (weight.dtype, None if bias is None else bias.dtype)
        return y.view(*x.shape[:-1], weight.shape[0])

    @staticmethod
    @once_differentiable
    def backward(ctx, gy):
        x, wq, ws = ctx.saved_tensors
        w_dtype, b_dtype = ctx.meta
        n, k = wq.shape
        g, gx, gw, gb = gy.reshape(-1, n), None, None, None
        if ctx.needs_input_grad[0]:
            gx = (dequantize_rows(*reference_quantize_rows(g)) @ dequantize_blocks(wq, ws)).to(x.dtype).view(x.shape)
        if ctx.needs_input_grad[1]:
            gw = (g.float().t() @ x.reshape(-1, k).float()).to(w_dtype)
        if ctx.needs_input_grad[2]:
            gb = g.sum(0, dtype=torch.float32).to(b_dtype)
        return gx, gw, gb


def fp8_linear(x: Tensor, weight: Tensor, bias: Tensor | None = None) -> Tensor:
    """x weight^T + bias with both operands quantised to e4m3 (see the module
    docstring), with autograd. The result has x's dtype, or the autocast dtype
    inside a CUDA autocast region."""
    if x.is_cuda:
        y = require_extension().fp8_linear(x, weight, bias, _result_dtype(x), _Status.get(x.device))
        _Status.after_launch(x.device)
        return y
    _check_input(x, 1, "fp8_linear")
    _check_input(weight, 2, "fp8_linear")
    if weight.dim() != 2 or x.shape[-1] != weight.shape[1] or (bias is not None and bias.shape != weight.shape[:1]):
        raise ValueError(f"fp8_linear: x {tuple(x.shape)}, weight {tuple(weight.shape)} and bias do not fit")
    if any(t is not None and t.device != x.device for t in (weight, bias)):
        raise ValueError("fp8_linear needs all of its tensors on one device")
    return _Fp8LinearCpuFn.apply(x, weight, bias)


class Fp8Linear(nn.Linear):
    """nn.Linear whose products run in 8 bits; its parameters stay as they are
    (fp32 masters) and are quantised by every call."""

    def forward(self, x: Tensor) -> Tensor:
        return fp8_linear(x, self.weight, self.bias)


class FrozenFp8Linear(nn.Module):
    """A linear layer that holds its weight in 8 bits (buffers ``weight_q``,
    ``weight_scale`` and ``bias``): for acting and serving, no gradient."""

    def __init__(self, weight: Tensor, bias: Tensor | None = None):
        super().__init__()
        q, scale = quantize_blocks(weight)
        self.out_features, self.in_features = weight.shape
        self.register_buffer("weight_q", q)
        self.register_buffer("weight_scale", scale)
        self.register_buffer("bias", None if bias is None else bias.detach().float().clone())

    def _apply(self, fn, recurse=True):
        """What is done to the tensors of a module (moved, shared, emptied, converted) is done to the buffers' bits, so
        that they keep their types and layout: ``half()`` or ``to(dtype)`` of a network change its other layers, not the
        8-bit numbers and their scales."""
        for name, t in self._buffers.items():
            if t is None:
                continue
            bits = _rows_with_padding(t) if name == "weight_q" else t.view(torch.int32)
            moved = fn(bits)
            if moved.dtype != bits.dtype:   # type(dst) converts whole numbers, too
                moved = bits.to(moved.device)
            if moved is not bits:
                self._buffers[name] = moved.view(E4M3)[:, :t.shape[1]] if name == "weight_q" else moved.view(t.dtype)
        return self

    @classmethod
    def from_linear(cls, linear: nn.Linear) -> "FrozenFp8Linear":
        return cls(linear.weight, linear.bias)

    def forward(self, x: Tensor) -> Tensor:
        if wants_derivative(x):
            raise ValueError("FrozenFp8Linear has no gradient: call it under torch.no_grad()")
        xq, xs = quantize_rows(x)
        return fp8_matmul(xq, xs, self.weight_q, self.weight_scale, self.bias, _result_dtype(x))


_FORWARD_HOOKS = ("_forward_hooks", "_forward_hooks_with_kwargs", "_forward_hooks_always_called", "_forward_pre_hooks",
                  "_forward_pre_hooks_with_kwargs")


def freeze_fp8(module: nn.Module, min_features: int = GROUP) -> nn.Module:
    """Replace, in place, every plain nn.Linear of `module` (recursively) whose
    two widths are at least `min_features` with a FrozenFp8Linear of its
    current weight: narrower layers, such as the policy heads, are not bound
    by their weights and keep their precision. Layers that ``tensorize`` has
    put on the bf16 GEMM stay as they are (a policy to be frozen is built with
    ``tensor_cores=False``), and so do those of an nn.TransformerEncoderLayer,
    which reads their weights itself. Forward hooks go with their layers.
    Returns the module, or the frozen layer where the module itself is such a layer."""
    return _freeze(module, min_features, {})


def _freeze(module: nn.Module, min_features: int, done: dict) -> nn.Module:
    """`done`: what has become of each module so far (one may stand in several places)."""
    if module not in done:
        done[module] = module
        if type(module) in (nn.Linear, Fp8Linear):
            if min(module.in_features, module.out_features) >= min_features:
                frozen = done[module] = FrozenFp8Linear.from_linear(module)
                frozen.training = module.training
                for hooks in _FORWARD_HOOKS:   # the same dictionaries, so that their handles still remove them
                    setattr(frozen, hooks, getattr(module, hooks))
        elif not isinstance(module, nn.TransformerEncoderLayer):
            for name, child in list(module._modules.items()):
                if child is not None and _freeze(child, min_features, done) is not child:
                    setattr(module, name, done[child])
    return done[module]
