"""Log-probabilities of given tokens (or actions) under masked logits, with the
entropy of each row's distribution and its most probable alternatives, on
fused sm_100a kernels (``csrc/token_logprobs.cu``).

``token_log_probs(logits, tokens, mask=None, temperature=1., top=0)`` takes
logits [..., V] (fp32, bf16 or fp16), tokens [...] and an optional boolean mask
of the valid entries that broadcasts against the logits, and returns
``TokenLogProbs(log_prob, entropy, top_log_prob, top_token)``:

* the distribution is the softmax of logits / temperature over the valid
  entries; masked entries are not read, whatever they hold;
* ``log_prob`` [...] and ``entropy`` [...] are fp32 and differentiable with
  respect to the logits; the log-probability of a masked token is -inf;
* ``top_log_prob`` / ``top_token`` [..., top] are the ``top`` (at most 64) most
  probable entries, equal ones by their index (on CUDA all values below fp32's
  normal range, 2^-126, equal zero), without gradient; where a row has fewer entries of positive probability they are -inf and -1;
* a negative token marks a row to be ignored: log_prob 0, no gradient from it
  (its entropy and alternatives are given all the same); a token beyond the
  last entry gives NaN;
* a row whose mask leaves nothing has log_prob -inf, entropy 0 and no
  gradient; a NaN or +inf among a row's valid entries makes it NaN.

On CPU the same values are computed in plain PyTorch.
"""
from __future__ import annotations

from typing import NamedTuple

import torch
from torch import Tensor
from torch.autograd.function import once_differentiable

from .ext import require_extension

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
MAX_TOP = 64


class TokenLogProbs(NamedTuple):
    log_prob: Tensor
    entropy: Tensor
    top_log_prob: Tensor
    top_token: Tensor


def _reference_parts(logits: Tensor, mask: Tensor | None, temperature: float):
    """(log-probabilities of all entries, probabilities, entropy, rows without an entry) in fp32 (fp64 for fp64)."""
    z = (logits.double() if logits.dtype == torch.float64 else logits.float()) / temperature
    if mask is not None:
        z = torch.where(mask, z, -torch.inf)
    m = z.amax(-1, keepdim=True)
    empty = m == -torch.inf
    m = torch.where(empty, 0., m)
    e = torch.exp(z - m)
    total = torch.where(empty, 1., e.sum(-1, keepdim=True))
    log_p = z - m - torch.log(total)
    p = e / total
    entropy = -torch.where(p == 0, 0., p * log_p).sum(-1, keepdim=True)
    return log_p, p, entropy, empty


def reference_token_log_probs(logits: Tensor, tokens: Tensor, mask: Tensor | None = None, temperature: float = 1.,
                              top: int = 0) -> TokenLogProbs:
    """The same operation on rows [R, V] in plain PyTorch (CPU path and test
    oracle), without gradient."""
    v = logits.shape[-1]
    log_p, p, entropy, empty = _reference_parts(logits, mask, temperature)
    t = tokens[:, None]
    lp = torch.where(empty, -torch.inf, log_p.gather(1, t.clamp(0, v - 1)))
    lp = torch.where(t < 0, 0., torch.where(t >= v, torch.nan, lp))
    order = logits if mask is None else torch.where(mask, logits, -torch.inf)
    order = torch.where(torch.isnan(order), -torch.inf, order)
    value, index = torch.sort(order, dim=-1, descending=True, stable=True)
    value, index = value[:, :top], index[:, :top]
    none = value == -torch.inf
    best = torch.where(none, -torch.inf, log_p.gather(1, index))
    index = torch.where(none, -1, index)
    pad = top - index.shape[1]
    best = torch.nn.functional.pad(best, (0, pad), value=-torch.inf)
    index = torch.nn.functional.pad(index, (0, pad), value=-1)
    return TokenLogProbs(lp[:, 0], entropy[:, 0], best, index)


def reference_token_log_probs_grad(logits: Tensor, tokens: Tensor, mask: Tensor | None, temperature: float,
                                   g_log_prob: Tensor | None, g_entropy: Tensor | None) -> Tensor:
    """Gradient of the log-probabilities and entropies of rows [R, V], in the
    precision of ``reference_token_log_probs``."""
    v = logits.shape[-1]
    log_p, p, entropy, empty = _reference_parts(logits, mask, temperature)
    counts = ((tokens >= 0) & (tokens < v))[:, None]
    gl = torch.zeros_like(entropy) if g_log_prob is None else torch.where(counts, g_log_prob[:, None].to(p.dtype), 0.)
    ge = torch.zeros_like(entropy) if g_entropy is None else g_entropy[:, None].to(p.dtype)
    d = torch.where(p == 0, 0., p * (-gl - ge * (log_p + entropy)))
    d = d.scatter_add(1, tokens[:, None].clamp(0, v - 1), gl) / temperature
    dead = empty if mask is None else empty | ~mask
    return torch.where(dead, 0., d)


class _TokenLogProbsCpuFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, mask, temperature, top):
        lp, ent, tv, tt = reference_token_log_probs(logits, tokens, mask, temperature, top)
        ctx.save_for_backward(logits, tokens, mask)
        ctx.temperature = temperature
        ctx.mark_non_differentiable(tv, tt)
        ctx.set_materialize_grads(False)
        return lp, ent, tv, tt

    @staticmethod
    @once_differentiable
    def backward(ctx, g_lp, g_ent, _tv, _tt):
        if g_lp is None and g_ent is None:
            return None, None, None, None, None
        logits, tokens, mask = ctx.saved_tensors
        dx = reference_token_log_probs_grad(logits, tokens, mask, ctx.temperature, g_lp, g_ent)
        return dx.to(logits.dtype), None, None, None, None


def token_log_probs(logits: Tensor, tokens: Tensor, mask: Tensor | None = None, temperature: float = 1.,
                    top: int = 0) -> TokenLogProbs:
    """Log-probabilities of `tokens`, entropies and alternatives of the rows of
    `logits` (see the module docstring)."""
    if logits.is_cuda:
        return TokenLogProbs._make(require_extension().token_log_probs(logits, tokens, mask, temperature, top))
    if logits.dim() < 1 or logits.shape[-1] < 1 or logits.dtype not in DTYPES:
        raise ValueError("token_log_probs takes fp32, bf16 or fp16 logits [..., V]")
    lead, v = logits.shape[:-1], logits.shape[-1]
    if tokens.shape != lead or tokens.dtype not in (torch.int64, torch.int32) or tokens.device != logits.device:
        raise ValueError(f"token_log_probs needs integer tokens {tuple(lead)} on {logits.device}")
    if not 1e-30 <= temperature <= 1e30:
        raise ValueError(f"the temperature must be in 1e-30..1e30, not {temperature}")
    if not 0 <= top <= MAX_TOP:
        raise ValueError(f"top must be in 0..{MAX_TOP}, not {top}")
    if mask is not None:
        if mask.dtype != torch.bool or mask.device != logits.device:
            raise ValueError("the mask must be boolean (true: valid) on the logits' device")
        try:
            mask = mask.expand(logits.shape).reshape(-1, v)
        except RuntimeError as exc:
            raise ValueError(f"the mask {tuple(mask.shape)} does not broadcast to {tuple(logits.shape)}") from exc
    lp, ent, tv, tt = _TokenLogProbsCpuFn.apply(logits.reshape(-1, v), tokens.reshape(-1).long(), mask, float(temperature),
                                                int(top))
    return TokenLogProbs(lp.view(lead), ent.view(lead), tv.view(*lead, top), tt.view(*lead, top))
