"""The language-model operators have no forward-mode derivatives: a dual tensor
is refused on either device, never answered without its tangent (which would
count as a zero derivative)."""
import pytest
import torch
from torch.autograd import forward_ad

from autodrive_b200.ops.fp8 import FrozenFp8Linear, fp8_linear, fp8_matmul, quantize_blocks, quantize_rows
from autodrive_b200.ops.rmsnorm import rms_norm, rms_norm_fp8
from autodrive_b200.ops.token_logprobs import token_log_probs

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _dual(t):
    return forward_ad.make_dual(t, torch.ones_like(t))


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("device", DEVICES)
def test_dual_tensors_are_refused(device, grad):
    x, w, b = torch.randn(4, 256, device=device), torch.randn(256, device=device), torch.randn(130, 256, device=device)
    t = torch.zeros(4, dtype=torch.long, device=device)
    with forward_ad.dual_level(), torch.set_grad_enabled(grad):
        for call in (lambda: rms_norm(_dual(x), w), lambda: rms_norm(x, _dual(w)), lambda: rms_norm(x, w, _dual(x)),
                     lambda: token_log_probs(_dual(x), t), lambda: token_log_probs(_dual(x), t, top=2),
                     lambda: fp8_linear(_dual(x), b), lambda: fp8_linear(x, _dual(b)),
                     lambda: fp8_linear(x, b, _dual(torch.zeros(130, device=device)))):
            with pytest.raises(NotImplementedError):
                call()


@pytest.mark.parametrize("device", DEVICES)
def test_operators_without_gradient_refuse_dual_tensors(device):
    x, w = torch.randn(4, 256, device=device), torch.randn(256, device=device)
    q, s = quantize_rows(x)
    wq, ws = quantize_blocks(torch.randn(130, 256, device=device))
    layer = FrozenFp8Linear(torch.randn(130, 256, device=device))
    with forward_ad.dual_level(), torch.no_grad():
        for call in (lambda: rms_norm_fp8(_dual(x), w), lambda: rms_norm_fp8(x, _dual(w)),
                     lambda: rms_norm_fp8(x, w, _dual(x)), lambda: fp8_matmul(q, _dual(s), wq, ws),
                     lambda: fp8_matmul(q, s, wq, _dual(ws)),
                     lambda: fp8_matmul(q, s, wq, ws, _dual(torch.zeros(130, device=device))), lambda: layer(_dual(x))):
            with pytest.raises(ValueError):
                call()
    # no tangent, no refusal
    with forward_ad.dual_level():
        assert rms_norm(x, w).shape == x.shape and token_log_probs(x, torch.zeros(4, dtype=torch.long, device=device)).log_prob.shape == (4,)
