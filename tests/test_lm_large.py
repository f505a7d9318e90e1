"""Tensors of more than 2^31 elements, whose last rows lie behind every 32-bit
offset: rows at both ends and beside the 2^31st element. Norms, quantised rows
and products work on a row in the same way wherever it lies, so they equal, bit
for bit, the same rows alone, which other sizes test against 64 bits."""
import pytest
import torch

from autodrive_b200.ops.fp8 import fp8_matmul, quantize_blocks, quantize_rows
from autodrive_b200.ops.rmsnorm import rms_norm, rms_norm_fp8
from autodrive_b200.ops.tc_linear import check_gemm_status
from autodrive_b200.ops.token_logprobs import TokenLogProbs, token_log_probs

from test_token_logprobs import _check, _check_grad

pytestmark = pytest.mark.gpu


def _rows(n, width):
    """Rows at the ends and around element 2^31 (and 2^32, where there is one)."""
    at = {0, 1, n - 2, n - 1}
    for e in (1 << 31, 1 << 32):
        at |= {r for r in range(e // width - 1, e // width + 2) if r < n}
    return torch.tensor(sorted(at), device="cuda")


def _bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.fixture(autouse=True)
def _room():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


@pytest.mark.parametrize("d", [1000, 1001])
def test_norm(d):
    n = (1 << 31) // d + 300
    x = torch.empty(n, d, dtype=torch.bfloat16, device="cuda").normal_()
    w = torch.rand(d, device="cuda") + .5
    at = _rows(n, d)
    y, h = rms_norm(x, w, x)
    y1, h1 = rms_norm(x[at], w, x[at])
    assert torch.equal(y[at], y1) and torch.equal(h[at], h1)
    del y, h
    q, s = rms_norm_fp8(x, w)
    q1, s1 = rms_norm_fp8(x[at], w)
    assert torch.equal(_bits(q.view(torch.uint8)[at]), _bits(q1)) and torch.equal(s[at], s1)
    del q, s
    x.requires_grad_(True)
    y = rms_norm(x, w)
    dx, = torch.autograd.grad(y, x, x.detach())
    x1 = x.detach()[at].requires_grad_(True)
    dx1, = torch.autograd.grad(rms_norm(x1, w), x1, x1.detach())
    assert torch.equal(dx[at], dx1)


def test_quantised_rows_and_product():
    n, k, m = (1 << 31) // 640 + 300, 640, 700
    x = torch.empty(n, k, dtype=torch.bfloat16, device="cuda").normal_()
    at = _rows(n, k)
    q, s = quantize_rows(x)
    q1, s1 = quantize_rows(x[at])
    assert torch.equal(_bits(q.view(torch.uint8)[at]), _bits(q1)) and torch.equal(s[at], s1)
    b, b_s = quantize_blocks(torch.randn(m, k, device="cuda"))
    del x
    y = fp8_matmul(q, s, b, b_s)
    at = torch.cat((at, _rows(n, m)))
    few = torch.cat((at, torch.arange(5000, device="cuda")))   # as many rows as keep the kernel
    y1 = fp8_matmul(q.view(torch.uint8)[few].view(torch.float8_e4m3fn), s[few], b, b_s)
    check_gemm_status()
    assert torch.equal(y[at], y1[:len(at)])


@pytest.mark.parametrize("v", [1000, 16001])
@pytest.mark.parametrize("mask", [False, True])
def test_scores(v, mask):
    """Against 64 bits, with the tolerances derived in test_token_logprobs.py: a row of 16001 starts 2 r bytes behind a
    16-byte boundary, where r is its number modulo eight, and is cut into vectors, and added up, from that boundary."""
    n = (1 << 31) // v + 300
    x = torch.empty(n, v, dtype=torch.bfloat16, device="cuda").normal_().requires_grad_(True)
    t = torch.randint(v, (n,), device="cuda")
    m = None
    if mask:
        m = torch.empty(n, v, dtype=torch.uint8, device="cuda").random_(0, 4).bool()
    at = torch.cat((_rows(n, v), torch.arange(600, device="cuda")))
    r = token_log_probs(x, t, m, top=3)
    x1, t1, m1 = x.detach()[at], t[at], None if m is None else m[at]
    _check(x1, t1, m1, 1., 3, TokenLogProbs(*(o.detach()[at] for o in r)))
    one = torch.ones(n, device="cuda")
    dx, = torch.autograd.grad((r.log_prob, r.entropy), x, (one, one))
    _check_grad(x1, t1, m1, 1., one[:len(at)], one[:len(at)], dx[at])
