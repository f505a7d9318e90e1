"""The status word that the tensor-core kernels of a device share: who makes it,
who clears it and who reads it."""
import pytest
import torch

from autodrive_b200.ops import tc_linear
from autodrive_b200.ops.fp8 import fp8_linear, fp8_matmul, quantize_blocks, quantize_rows
from autodrive_b200.ops.tc_linear import TensorCoreTimeout, check_gemm_status, gemm

pytestmark = pytest.mark.gpu


@pytest.fixture
def fresh(monkeypatch):
    """As in a process that has made no tensor-core call yet."""
    monkeypatch.setattr(tc_linear._Status, "_state", {})


def _operands():
    g = torch.Generator(device="cuda").manual_seed(0)
    x = torch.randn(40, 256, device="cuda", generator=g).bfloat16().requires_grad_(True)
    w = torch.randn(130, 256, device="cuda", generator=g).requires_grad_(True)
    return x, w


def _quantised():
    x, w = _operands()
    return (*quantize_rows(x), *quantize_blocks(w))


def test_first_call_in_inference_mode(fresh):
    """Training and polling go on as after any other first call."""
    with torch.inference_mode():
        fp8_matmul(*_quantised())
    x, w = _operands()
    fp8_linear(x, w).sum().backward()
    assert x.grad is not None and w.grad is not None
    with pytest.raises(TensorCoreTimeout):
        fp8_matmul(*_quantised(), wait_ns=0)
        check_gemm_status()
    check_gemm_status()


def test_a_cleared_timeout_leaves_pending_backwards_alone():
    x, w = _operands()
    y = fp8_linear(x, w)
    with pytest.raises(TensorCoreTimeout):
        fp8_matmul(*_quantised(), wait_ns=0)
        check_gemm_status()
    y.sum().backward()
    check_gemm_status()
    assert x.grad is not None and w.grad is not None


def test_first_call_inside_a_capture(fresh):
    """The word lies outside the graph's memory: replays leave it alone, and a replayed call's failure is reported."""
    ops = _quantised()
    x, w = _operands()
    xb, wb = x.detach(), w.detach().bfloat16()
    want, want2 = fp8_matmul(*ops), gemm(xb, wb)         # kernels loaded; their word is forgotten below
    torch.cuda.synchronize()
    tc_linear._Status._state.clear()
    graph, bad = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, y2 = fp8_matmul(*ops), gemm(xb, wb)
    check_gemm_status()                                  # nothing has run yet
    for _ in range(3):
        graph.replay()
        check_gemm_status()
        assert torch.equal(y, want) and torch.equal(y2, want2)
    with torch.cuda.graph(bad):
        fp8_matmul(*ops, wait_ns=0)
    bad.replay()
    graph.replay()
    with pytest.raises(TensorCoreTimeout):
        check_gemm_status()
    check_gemm_status()


def test_a_device_without_a_number_is_the_current_one():
    fp8_matmul(*_quantised(), wait_ns=0)
    with pytest.raises(TensorCoreTimeout):
        check_gemm_status("cuda")
    check_gemm_status()


def test_backwards_are_polled(monkeypatch):
    """A wait that runs out is reported by the backwards that follow, as by forwards: the first queues the read-back."""
    monkeypatch.setattr(tc_linear._Status, "poll_every", 1)
    check_gemm_status()
    x, w = _operands()
    first, second = fp8_linear(x, w), fp8_linear(x, w)
    check_gemm_status()
    tc_linear._Status.get(x.device).fill_(2)   # as a kernel would
    first.sum().backward()
    torch.cuda.synchronize()
    with pytest.raises(TensorCoreTimeout, match="stage loaded"):
        second.sum().backward()
    check_gemm_status()
    fp8_linear(x, w).sum().backward()          # and the engine goes on
    check_gemm_status()
