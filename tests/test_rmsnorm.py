"""RMS norm with the residual's addition against the formula in 64 bits.

Tolerances: u is half a step of the output's type (eps / 2), f = 2^-24 that of
fp32. The sum of a row's squares is added in chains of at most 64 terms and a
tree of at most 10 levels, which moves it by less than 80 f and rstd by half
of that; the products after it round three times: y is off by at most
(u + 48 f) |y|. The backward's mean is off by at most 80 f of the mean of its
terms' magnitudes, and dx by u |dx| plus 160 f of the magnitudes of what it
is made of. A weight gradient is a sum over R rows in some order: at most
(R + 64) f of the sum of its terms' magnitudes.
"""
import pytest
import torch
from torch import nn

from autodrive_b200.ops.fp8 import dequantize_rows, reference_quantize_rows
from autodrive_b200.ops.rmsnorm import FusedRMSNorm, rms_norm, rms_norm_fp8

F = 2. ** -24
EPS = 1e-6
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _inputs(rows, d, dtype, device, seed=0, residual=True):
    g = torch.Generator().manual_seed(seed + 1000 * rows + d)
    x = torch.randn(rows, d, generator=g).to(dtype).to(device)
    r = (2 * torch.randn(rows, d, generator=g)).to(dtype).to(device) if residual else None
    w = (1 + .2 * torch.randn(d, generator=g)).to(device)
    return x, r, w


def _oracle(h, w):
    """(rstd, y) in 64 bits of the rows that are normalised."""
    hd = h.double()
    rstd = (hd.square().mean(-1, keepdim=True) + EPS).rsqrt()
    return rstd, hd * rstd * w.double()


def _check_forward(x, r, w, y, h):
    u = torch.finfo(x.dtype).eps / 2
    if r is not None:
        assert torch.equal(h, (x.float() + r.float()).to(x.dtype))
    _, want = _oracle(x if r is None else h, w)
    assert y.dtype == x.dtype and y.shape == x.shape
    tiny = torch.finfo(x.dtype).tiny   # fp16 rounds small values to its smallest steps
    assert ((y.double() - want).abs() <= (u + 48 * F) * want.abs() + tiny * u * 2).all()


def _check_backward(h, w, dy, dh, dx, dw):
    u = torch.finfo(h.dtype).eps / 2
    rstd, _ = _oracle(h, w)
    n, g = h.double() * rstd, dy.double() * w.double()
    want = rstd * (g - n * (g * n).mean(-1, keepdim=True))
    size = rstd * (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True))
    if dh is not None:
        want, size = want + dh.double(), size + dh.double().abs()
    tiny = torch.finfo(h.dtype).tiny
    assert ((dx.double() - want).abs() <= u * want.abs() + 160 * F * size + 2 * u * tiny).all()
    terms = dy.double() * n
    uw = torch.finfo(dw.dtype).eps / 2 if dw.dtype != torch.float32 else 0.
    bound = (h.shape[0] + 64) * F * terms.abs().sum(0) + uw * terms.sum(0).abs()
    assert ((dw.double() - terms.sum(0)).abs() <= bound).all()


def _run(x, r, w):
    x, w = x.clone().requires_grad_(True), w.clone().requires_grad_(True)
    r = None if r is None else r.clone().requires_grad_(True)
    out = rms_norm(x, w, r, eps=EPS)
    y, h = (out, None) if r is None else out
    _check_forward(x.detach(), None if r is None else r.detach(), w.detach(), y.detach(),
                   None if h is None else h.detach())
    g = torch.Generator().manual_seed(7)
    dy = torch.randn(x.shape, generator=g).to(x.dtype).to(x.device)
    dh = None if r is None else torch.randn(x.shape, generator=g).to(x.dtype).to(x.device)
    grads = torch.autograd.grad((y,) if r is None else (y, h), (x, w) if r is None else (x, w, r),
                                (dy,) if r is None else (dy, dh))
    _check_backward((x if h is None else h).detach(), w.detach(), dy, dh, grads[0], grads[1])
    if r is not None:
        assert torch.equal(grads[0], grads[2])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("residual", [False, True])
def test_cpu(dtype, residual):
    _run(*_inputs(5, 37, dtype, "cpu", residual=residual))


def test_module_is_rms_norm_on_cpu():
    ref, fused = nn.RMSNorm(24, eps=EPS), FusedRMSNorm(24, eps=EPS)
    with torch.no_grad():
        ref.weight.uniform_(.5, 1.5)
    fused.load_state_dict(ref.state_dict())
    x, r = torch.randn(3, 4, 24), torch.randn(3, 4, 24)
    assert torch.allclose(fused(x), ref(x), atol=1e-6)
    y, h = fused(x, r)
    assert torch.equal(h, x + r) and torch.allclose(y, ref(h), atol=1e-6)


def _refusals(device):
    x, w = torch.randn(4, 32, device=device), torch.ones(32, device=device)
    with pytest.raises(ValueError):
        rms_norm(x.double(), w)
    with pytest.raises(ValueError):
        rms_norm(x, w[:31])
    with pytest.raises(ValueError):
        rms_norm(x, w, torch.randn(4, 31, device=device))
    with pytest.raises(ValueError):
        rms_norm(x, w, x.bfloat16())
    with pytest.raises(ValueError):
        rms_norm(torch.zeros(4, 0, device=device), w[:0])
    with pytest.raises(ValueError):
        rms_norm(torch.zeros(1, 40000, device=device), torch.ones(40000, device=device))
    with pytest.raises(ValueError):
        rms_norm_fp8(x.requires_grad_(True), w)


def test_refusals_cpu():
    _refusals("cpu")


@pytest.mark.gpu
def test_refusals_gpu():
    _refusals("cuda")
    with pytest.raises(ValueError):
        rms_norm(torch.randn(4, 32, device="cuda"), torch.ones(32))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (1, 256), (9, 256), (301, 257), (17, 512), (5, 1000), (33, 1024),
                                    (1500, 137), (40, 2048), (7, 2056), (13, 4099), (6, 8192), (5, 8200), (3, 16384),
                                    (4, 20001), (2, 32768), (4500, 64)])
@pytest.mark.parametrize("residual", [False, True])
def test_matches_formula(dtype, rows, d, residual):
    _run(*_inputs(rows, d, dtype, "cuda", residual=residual))


@pytest.mark.gpu
@pytest.mark.parametrize("wdtype", TYPES)
def test_weight_types(wdtype):
    x, r, w = _inputs(50, 264, torch.bfloat16, "cuda")
    _run(x, r, w.to(wdtype))


@pytest.mark.gpu
def test_strided_rows_and_leading_dimensions():
    g = torch.Generator(device="cuda").manual_seed(1)
    big = torch.randn(6, 5, 2, 96, device="cuda", generator=g).bfloat16()
    w = torch.ones(96, device="cuda")
    for x in (big[:, :, 0], big[..., 1, 3:60], big.transpose(-1, -2)[..., 0], big[2:4].expand(2, 5, 2, 96)):
        w = torch.rand(x.shape[-1], device="cuda") + .5
        y, h = rms_norm(x, w, x, eps=EPS)
        assert y.shape == x.shape and h.shape == x.shape
        d = x.shape[-1]
        _check_forward(x.reshape(-1, d), x.reshape(-1, d), w, y.reshape(-1, d), h.reshape(-1, d))
    # a base that is not 16-byte aligned
    flat = torch.randn(1 + 4 * 64, device="cuda").bfloat16()
    x = flat[1:].view(4, 64)
    _check_forward(x, None, torch.ones(64, device="cuda"), rms_norm(x, torch.ones(64, device="cuda"), eps=EPS), None)


@pytest.mark.gpu
def test_no_rows_zero_rows_and_non_finite_rows():
    w = torch.ones(48, device="cuda", requires_grad=True)
    x = torch.zeros(0, 48, device="cuda", requires_grad=True)
    y = rms_norm(x, w)
    y.sum().backward()
    assert y.shape == (0, 48) and x.grad.shape == (0, 48) and torch.equal(w.grad, torch.zeros_like(w))
    q, s = rms_norm_fp8(x.detach(), w.detach())
    assert q.shape == (0, 48) and s.shape == (0, 1)
    x = torch.randn(4, 48, device="cuda")
    x[1] = 0.
    x[2, 5] = torch.nan
    y = rms_norm(x, w.detach())
    assert (y[1] == 0).all() and y[2].isnan().all() and y[[0, 3]].isfinite().all()
    q, s = rms_norm_fp8(x, w.detach())
    assert (q[1].float() == 0).all() and s[1, 0] == 2. ** -126 and q[2].float().isnan().all()


@pytest.mark.gpu
def test_only_one_of_the_outputs_is_used():
    x, r, w = _inputs(20, 72, torch.float32, "cuda")
    x.requires_grad_(True), w.requires_grad_(True), r.requires_grad_(True)
    y, h = rms_norm(x, w, r)
    gx, gw, gr = torch.autograd.grad(h.sum(), (x, w, r), allow_unused=True, retain_graph=True)
    assert gw is None and (gx == 1).all() and (gr == 1).all()
    gx, gw = torch.autograd.grad(y, (x, w), torch.ones_like(y))
    _check_backward(h.detach(), w.detach(), torch.ones_like(y), None, gx, gw)


@pytest.mark.gpu
def test_gradient_is_the_difference_quotient():
    """Central differences of the kernel's own fp32 forward: with a step of 2^-6 their truncation is below 1e-3 of the
    second-derivative scale and their rounding 2^-24 * |loss| / 2^-6, both under the 2 % asked for."""
    x, r, w = _inputs(3, 40, torch.float32, "cuda")
    c = torch.randn(3, 40, device="cuda", generator=torch.Generator(device="cuda").manual_seed(3))
    x.requires_grad_(True), w.requires_grad_(True)
    loss = lambda a, b: (rms_norm(a, b, r)[0].double() * c.double()).sum()  # noqa: E731
    gx, gw = torch.autograd.grad(loss(x, w), (x, w))
    step = 2. ** -6
    for i, j in ((0, 0), (1, 17), (2, 39)):
        e = torch.zeros_like(x)
        e[i, j] = step
        with torch.no_grad():
            num = (loss(x + e, w) - loss(x - e, w)) / (2 * step)
            numw = (loss(x, w + e[i]) - loss(x, w - e[i])) / (2 * step)
        assert abs(num - gx[i, j]) <= .02 * gx.abs().max()
        assert abs(numw - gw[j]) <= .02 * gw.abs().max()


def _check_fp8(x, r, w, q, scale, h):
    _, y = _oracle(x if r is None else h, w)
    rows, d = y.shape
    groups = -(-d // 128)
    padded = torch.zeros(rows, groups * 128, dtype=torch.float64, device=x.device)
    padded[:, :d] = y
    amax = padded.view(rows, groups, 128).abs().amax(-1)
    # y is off by 48 f before it is quantised (its own type does not come in), the scale rounds once more
    assert ((scale.double() - amax / 448).abs() <= 50 * F * amax / 448).all()
    # half a step of e4m3: 2^-4 of the value, at least half its smallest step, 2^-10 scales
    got, sc = dequantize_rows(q, scale).double(), scale.double().repeat_interleave(128, 1)[:, :d]
    assert ((got - y).abs() <= torch.maximum(2. ** -4 * y.abs(), 2. ** -10 * sc) + 100 * F * y.abs()).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 128), (5, 129), (9, 256), (301, 257), (5, 1000), (33, 1024), (40, 2048),
                                    (13, 4099), (6, 8192), (4, 20001), (2, 32768)])
@pytest.mark.parametrize("residual", [False, True])
def test_fp8_matches_formula(dtype, rows, d, residual):
    x, r, w = _inputs(rows, d, dtype, "cuda", residual=residual)
    q, scale, *h = rms_norm_fp8(x, w, r, eps=EPS)
    assert q.dtype == torch.float8_e4m3fn and q.stride(0) % 16 == 0 and scale.shape == (rows, -(-d // 128))
    if residual:
        assert torch.equal(h[0], (x.float() + r.float()).to(dtype))
    _check_fp8(x, r, w, q, scale, h[0] if residual else None)


@pytest.mark.gpu
def test_fp8_is_the_quantised_fp32_norm():
    """In fp32 the 8-bit form quantises the very numbers that rms_norm returns."""
    for d in (384, 385):
        x, r, w = _inputs(65, d, torch.float32, "cuda")
        y, h = rms_norm(x, w, r, eps=EPS)
        q, scale, h8 = rms_norm_fp8(x, w, r, eps=EPS)
        wq, ws = reference_quantize_rows(y)
        assert torch.equal(h, h8) and torch.equal(scale, ws) and torch.equal(q.float(), wq.float())


@pytest.mark.gpu
def test_captured_and_replayed():
    x, r, w = _inputs(65, 384, torch.bfloat16, "cuda")
    x.requires_grad_(True), w.requires_grad_(True)
    dy = torch.randn_like(x)

    def step():
        y, h = rms_norm(x, w, r)
        return (y, h, *torch.autograd.grad(y, (x, w), dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(torch.randn_like(x))
    graph.replay()
    want = step()
    for a, b in zip(out, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_changes_in_place_and_second_derivatives_are_refused():
    x, r, w = _inputs(4, 64, torch.float32, "cuda")
    x.requires_grad_(True)
    y, h = rms_norm(x, w, r)
    h.data_ptr()
    with torch.no_grad():
        h += 1.   # the backward would read it
    with pytest.raises(RuntimeError):
        y.sum().backward()
    y = rms_norm(x, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), x, create_graph=True)
