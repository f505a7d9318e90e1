"""8-bit products with a scale for each block of 128 against 64-bit arithmetic.

Quantisation is exact: values and scales equal the plain implementation's bit
for bit. A product of K columns is a sum of K exact terms; whichever order and
whether the adders round or truncate, fp32 sums are off by at most (K + 8)
times 2^-23 of the sum of the terms' magnitudes, to which the rounding to the
output's type adds eps / 2 of the result.
"""
import pytest
import torch
from torch import nn

from autodrive_b200.ops import fp8
from autodrive_b200.ops.fp8 import (Fp8Linear, FrozenFp8Linear, dequantize_blocks, dequantize_rows, fp8_linear, fp8_matmul,
                                    freeze_fp8, quantize_blocks, quantize_rows, reference_quantize_blocks,
                                    reference_quantize_rows)
from autodrive_b200.ops.tc_linear import TensorCoreTimeout, check_gemm_status

E = 2. ** -23
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _values(rows, k, seed, dtype=torch.float32, device="cpu"):
    g = _gen(seed)
    x = torch.randn(rows, k, generator=g) * (.7 * torch.randn(rows, 1, generator=g)).exp()
    return x.to(dtype).to(device)


def _slow_e4m3():
    """All finite e4m3 magnitudes with their bits."""
    v = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    return v


def test_reference_rounds_to_the_nearest_e4m3():
    table = _slow_e4m3()
    x = torch.cat((torch.rand(3000, generator=_gen(0), dtype=torch.float64) * 448, table, (table[1:] + table[:-1]) / 2,
                   torch.rand(300, generator=_gen(1), dtype=torch.float64) * 2 ** -6))
    got = fp8._round_e4m3(x)
    dist = (x[:, None] - table).abs()
    best = dist.amin(1)
    assert torch.equal((x - got).abs(), best)
    # ties go to the even code
    tie = (dist == best[:, None]).sum(1) == 2
    code = got.float().to(torch.float8_e4m3fn).view(torch.uint8)
    assert tie.sum() >= 126 and (code[tie] % 2 == 0).all()


def test_cpu_linear_and_frozen_agree_with_dequantised_products():
    x, w = _values(6, 200, 0), _values(130, 200, 1)
    b = torch.randn(130, generator=_gen(2))
    x.requires_grad_(True), w.requires_grad_(True), b.requires_grad_(True)
    y = fp8_linear(x.view(2, 3, 200), w, b)
    xd, wd = dequantize_rows(*reference_quantize_rows(x.detach())), dequantize_blocks(*reference_quantize_blocks(w.detach()))
    want = xd.double() @ wd.double().t() + b.double()
    assert y.shape == (2, 3, 130)
    assert ((y.view(6, 130) - want).abs() <= 210 * E * (xd.abs().double() @ wd.abs().double().t() + b.abs())).all()
    dy = torch.randn(6, 130, generator=_gen(3))
    y.backward(dy.view(2, 3, 130))
    gd = dequantize_rows(*reference_quantize_rows(dy))
    assert torch.allclose(x.grad, gd @ wd, atol=1e-4) and torch.allclose(w.grad, dy.t() @ x.detach(), atol=1e-4)
    assert torch.allclose(b.grad, dy.sum(0), atol=1e-5)
    lin = Fp8Linear(200, 130)
    with torch.no_grad():
        lin.weight.copy_(w), lin.bias.copy_(b)
        assert torch.equal(FrozenFp8Linear.from_linear(lin)(x), lin(x))


def test_freeze_keeps_narrow_layers():
    net = nn.Sequential(nn.Linear(256, 128), nn.GELU(), nn.Sequential(nn.Linear(128, 8)), Fp8Linear(300, 128))
    freeze_fp8(net)
    assert isinstance(net[0], FrozenFp8Linear) and isinstance(net[3], FrozenFp8Linear) and type(net[2][0]) is nn.Linear
    assert set(net[0].state_dict()) == {"weight_q", "weight_scale", "bias"}


def _refusals(dev):
    xq, xs = quantize_rows(torch.randn(4, 256, device=dev))
    wq, ws = quantize_blocks(torch.randn(130, 256, device=dev))
    for bad in (lambda: fp8_matmul(xq.float(), xs, wq, ws), lambda: fp8_matmul(xq[:, :128], xs, wq, ws),
                lambda: fp8_matmul(xq, xs[:, :1], wq, ws), lambda: fp8_matmul(xq, xs, wq, ws[:1]),
                lambda: fp8_matmul(xq, xs.double(), wq, ws), lambda: fp8_matmul(xq, xs, wq, ws, torch.zeros(3, device=dev)),
                lambda: fp8_matmul(xq, xs, wq, ws, out_dtype=torch.float64),
                lambda: fp8_matmul(xq, xs.clone().requires_grad_(True), wq, ws),
                lambda: quantize_rows(torch.zeros(3, 4, device=dev, dtype=torch.int32)),
                lambda: quantize_blocks(torch.zeros(3, device=dev)), lambda: quantize_blocks(torch.zeros(3, 4, 5, device=dev)),
                lambda: fp8_linear(torch.randn(4, 255, device=dev), torch.randn(130, 256, device=dev)),
                lambda: FrozenFp8Linear(torch.randn(8, 256, device=dev))(torch.randn(2, 256, device=dev, requires_grad=True))):
        with pytest.raises(ValueError):
            bad()


def test_refusals_cpu():
    _refusals("cpu")


@pytest.mark.gpu
def test_refusals_gpu():
    _refusals("cuda")
    xq, xs = quantize_rows(torch.randn(4, 256, device="cuda"))
    wq, ws = quantize_blocks(torch.randn(130, 256))
    with pytest.raises(ValueError):
        fp8_matmul(xq, xs, wq, ws)


def _same(got, want):
    return torch.equal(got.contiguous().view(torch.uint8), want.contiguous().view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k", [(1, 1), (1, 16), (3, 127), (5, 128), (4, 136), (7, 2008), (300, 257), (2, 16640), (1000, 64)])
def test_quantised_rows_are_exact(dtype, rows, k):
    x = _values(rows, k, rows + k, dtype, "cuda")
    q, s = quantize_rows(x)
    rq, rs = reference_quantize_rows(x)
    assert torch.equal(s, rs) and _same(q, rq) and q.stride(0) % 16 == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (8, 128), (128, 128), (130, 257), (1000, 2008), (3, 16640)])
def test_quantised_blocks_are_exact(dtype, n, k):
    w = _values(n, k, n + k, dtype, "cuda")
    q, s, qt, st = quantize_blocks(w, transposed=True)
    rq, rs = reference_quantize_blocks(w)
    assert torch.equal(s, rs) and _same(q, rq) and torch.equal(st, s.t()) and _same(qt, q.t())
    q2, s2 = quantize_blocks(w)
    assert _same(q2, q) and torch.equal(s2, s)


@pytest.mark.gpu
def test_quantised_ties_and_ends_of_the_range():
    """Quotients that lie on the middle of two e4m3 numbers, or next to it: multiples of an odd scale, and all of the
    group's bf16 neighbours of such middles; rows near both ends of fp32; subnormal inputs; zeros."""
    mid = (_slow_e4m3()[1:] + _slow_e4m3()[:-1]) / 2
    rows = []
    for amax in (448., 1., 3., 7.3, 2. ** -100, 2. ** 100, 3e38, 1e-30, 2e-38):
        v = (mid * amax / 448).float()
        for x in (v, torch.nextafter(v, torch.tensor(0.)), torch.nextafter(v, torch.tensor(1e38)), v.bfloat16().float()):
            rows.append(torch.cat((torch.tensor([amax], dtype=torch.float64).float(), x, torch.zeros(1))))
    rows.append(torch.full((128,), 1e-40))
    rows.append(torch.zeros(128))
    x = torch.stack(rows)
    x[::2] *= -1
    q, s = quantize_rows(x.cuda())
    rq, rs = reference_quantize_rows(x)
    assert torch.equal(s.cpu(), rs)
    assert torch.equal(q.float().cpu(), rq.float())


@pytest.mark.gpu
def test_non_finite_groups_become_nan():
    x = torch.randn(3, 300, device="cuda")
    x[0, 5], x[1, 200], x[2, 299] = torch.nan, torch.inf, -torch.inf
    q, s = quantize_rows(x)
    bad = torch.zeros(3, 300, dtype=torch.bool, device="cuda")
    bad[0, :128] = bad[1, 128:256] = bad[2, 256:] = True
    assert torch.equal(q.float().isnan(), bad)
    wq, ws = quantize_blocks(torch.randn(40, 300, device="cuda"))
    assert fp8_matmul(q, s, wq, ws).isnan().all()


@pytest.mark.gpu
def test_strided_inputs():
    big = torch.randn(40, 3, 520, device="cuda")
    for x in (big[:, 1], big[:, 1, 4:300], big[..., 1:257][:, 2], big.transpose(0, 2)[..., 0], big[0, 0].expand(7, 520),
              big.bfloat16()[:, 0, 1:130]):
        q, s = quantize_rows(x)
        rq, rs = reference_quantize_rows(x)
        assert torch.equal(s, rs) and _same(q, rq)
        q, s = quantize_blocks(x)
        rq, rs = reference_quantize_blocks(x)
        assert torch.equal(s, rs) and _same(q, rq)


def _check_product(y, a, a_s, b, b_s, bias, out):
    ad, bd = dequantize_rows(a, a_s).double(), dequantize_blocks(b, b_s).double()
    want, size = ad @ bd.t(), ad.abs() @ bd.abs().t()
    if bias is not None:
        want, size = want + bias.double(), size + bias.double().abs()
    tol = (a.shape[1] + 8) * E * size + torch.finfo(out).eps / 2 * want.abs() + torch.finfo(out).tiny
    assert y.dtype == out and ((y.double() - want).abs() <= tol).all(), ((y.double() - want).abs() / tol).max()


SHAPES = [(1, 1, 1), (1, 8, 128), (3, 130, 100), (16, 128, 128), (17, 200, 264), (33, 1408, 1000), (64, 64, 2008),
          (128, 128, 4096), (129, 257, 513), (300, 1000, 136), (1, 1408, 16640), (8, 4096, 1024), (1000, 136, 2000),
          (2500, 1500, 640), (130, 3000, 256), (20000, 300, 384),
          (6000, 900, 1000), (2050, 4100, 520), (5000, 1030, 2000),
          (64, 130, 5000), (65, 300, 5000), (31, 20000, 300), (7, 128, 100000), (60, 100, 40000)]


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", SHAPES)
@pytest.mark.parametrize("out", TYPES)
def test_product_matches_64_bits(m, n, k, out):
    a, a_s = quantize_rows(_values(m, k, m + k, device="cuda"))
    b, b_s = quantize_blocks(_values(n, k, n + k + 1, device="cuda") * k ** -.5)
    bias = torch.randn(n, generator=_gen(5)).cuda() if (m + n) % 2 else None
    with torch.no_grad():
        y = fp8_matmul(a, a_s, b, b_s, bias, out)
    check_gemm_status(torch.device("cuda", 0))
    _check_product(y, a, a_s, b, b_s, bias, out)


@pytest.mark.gpu
def test_product_of_any_scales():
    """Scales need not come from the quantisers: zero, negative, tiny and large ones."""
    a, a_s = quantize_rows(_values(200, 700, 1, device="cuda"))
    b, b_s = quantize_blocks(_values(300, 700, 2, device="cuda"))
    a_s[::3] *= -1e6
    a_s[:, 2] = 0.
    b_s[1] *= 1e-6
    _check_product(fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32), a, a_s, b, b_s, None, torch.float32)
    _check_product(fp8_matmul(a[:3], a_s[:3], b, b_s, out_dtype=torch.float32), a[:3], a_s[:3], b, b_s, None, torch.float32)


@pytest.mark.gpu
def test_product_of_unaligned_and_strided_operands():
    a, a_s = quantize_rows(_values(60, 700, 1, device="cuda"))
    b, b_s = quantize_blocks(_values(300, 700, 2, device="cuda"))
    want = fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32)
    ac, bc = a.contiguous(), b.contiguous()          # 700-byte rows
    assert ac.stride(0) == 700
    assert torch.equal(fp8_matmul(ac, a_s, bc, b_s, out_dtype=torch.float32), want)
    off = torch.zeros(60 * 704 + 1, dtype=torch.uint8, device="cuda")[1:].view(60, 704)
    off[:, :700] = a.view(torch.uint8)
    assert torch.equal(fp8_matmul(off.view(torch.float8_e4m3fn)[:, :700], a_s, b, b_s, out_dtype=torch.float32), want)
    at = a.view(torch.uint8).t().contiguous().t().view(torch.float8_e4m3fn)
    ast = a_s.t().contiguous().t()
    assert torch.equal(fp8_matmul(at, ast, b, b_s, out_dtype=torch.float32), want)
    y = fp8_matmul(a.unflatten(0, (3, 4, 5)), a_s.view(3, 4, 5, 6), b, b_s, out_dtype=torch.float32)
    assert torch.equal(y.view(60, 300), want)
    one = fp8_matmul(a[7], a_s[7], b, b_s, out_dtype=torch.float32)   # a vector
    _check_product(one[None], a[7:8], a_s[7:8], b, b_s, None, torch.float32)


@pytest.mark.gpu
def test_empty_products():
    for m, n, k in ((0, 5, 64), (4, 0, 64), (4, 5, 0)):
        a, a_s = quantize_rows(torch.randn(m, k, device="cuda"))
        b, b_s = quantize_blocks(torch.randn(n, k, device="cuda"))
        bias = torch.arange(n, device="cuda").float()
        y = fp8_matmul(a, a_s, b, b_s, bias)
        assert y.shape == (m, n) and (k or torch.equal(y.float(), bias.expand(m, n)))


@pytest.mark.gpu
def test_results_do_not_depend_on_the_run():
    a, a_s = quantize_rows(_values(5, 16640, 1, device="cuda"))
    b, b_s = quantize_blocks(_values(1408, 16640, 2, device="cuda"))
    first = fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32)
    for _ in range(5):
        assert torch.equal(fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32), first)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (257, 130, 200), (1024, 256, 520), (33, 1000, 127), (9000, 520, 264),
                                   (300, 5000, 4100)])
def test_linear_gradients_match_the_formula(dtype, m, n, k):
    x = _values(m, k, 1, torch.bfloat16, "cuda").to(dtype).requires_grad_(True)
    w = (_values(n, k, 2, device="cuda") * k ** -.5).requires_grad_(True)
    b = torch.randn(n, generator=_gen(4)).cuda().requires_grad_(True)
    dy = torch.randn(m, n, generator=_gen(3)).bfloat16().to(dtype).cuda()
    y = fp8_linear(x, w, b)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    xq, xs = quantize_rows(x)
    wq, ws = quantize_blocks(w)
    _check_product(y, xq, xs, wq, ws, b.detach(), dtype)
    gq, gs = quantize_rows(dy)
    _check_product(dx, gq, gs, *quantize_blocks(w.detach().t().contiguous()), None, dtype)
    # bf16 values, so the bf16 operands are exact (an fp16 x holds them but for its own rounding, 2^-11)
    terms = dy.double().abs().t() @ x.detach().double().abs()
    op = 2. ** -8 if dtype == torch.float16 else 0.   # fp16 values are rounded to bf16 operands
    assert ((dw.double() - dy.double().t() @ x.detach().double()).abs() <= ((m + 8) * E + 2.1 * op) * terms).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= (m + 8) * E * dy.double().abs().sum(0)).all()


@pytest.mark.gpu
def test_linear_input_gradient_is_the_difference_quotient():
    """With the group's largest value fixed at 448 the scale is 1 and e4m3 inputs are held exactly, so the layer is
    linear in them and its differences, sums of few small integers, are exact."""
    g = _gen(9)
    x = torch.randint(-8, 9, (3, 128), generator=g).float()
    w = torch.randint(-4, 5, (128, 128), generator=g).float()
    x[:, 0], w[0, 0] = 448., 448.
    x, w = x.cuda().requires_grad_(True), w.cuda()
    c = torch.zeros(3, 128, device="cuda")
    c[0, 5] = c[1, 77] = c[2, 127] = 1.
    gx, = torch.autograd.grad(fp8_linear(x, w), x, c)
    for i, n in ((0, 5), (1, 77), (2, 127)):
        for j in (1, 64, 127):
            e = torch.zeros_like(x)
            e[i, j] = 1.
            with torch.no_grad():
                up, down = x.clamp(-7, 7), None
                up[:, 0] = 448.
                d = (fp8_linear(up + e, w) - fp8_linear(up - e, w))[i, n] / 2
            assert d == w[n, j]
            # the gradient 1 is held as 448 times fp32(1 / 448)
            assert abs(gx[i, j] - w[n, j]) <= 2. ** -22 * abs(w[n, j])


@pytest.mark.gpu
def test_modules_under_autocast_and_frozen():
    lin = Fp8Linear(256, 384).cuda()
    x = torch.randn(70, 256, device="cuda")
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        y = lin(x)
        z = FrozenFp8Linear.from_linear(lin)(x)
    assert y.dtype == torch.bfloat16 and torch.equal(y, z)
    state = FrozenFp8Linear.from_linear(lin).state_dict()
    other = FrozenFp8Linear(torch.zeros(384, 256, device="cuda"), torch.zeros(384, device="cuda"))
    other.load_state_dict(state)
    # the fp32 input itself is quantised, inside the region as outside
    with torch.autocast("cuda", dtype=torch.bfloat16), torch.no_grad():
        assert torch.equal(other(x), z)


@pytest.mark.gpu
def test_captured_and_replayed_on_a_side_stream():
    lin = Fp8Linear(520, 300).cuda()
    x = torch.randn(77, 520, device="cuda").requires_grad_(True)
    dy = torch.randn(77, 300, device="cuda")

    def step():
        y = lin(x)
        return (y, *torch.autograd.grad(y, (x, lin.weight, lin.bias), dy))

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
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [20000, 300, 4])
def test_a_wait_that_runs_out_is_reported(m):
    dev = torch.device("cuda", 0)
    a, a_s = quantize_rows(_values(m, 4096, 1, device="cuda"))
    b, b_s = quantize_blocks(_values(512, 4096, 2, device="cuda"))
    fp8_matmul(a, a_s, b, b_s)
    check_gemm_status(dev)
    with pytest.raises(TensorCoreTimeout):
        fp8_matmul(a, a_s, b, b_s, wait_ns=0)
        check_gemm_status(dev)
    y = fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32)   # the next call is sound
    check_gemm_status(dev)
    _check_product(y, a, a_s, b, b_s, None, torch.float32)


@pytest.mark.gpu
def test_changes_in_place_and_second_derivatives_are_refused():
    x = torch.randn(8, 64, device="cuda").bfloat16()
    w = torch.randn(32, 64, device="cuda", requires_grad=True)
    y = fp8_linear(x, w)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y.sum(), w, create_graph=True)
    y = fp8_linear(x, w)
    x += 1.   # the weight gradient would read it
    with pytest.raises(RuntimeError):
        y.sum().backward()


@pytest.mark.gpu
def test_frozen_raster_policy_acts_as_its_dequantised_weights_would():
    """The raster network's wide layers (16640 -> 1408 -> 256) frozen: the logits against the same network with the
    quantised weights and inputs in fp32, 16640 terms off by at most (K + 8) 2^-23 of their magnitudes each, which
    moves a hidden value across a rounding of the next layer at times: one step of e4m3, 2^-3, of single values among
    hundreds, well under 5 % of the logits. size."""
    from autodrive_b200.models.zoo import PerceptionActorCritic
    torch.manual_seed(0)
    policy = PerceptionActorCritic("raster_cnn_large", tensor_cores=False).cuda()
    inputs = {"scalars": torch.randn(5, 137, device="cuda"), "field": torch.rand(5, 12, 64, 128, device="cuda")}
    freeze_fp8(policy)
    frozen = [m for m in policy.modules() if isinstance(m, FrozenFp8Linear)]
    assert len(frozen) == 3
    with torch.no_grad():
        got = policy(inputs)[0]
        for m in frozen:
            m.forward = lambda x, m=m: torch.nn.functional.linear(
                dequantize_rows(*quantize_rows(x)), dequantize_blocks(m.weight_q, m.weight_scale), m.bias)
        want = policy(inputs)[0]
    check_gemm_status(torch.device("cuda", 0))
    assert got.shape == (5, 8) and (got - want).abs().max() <= .05 * want.abs().max()


@pytest.mark.gpu
def test_no_gradient_is_prepared_where_none_is_taken():
    x = torch.randn(40, 300, device="cuda", requires_grad=True)
    w = torch.randn(130, 300, device="cuda", requires_grad=True)
    with torch.no_grad():
        y = fp8_linear(x, w)
    assert not y.requires_grad and torch.equal(y, fp8_linear(x, w))
    y = fp8_linear(x, w.detach())
    gx, = torch.autograd.grad(y, x, torch.ones_like(y))
    assert gx.shape == x.shape
    y = fp8_linear(x.detach(), w)
    gw, = torch.autograd.grad(y, w, torch.ones_like(y))
    assert gw.shape == w.shape


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_frozen_layers_keep_their_types_when_the_network_is_converted(device):
    net = freeze_fp8(nn.Sequential(nn.Linear(300, 200), nn.Linear(200, 5)))
    x = torch.randn(4, 300)
    with torch.no_grad():
        want = net[0](x)
        net.half().to(device)
        layer = net[0]
        assert layer.weight_q.dtype == torch.float8_e4m3fn and layer.weight_scale.dtype == layer.bias.dtype == torch.float32
        assert layer.weight_q.device.type == device and layer.weight_q.stride(0) % 16 == 0
        assert net[1].weight.dtype == torch.float16
        got = layer(x.to(device))
        assert net(x.half().to(device)).shape == (4, 5)
    # fp32 sums of 300 terms of size 1 on either device
    assert (got.cpu() - want).abs().max() <= 310 * E * 40


@pytest.mark.gpu
def test_pairs_of_ctas_read_each_others_tiles_when_they_are_there():
    """Two sets of operands of other sizes of value in turn, a different value in every group of 128: a tile that the
    pair's products read before the second CTA's loads have landed would be the other call's or an earlier group's.
    Products and weight gradients are sums of small integers, below 2^24, so every order of addition gives them exactly."""
    def operands(seed):
        g = _gen(seed)
        a = torch.randint(-3 * seed, 3 * seed + 1, (2500, 1408), generator=g).float()
        b = torch.randint(-3, 4, (1500, 1408), generator=g).float()
        q = [t.to(fp8.E4M3).cuda() for t in (a, b)]
        scales = (torch.arange(1, 12).float().repeat(2500, 1).cuda(), torch.ones(12, 11).cuda())
        want = ((a * torch.arange(1, 12).repeat_interleave(128)).double() @ b.double().t()).cuda()
        dy = torch.randint(-3 * seed, 3 * seed + 1, (5000, 520), generator=g).float().bfloat16().cuda()
        x = torch.randint(-3, 4, (5000, 648), generator=g).float().bfloat16().cuda()
        return q, scales, want.float(), dy, x, (dy.double().t() @ x.double()).float()

    sets = [operands(1), operands(4)]
    w = torch.zeros(520, 648, device="cuda", requires_grad=True)
    for _ in range(40):
        for (a, b), (a_s, b_s), want, dy, x, dw in sets:
            assert torch.equal(fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32), want)
            assert torch.equal(torch.autograd.grad(fp8_linear(x, w), w, dy)[0], dw)
    check_gemm_status(torch.device("cuda", 0))


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(20000, 512, 2048), (300, 512, 2048), (4, 512, 2048), (4, 512, 512), (40, 300, 128)])
def test_waits_of_any_length_leave_nothing_in_flight(m, n, k):
    """Waits that run out somewhere between the first load and the last product, or not at all: the call either reports
    them or is right, and the next call on the same shared memory and TMEM is right in any case."""
    dev = torch.device("cuda", 0)
    a, a_s = quantize_rows(_values(m, k, 1, device="cuda"))
    b, b_s = quantize_blocks(_values(n, k, 2, device="cuda"))
    want = fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32)
    check_gemm_status(dev)
    for wait_ns in (0, 200, 500, 1000, 1500, 2000, 3000, 5000, 10000, 20000) * 3:
        try:
            y = fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32, wait_ns=wait_ns)
            z = fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32)   # may report it as well
            check_gemm_status(dev)
        except TensorCoreTimeout:
            y, z = want, fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32)
        assert torch.equal(y, want) and torch.equal(z, want)
    check_gemm_status(dev)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (257, 130, 200), (3000, 256, 521)])
def test_operands_of_the_weight_gradient(dtype, m, n, k):
    """Values that use all bits of their type: fp16 and bf16 operands enter the product as they are, fp32 ones rounded to
    bf16, and the sums are fp32."""
    x = _values(m, k, 1, dtype, "cuda")
    w = (_values(n, k, 2, device="cuda") * k ** -.5).requires_grad_(True)
    dy = _values(m, n, 3, dtype, "cuda")
    dw, = torch.autograd.grad(fp8_linear(x, w), w, dy)
    a, b = (t.bfloat16().double() if dtype == torch.float32 else t.double() for t in (dy, x))
    assert ((dw.double() - a.t() @ b).abs() <= (m + 8) * E * (a.abs().t() @ b.abs())).all()
    # against the unrounded gradient: 2^-8 of the terms for each bf16 operand, to first order
    a, b = dy.double(), x.double()
    op = 2. ** -8 if dtype == torch.float32 else 0.
    assert ((dw.double() - a.t() @ b).abs() <= ((m + 8) * E + 2.1 * op) * (a.abs().t() @ b.abs())).all()


@pytest.mark.gpu
def test_weight_gradient_of_mixed_types():
    """An fp16 input whose gradient comes in bf16 (autocast), or the reverse: both operands in bf16."""
    for xt, out in ((torch.float16, torch.bfloat16), (torch.float32, torch.float16), (torch.bfloat16, torch.float16)):
        x, w = _values(300, 200, 1, xt, "cuda"), _values(130, 200, 2, device="cuda").requires_grad_(True)
        with torch.autocast("cuda", dtype=out):
            y = fp8_linear(x, w)
        assert y.dtype == out
        dy = _values(300, 130, 3, out, "cuda")
        dw, = torch.autograd.grad(y, w, dy)
        a, b = dy.bfloat16().double(), x.bfloat16().double()
        assert ((dw.double() - a.t() @ b).abs() <= 308 * E * (a.abs().t() @ b.abs())).all()


def test_frozen_layers_of_a_skeleton_and_in_shared_memory():
    x = torch.randn(3, 300)
    net = nn.Sequential(freeze_fp8(nn.Sequential(nn.Linear(300, 200))), nn.Linear(200, 5))
    state = net.state_dict()
    with torch.device("meta"):
        skeleton = nn.Sequential(nn.Sequential(FrozenFp8Linear(torch.empty(200, 300), torch.empty(200))), nn.Linear(200, 5))
    skeleton.to_empty(device="cpu").load_state_dict(state)
    layer = skeleton[0][0]
    assert layer.weight_q.dtype == fp8.E4M3 and layer.weight_q.stride() == (304, 1)
    with torch.no_grad():
        assert torch.equal(skeleton(x), net(x))
    net.share_memory()
    assert all(t.is_shared() for t in net.state_dict().values())
    with torch.no_grad():
        assert torch.equal(skeleton(x), net(x))
    for change in (lambda n: n.half().float(), lambda n: n.type(torch.float64).float(), lambda n: n.to(torch.bfloat16).float()):
        assert change(net)[0][0].weight_q.dtype == fp8.E4M3 and net[0][0].weight_scale.dtype == torch.float32
        assert torch.equal(net[0][0].weight_scale, layer.weight_scale)
        assert torch.equal(net[0][0].weight_q.float(), layer.weight_q.float())


def test_freeze_of_a_layer_itself():
    lin, narrow = nn.Linear(300, 200), nn.Linear(300, 5)
    frozen = freeze_fp8(lin)
    x = torch.randn(3, 300)
    with torch.no_grad():
        assert isinstance(frozen, FrozenFp8Linear) and torch.equal(frozen(x), FrozenFp8Linear.from_linear(lin)(x))
    assert freeze_fp8(narrow) is narrow


def test_freeze_of_a_layer_that_stands_in_several_places():
    class Net(nn.Module):
        def __init__(self):
            super().__init__()
            self.a = nn.Linear(256, 256)
            self.b, self.inner = self.a, nn.Sequential(self.a, nn.Linear(256, 4))

    net = freeze_fp8(Net())
    assert isinstance(net.a, FrozenFp8Linear) and net.b is net.a and net.inner[0] is net.a and type(net.inner[1]) is nn.Linear


def test_freeze_keeps_hooks_and_mode():
    net = nn.Sequential(nn.Linear(256, 256), nn.Linear(256, 256)).eval()
    seen = []
    handle = net[0].register_forward_hook(lambda m, a, y: seen.append(("after", type(m), y.shape)))
    net[1].register_forward_pre_hook(lambda m, a: seen.append(("before", type(m), a[0].shape)))
    net[1].register_forward_hook(lambda m, a, k, y: y + 1., with_kwargs=True)
    freeze_fp8(net)
    x = torch.randn(2, 256)
    with torch.no_grad():
        y = net(x)
        want = net[1].forward(net[0].forward(x)) + 1.
    assert seen == [("after", FrozenFp8Linear, (2, 256)), ("before", FrozenFp8Linear, (2, 256))]
    assert torch.equal(y, want) and not net[0].training
    handle.remove()
    with torch.no_grad():
        net(x)
    assert len(seen) == 3


def test_freeze_leaves_layers_whose_weights_others_read():
    net = nn.Sequential(nn.TransformerEncoderLayer(256, 4, 512, batch_first=True), nn.Linear(256, 256)).eval()
    x = torch.randn(2, 3, 256)
    with torch.no_grad():
        want = net[0](x)
        freeze_fp8(net)
        assert torch.equal(net[0](x), want) and isinstance(net[1], FrozenFp8Linear)


@pytest.mark.gpu
@pytest.mark.parametrize("m,n,k", [(16, 2048, 2048), (32, 2560, 2048), (3, 4480, 1100), (16, 9500, 700), (640, 512, 2100),
                                   (1400, 1000, 1024)])
def test_product_where_the_number_of_clusters_decides(m, n, k):
    a, a_s = quantize_rows(_values(m, k, 1, device="cuda"))
    b, b_s = quantize_blocks(_values(n, k, 2, device="cuda") * k ** -.5)
    _check_product(fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32), a, a_s, b, b_s, None, torch.float32)
    check_gemm_status(torch.device("cuda", 0))


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_product_refuses_operands_that_want_a_gradient(device):
    q, s = quantize_rows(torch.randn(4, 256, device=device))
    wq, ws = quantize_blocks(torch.randn(130, 256, device=device))
    for bad in (lambda: fp8_matmul(q.clone().requires_grad_(True), s, wq, ws),
                lambda: fp8_matmul(q, s, wq.clone().requires_grad_(True), ws)):
        with pytest.raises(ValueError):
            bad()
        with torch.no_grad():
            assert bad().shape == (4, 130)


@pytest.mark.gpu
@pytest.mark.parametrize("m", [4, 200, 5000])
def test_products_of_scales_at_the_end_of_the_range(m):
    """2^-63 times 2^-62 is a normal fp32 number; 2^-64 times 2^-63 is below them and counts as zero."""
    a, a_s = quantize_rows(_values(m, 256, 1, device="cuda"))
    b, b_s = quantize_blocks(_values(600, 256, 2, device="cuda"))
    a_s, b_s = torch.full_like(a_s, 2. ** -63), torch.full_like(b_s, 2. ** -62)
    _check_product(fp8_matmul(a, a_s, b, b_s, out_dtype=torch.float32), a, a_s, b, b_s, None, torch.float32)
    assert (fp8_matmul(a, a_s / 2, b, b_s / 2, out_dtype=torch.float32) == 0).all()
