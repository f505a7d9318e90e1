"""Log-probabilities of given tokens, entropy, alternatives and the gradient
against 64-bit softmax arithmetic.

Tolerances, with f = 2^-24. log_prob = (x_t - m) / T - log s: the first term
is rounded three times (3 f of it). Each exp is off by 2^-22 for the function
and 4 f |d| for its argument d / T, whose mean over the distribution is at most
log V; s is a sum of V terms, added in chains of at most 32 + V / 512 and
joined over at most 9 levels that round 4 times each: together
S = f (8 + 4 log V + V / 512 + 72), and as much again for the logarithm.
The entropy log s - t / (T s) has the same errors twice, relative to its terms,
which are at most its value: 3 S (1 + H). A gradient entry has the errors of p
(exp and argument) and of log p and H in its factor, and its type's rounding.
"""
import math

import pytest
import torch

from autodrive_b200.ops.token_logprobs import TokenLogProbs, reference_token_log_probs, token_log_probs

F = 2. ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def _make(rows, v, dtype, device, mask=False, seed=0, spread=3.):
    g = torch.Generator().manual_seed(seed + 7 * rows + v)
    x = (spread * torch.randn(rows, v, generator=g)).to(dtype).to(device)
    t = torch.randint(v, (rows,), generator=g).to(device)
    m = None
    if mask:
        m = (torch.rand(rows, v, generator=g) < .6).to(device)
        m[1::5] = False
    return x, t, m


def _oracle(x, t, mask, temperature, gl=None, ge=None):
    """(log_prob, entropy, log p, empty rows, gradient) in 64 bits."""
    z = x.detach().double().requires_grad_(True)
    ok = torch.ones_like(x, dtype=torch.bool) if mask is None else mask
    ok = ok & ~(x == -torch.inf)
    empty = ~ok.any(-1)
    use = ok | empty[:, None]
    lp = torch.log_softmax(torch.where(use, torch.where(use, z, 0.) / temperature, -torch.inf), -1)
    p = lp.exp()
    h = -(p * torch.where(use, lp, 0.)).sum(-1)
    lt = lp.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
    grad = None
    if gl is not None:
        live = (~empty).double()
        counted = live * ((t >= 0) & (t < x.shape[1]))
        valid = use.gather(1, t.clamp(0, x.shape[1] - 1)[:, None])[:, 0]
        # d(-inf) of a masked token: the logsumexp's part alone
        lt_g = torch.where(valid, lt, -torch.logsumexp(torch.where(use, z / temperature, -torch.inf), -1))
        grad, = torch.autograd.grad((lt_g, h), z, (gl.double() * counted, ge.double() * live))
        grad = torch.where(ok, grad, 0.)
    lp, h, lt = lp.detach(), h.detach(), lt.detach()
    return torch.where(empty, -torch.inf, lt), torch.where(empty, 0., h), lp, empty, grad


def _s(v):
    return F * (8 + 4 * math.log(v + 1) + v / 512 + 72)


def _close(got, want, tol):
    same = (got == want) | (got.isnan() & want.isnan())
    assert (same | ((got.double() - want).abs() <= tol)).all(), float(((got.double() - want).abs() / tol)[~same].max())


def _check(x, t, mask, temperature, top, r: TokenLogProbs):
    lt, h, lp, empty, _ = _oracle(x, t, mask, temperature)
    v = x.shape[1]
    lt = torch.where(t < 0, 0., torch.where(t >= v, torch.nan, lt))
    far = 3 * F * (lt.abs() + 2 * math.log(v + 1)).nan_to_num(posinf=0.)
    assert r.log_prob.dtype == r.entropy.dtype == torch.float32
    _close(r.log_prob, lt, far + 3 * _s(v))
    _close(r.entropy, h, 3 * _s(v) * (1 + h))
    order = x.float() if mask is None else torch.where(mask, x.float(), -torch.inf)
    value, index = torch.sort(order, dim=-1, descending=True, stable=True)
    value, index = value[:, :top], index[:, :top]
    index = torch.where(value == -torch.inf, -1, index)
    best = torch.where(index < 0, -torch.inf, lp.gather(1, index.clamp_min(0)))
    n = index.shape[1]
    assert r.top_token.shape == r.top_log_prob.shape == (x.shape[0], top)
    assert torch.equal(r.top_token[:, :n], index) and (r.top_token[:, n:] == -1).all()
    _close(r.top_log_prob[:, :n], best, 3 * F * (best.abs().nan_to_num(posinf=0.) + 2 * math.log(v + 1)) + 3 * _s(v))
    assert (r.top_log_prob[:, n:] == -torch.inf).all()


def _check_grad(x, t, mask, temperature, gl, ge, dx):
    lt, h, lp, empty, want = _oracle(x, t, mask, temperature, gl, ge)
    u, v = torch.finfo(x.dtype).eps / 2, x.shape[1]
    p, a = lp.exp(), lp.abs().nan_to_num(posinf=0.)
    gl, ge = gl.double().abs()[:, None], ge.double().abs()[:, None]
    hot = torch.zeros_like(p).scatter_(1, t.clamp(0, v - 1)[:, None], 1.)
    log_tol = 3 * F * (a + 2 * math.log(v + 1)) + 3 * _s(v)
    tol = p * (gl + ge * (a + h[:, None])) * (4 * log_tol + 2. ** -21) + p * ge * (log_tol + 3 * _s(v) * (1 + h[:, None]))
    tol = (tol + 4 * F * gl * (hot + p)) / temperature + u * want.abs() + 2 * u * torch.finfo(x.dtype).tiny
    _close(dx.double(), want, tol + 1e-36)   # below fp32's normal range values are flushed to zero


def _run(x, t, mask=None, temperature=1., top=0):
    g = torch.Generator().manual_seed(5)
    gl, ge = (torch.randn(x.shape[0], generator=g).to(x.device) for _ in range(2))
    x = x.clone().requires_grad_(True)
    r = token_log_probs(x, t, mask, temperature, top)
    _check(x.detach(), t, mask, temperature, top, TokenLogProbs(*(o.detach() for o in r)))
    dx, = torch.autograd.grad((r.log_prob, r.entropy), x, (gl, ge))
    assert dx.dtype == x.dtype
    _check_grad(x.detach(), t, mask, temperature, gl, ge, dx)
    with torch.no_grad():
        for a, b in zip(token_log_probs(x, t, mask, temperature, top), r):
            assert torch.equal(a.nan_to_num(nan=7.), b.nan_to_num(nan=7.)) if a.is_floating_point() else torch.equal(a, b)


@pytest.mark.parametrize("mask", [False, True])
def test_cpu(mask):
    x, t, m = _make(12, 40, torch.float32, "cpu", mask)
    t[3], t[4] = -1, 40
    _run(x, t, m, .7, 5)


def test_cpu_agrees_with_the_categorical_distribution():
    x, t, _ = _make(9, 8, torch.float32, "cpu")
    r = token_log_probs(x, t)
    d = torch.distributions.Categorical(logits=x)
    assert torch.allclose(r.log_prob, d.log_prob(t), atol=1e-6) and torch.allclose(r.entropy, d.entropy(), atol=1e-6)


def _refusals(dev):
    x, t = torch.randn(4, 9, device=dev), torch.zeros(4, dtype=torch.long, device=dev)
    for bad in (lambda: token_log_probs(x.double(), t), lambda: token_log_probs(x, t[:3]), lambda: token_log_probs(x, t.float()),
                lambda: token_log_probs(x, t, temperature=0.), lambda: token_log_probs(x, t, temperature=float("nan")),
                lambda: token_log_probs(x, t, temperature=float("inf")),
                lambda: token_log_probs(x, t, top=65), lambda: token_log_probs(x, t, top=-1),
                lambda: token_log_probs(x, t, mask=torch.ones(4, 9, device=dev)),
                lambda: token_log_probs(x, t, mask=torch.ones(4, 8, dtype=torch.bool, device=dev)),
                lambda: token_log_probs(x[:, :0], t)):
        with pytest.raises(ValueError):
            bad()


def test_refusals_cpu():
    _refusals("cpu")


@pytest.mark.gpu
def test_refusals_gpu():
    _refusals("cuda")
    with pytest.raises(ValueError):
        token_log_probs(torch.randn(4, 9, device="cuda"), torch.zeros(4, dtype=torch.long))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,v", [(1, 1), (3, 2), (70, 8), (300, 9), (7, 33), (5, 128), (40, 137), (6, 512), (9, 1000),
                                    (3, 1024), (3, 1025), (4, 2047), (5, 4104), (7, 32003), (2, 131072), (1, 200003)])
@pytest.mark.parametrize("mask", [False, True])
def test_matches_64_bits(dtype, rows, v, mask):
    _run(*_make(rows, v, dtype, "cuda", mask), .7 if rows % 2 else 1., 5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,v", [(4096, 8), (40000, 5), (1000, 4099), (600, 32000)])
def test_many_rows(rows, v):
    _run(*_make(rows, v, torch.bfloat16, "cuda", rows > 999), 1., 0)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [20, 64, 700, 1025, 40000])
@pytest.mark.parametrize("top", [1, 20, 64])
def test_alternatives(v, top):
    x, t, m = _make(6, v, torch.bfloat16, "cuda", True)   # bf16: many equal logits
    _run(x, t, m, 1.3, top)
    _run(x, t, None, 1.3, top)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 500, 5000, 70001])
def test_equal_sorted_and_clustered_rows(v):
    """Rows whose largest entries are all equal, in order, in one place, or in the strides of a thread."""
    x = torch.zeros(9, v, device="cuda")
    x[1] = torch.arange(v) / v
    x[2] = -torch.arange(v) / v
    x[3, v // 2:] = 1.
    x[4, ::7] = 2.
    x[5] = torch.where(torch.arange(v) // 8 % 512 < 3, torch.arange(v) % 11, -1.)
    x[6] = -0.
    x[6, 1::2] = 0.
    x[7] = torch.where(torch.arange(v) % 4096 < 24, 1., 0.) + torch.rand(v) / 4
    x[8] = torch.finfo(torch.float32).min
    t = torch.arange(9, device="cuda") % v
    for top in (3, 64):
        _check(x, t, None, 1., top, token_log_probs(x, t, top=top))


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 300, 3000])
@pytest.mark.parametrize("dtype", TYPES)
def test_masked_values_are_not_read(v, dtype):
    x, t, m = _make(20, v, dtype, "cuda", True)
    for bad in (torch.nan, torch.inf, -torch.inf, torch.finfo(dtype).max, torch.finfo(dtype).min):
        y = torch.where(m, x, torch.full_like(x, bad))
        _run(y, t, m, 1., 4)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 300, 3000])
def test_lowest_values_and_infinities_as_masks(v):
    """Logits that were masked by hand: the type's lowest value keeps its (vanishing) entry, -inf has none."""
    for dtype in TYPES:
        x, t, m = _make(20, v, dtype, "cuda", True)
        m[:, 0] = True
        t.zero_()
        _run(torch.where(m, x, torch.full_like(x, torch.finfo(dtype).min)), t, None, 1., 3)
        _run(torch.where(m, x, torch.full_like(x, -torch.inf)), t, None, 1., 3)
    x = torch.full((3, v), -torch.inf, device="cuda")
    x[1] = torch.finfo(torch.float32).min
    x[2] = torch.finfo(torch.float32).max
    t = torch.zeros(3, dtype=torch.long, device="cuda")
    r = token_log_probs(x, t, top=2)
    assert r.log_prob[0] == -torch.inf and r.entropy[0] == 0 and (r.top_token[0] == -1).all()
    assert torch.allclose(r.log_prob[1:], torch.full((2,), -math.log(v), device="cuda"), atol=1e-5)
    assert r.top_token[1:].tolist() == [[0, 1], [0, 1]]


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 300, 3000])
def test_non_finite_rows_are_nan(v):
    x = torch.randn(5, v, device="cuda")
    x[1, v // 2], x[2, v - 1], x[3] = torch.nan, torch.inf, torch.nan
    x[4], x[4, 3] = -torch.inf, torch.nan
    x.requires_grad_(True)
    r = token_log_probs(x, torch.zeros(5, dtype=torch.long, device="cuda"), top=1)
    assert r.log_prob[0].isfinite() and r.log_prob[1:].isnan().all() and r.entropy[1:].isnan().all()
    (r.log_prob.sum() + r.entropy.sum()).backward()
    assert x.grad[0].isfinite().all() and x.grad[1:3].isnan().all()


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 3000])
def test_ignored_unknown_and_masked_tokens(v):
    x, t, m = _make(20, v, torch.float32, "cuda", True)
    t[0], t[6], t[7], t[2] = -1, -100, v, 2 ** 40
    m[10, t[10]] = False
    m[12] = False
    m[12, (t[12] + 1) % v] = True   # one entry left, and it is not the token
    r = token_log_probs(x, t, m)
    assert r.log_prob[0] == 0 and r.log_prob[6] == 0 and r.log_prob[7].isnan() and r.log_prob[10] == -torch.inf
    _run(x, t, m)


@pytest.mark.gpu
def test_leading_dimensions_strides_and_broadcast_masks():
    g = torch.Generator(device="cuda").manual_seed(0)
    for v in (40, 2000):
        big = torch.randn(3, 4, 2, v + 9, device="cuda", generator=g)
        x = big[:, :, 1, 5:5 + v]
        t = torch.randint(v, (3, 4), device="cuda", generator=g, dtype=torch.int32)
        flat, tf = x.reshape(12, v).contiguous(), t.reshape(12).long()
        for mask in (None, torch.rand(v, device="cuda", generator=g) < .5, torch.rand(4, 1, device="cuda", generator=g) < .5,
                     torch.rand(3, 4, v, device="cuda", generator=g) < .5):
            r = token_log_probs(x, t, mask, top=3)
            assert r.log_prob.shape == (3, 4) and r.top_token.shape == (3, 4, 3)
            mf = None if mask is None else mask.expand(3, 4, v).reshape(12, v)
            _check(flat, tf, mf, 1., 3, TokenLogProbs(*(o.reshape(12, *o.shape[2:]) for o in r)))
        # every row the same row: the gradient comes back summed
        row = torch.randn(v, device="cuda", generator=g, requires_grad=True)
        r = token_log_probs(row.expand(6, v), tf[:6])
        (r.log_prob.sum() + 2 * r.entropy.sum()).backward()
        one = row.detach().expand(6, v)
        want = _oracle(one, tf[:6], None, 1., torch.ones(6, device="cuda"), torch.full((6,), 2., device="cuda"))[4].sum(0)
        assert torch.allclose(row.grad.double(), want, atol=1e-4)
        single = token_log_probs(row.detach(), tf[0], top=2)
        assert single.log_prob.shape == () and single.top_token.shape == (2,)
    e = token_log_probs(torch.randn(0, 9, device="cuda", requires_grad=True), torch.zeros(0, dtype=torch.long, device="cuda"))
    assert e.log_prob.shape == (0,)


@pytest.mark.gpu
def test_gradient_is_the_difference_quotient():
    """Central differences with a step of 2^-5: their truncation, step^2 / 6 of a third derivative that is at most a few
    units, is below 1e-3, their rounding 2^-20 / 2^-5 below 1e-4."""
    for v in (8, 1500):
        x, t, m = _make(4, v, torch.float32, "cuda", True, spread=1.)
        x.requires_grad_(True)
        f = lambda a: (lambda r: r.log_prob[[0, 2]].double().sum() + .5 * r.entropy.double().sum())(token_log_probs(a, t, m, .8))  # noqa: E731
        m[0, t[0]] = m[2, t[2]] = True
        gx, = torch.autograd.grad(f(x), x)
        for i, j in ((0, int(t[0])), (2, int(t[2])), (2, 3), (3, v - 1), (1, 0)):
            e = torch.zeros_like(x)
            e[i, j] = 2. ** -5
            with torch.no_grad():
                num = (f(x + e) - f(x - e)) / 2. ** -4
            assert abs(num - gx[i, j]) < 2e-3


@pytest.mark.gpu
def test_only_one_of_the_outputs_is_used():
    x, t, _ = _make(6, 50, torch.float32, "cuda")
    x.requires_grad_(True)
    z, o = torch.zeros(6, device="cuda"), torch.ones(6, device="cuda")
    r = token_log_probs(x, t, top=2)
    assert not r.top_log_prob.requires_grad
    a, = torch.autograd.grad(r.log_prob.sum(), x, retain_graph=True)
    b, = torch.autograd.grad(r.entropy.sum(), x)
    _check_grad(x.detach(), t, None, 1., o, z, a)
    _check_grad(x.detach(), t, None, 1., z, o, b)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 5000])
def test_captured_and_replayed(v):
    x, t, m = _make(30, v, torch.bfloat16, "cuda", True)
    x.requires_grad_(True)
    gl = torch.randn(30, device="cuda")

    def step():
        r = token_log_probs(x, t, m, .9, 4)
        return (*r, *torch.autograd.grad((r.log_prob, r.entropy), x, (gl, gl)))

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
        t.copy_(t.flip(0))
    graph.replay()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_reference_pads_and_breaks_ties_by_index():
    x = torch.tensor([[1., 3., 3., -torch.inf]])
    r = reference_token_log_probs(x, torch.tensor([1]), top=5)
    assert r.top_token.tolist() == [[1, 2, 0, -1, -1]]


@pytest.mark.gpu
def test_changes_in_place_and_second_derivatives_are_refused():
    x, t, _ = _make(4, 64, torch.float32, "cuda")
    x.requires_grad_(True)
    r = token_log_probs(x, t)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(r.log_prob.sum(), x, create_graph=True)
    r = token_log_probs(x, t)
    with torch.no_grad():
        x += 1.
    with pytest.raises(RuntimeError):
        r.entropy.sum().backward()


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 40, 900, 5000])
@pytest.mark.parametrize("temperature", [1., .25])
def test_peaked_rows(v, temperature):
    """One entry holds all but d of the probability, d from 1e-7 to a half, among seven others that are valid: the sum is
    1 + d', and its logarithm all of the answer. The 1 is rounded by three joins of lanes (seven additions by the one
    thread that has them all, in long rows), F each as the sum stays below 2; the exponentials are off by 2^-22 + 4 F |x / T| of themselves, with |x / T| up to 20 less than 96 F; the logarithm
    is off by 6 F of itself, and the entropy's second term by less than 100 F. No log-probability is above 0, and no
    entropy below."""
    g = torch.Generator().manual_seed(v)
    rows = 3000
    d = 10. ** (-7 + 6.7 * torch.rand(rows, generator=g, dtype=torch.float64))
    x = torch.full((rows, v), -50.)
    x[:, 1:8] = (temperature * ((d / 7)[:, None].log() + .3 * torch.randn(rows, 7, generator=g, dtype=torch.float64))).float()
    x[:, 0] = 0.
    x, t = x.cuda(), torch.zeros(rows, dtype=torch.long, device="cuda")
    mask = torch.arange(v, device="cuda") < 8
    z = x[:, :8].double() / temperature
    rest = z[:, 1:].exp().sum(1)
    lp, h = -torch.log1p(rest), torch.log1p(rest) - (z * z.exp()).sum(1) / (1 + rest)
    r = token_log_probs(x, t, mask, temperature, top=1)
    tol = F * ((3 if v <= 1024 else 7) + 100 * rest + 8 * lp.abs())
    assert ((r.log_prob - lp).abs() <= tol).all(), float(((r.log_prob - lp).abs() / tol).max())
    assert torch.equal(r.top_log_prob[:, 0], r.log_prob) and (r.log_prob <= 0).all()
    tol = tol + 100 * F * h
    assert ((r.entropy - h).abs() <= tol).all(), float(((r.entropy - h).abs() / tol).max())
    assert (r.entropy >= 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 1000, 9000])
def test_equal_entries(v):
    """n equal entries: the sum is n exactly, and the entropy its logarithm, which is off by at most six roundings."""
    x, n = torch.full((v, v), 2.5, device="cuda"), torch.arange(1, v + 1, device="cuda")
    r = token_log_probs(x, torch.zeros(v, dtype=torch.long, device="cuda"), torch.arange(v, device="cuda") < n[:, None])
    want = n.double().log()
    assert ((r.entropy - want).abs() <= 6 * F * want).all() and torch.equal(r.log_prob, -r.entropy)


@pytest.mark.gpu
@pytest.mark.parametrize("v", [8, 3000])
def test_values_below_the_normal_range_equal_zero(v):
    x = torch.full((2, v), -1., device="cuda")
    x[0, 2], x[0, 5], x[1, 1], x[1, 4], x[1, 6] = 0., 1e-40, -1e-40, 1e-39, 2. ** -126
    r = token_log_probs(x, torch.zeros(2, dtype=torch.long, device="cuda"), top=3)
    assert r.top_token[0, :2].tolist() == [2, 5] and r.top_token[1].tolist() == [6, 1, 4]
