"""The operators as they are used together: norm -> 8-bit product -> scored
tokens, serving and training, each stage against 64-bit arithmetic on what the
stage before it gave.

Tolerances: logits of K columns are off by at most (K + 8) 2^-23 of the sum of
their terms' magnitudes (see test_fp8.py); a log-probability moves by at most
twice the largest logit's error, and by the 1e-5 that test_token_logprobs.py
derives for these lengths.
"""
import pytest
import torch

from autodrive_b200.models.actor_critic import ActorCritic
from autodrive_b200.models.zoo import PerceptionActorCritic
from autodrive_b200.ops.fp8 import (FrozenFp8Linear, dequantize_blocks, dequantize_rows, fp8_linear, fp8_matmul, quantize_blocks,
                                    quantize_rows)
from autodrive_b200.ops.rmsnorm import FusedRMSNorm, rms_norm, rms_norm_fp8
from autodrive_b200.ops.tc_linear import check_gemm_status
from autodrive_b200.ops.token_logprobs import token_log_probs

E = 2. ** -23


def _inputs(m, k, v):
    g = torch.Generator().manual_seed(m + k + v)
    x, r = (torch.randn(m, k, generator=g).bfloat16().cuda() for _ in range(2))
    w = (1 + .1 * torch.randn(k, generator=g)).cuda()
    head = (2 * torch.randn(v, k, generator=g) * k ** -.5).cuda()
    t = torch.randint(v, (m,), generator=g).cuda()
    return x, r, w, head, t


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,v", [(1, 256, 1000), (7, 520, 8), (40, 1000, 5003), (700, 256, 1408), (2000, 384, 6000)])
def test_serving(m, k, v):
    x, r, w, head, t = _inputs(m, k, v)
    layer = FrozenFp8Linear(head)
    with torch.no_grad():
        q, s, h = rms_norm_fp8(x, w, r)
        logits = fp8_matmul(q, s, layer.weight_q, layer.weight_scale, out_dtype=torch.float32)
        out = token_log_probs(logits, t, top=4)
    check_gemm_status(torch.device("cuda", 0))
    a, b = dequantize_rows(q, s).double(), dequantize_blocks(layer.weight_q, layer.weight_scale).double()
    want, off = a @ b.t(), (k + 8) * E * (a.abs() @ b.abs().t()).amax(-1)
    assert ((logits - want).abs() <= off[:, None]).all()
    lp = torch.log_softmax(want, -1)
    assert ((out.log_prob - lp.gather(1, t[:, None])[:, 0]).abs() <= 2 * off + 1e-5).all()
    best = lp.topk(min(4, v), -1).values
    assert ((out.top_log_prob - best).abs() <= 2 * off[:, None] + 1e-5).all()
    assert ((lp.gather(1, out.top_token) - best).abs() <= 2 * off[:, None]).all()
    # the norm's 8-bit values are what quantising its fp32 result would give, to a rounding
    y, _ = rms_norm(x.float(), w, r.float())
    assert ((dequantize_rows(q, s) - y).abs() <= 2. ** -4 * y.abs() + 2. ** -9 * y.abs().amax(-1, keepdim=True)).float().mean() > .99


@pytest.mark.gpu
@pytest.mark.parametrize("m,k,v", [(5, 256, 8), (300, 520, 1000), (1500, 256, 2000)])
def test_training(m, k, v):
    x, r, w, head, t = _inputs(m, k, v)
    norm = FusedRMSNorm(k).cuda()
    with torch.no_grad():
        norm.weight.copy_(w)
    x.requires_grad_(True), head.requires_grad_(True)
    n, h = norm(x, r)
    logits = fp8_linear(n, head)
    n.retain_grad(), logits.retain_grad()
    out = token_log_probs(logits, t)
    (out.log_prob.mean() + .01 * out.entropy.mean() + h.float().mean()).backward()
    # scored tokens: the gradient in 64 bits at the logits that were scored
    z = logits.detach().double().requires_grad_(True)
    lp = torch.log_softmax(z, -1)
    ent = -(lp.exp() * lp).sum(-1)
    dz, = torch.autograd.grad(lp.gather(1, t[:, None]).mean() + .01 * ent.mean(), z)
    assert ((logits.grad.double() - dz).abs() <= 2. ** -8 * dz.abs() + 2e-5 / m).all()   # half a step of bf16, eps / 2 = 2^-8
    # the layer: both products on the quantised operands, the weight's gradient on bf16
    gq, wq = dequantize_rows(*quantize_rows(logits.grad)).double(), dequantize_blocks(*quantize_blocks(head)).double()
    dn, size = gq @ wq, gq.abs() @ wq.abs()
    assert ((n.grad.double() - dn).abs() <= 2. ** -8 * dn.abs() + (v + 8) * E * size).all()
    g, a = logits.grad.double(), n.detach().double()
    assert ((head.grad.double() - g.t() @ a).abs() <= (m + 8) * E * (g.abs().t() @ a.abs())).all()
    # the norm: rows' gradient with what flows along the residual
    hd = h.detach().double()
    rstd = (hd.square().mean(-1, keepdim=True) + norm.eps).rsqrt()
    u, c = n.grad.double() * w.double(), hd * rstd
    dx = rstd * (u - c * (u * c).mean(-1, keepdim=True)) + 1. / h.numel()
    scale = rstd * (u.abs() + c.abs() * (u * c).abs().mean(-1, keepdim=True)) + 1. / h.numel()
    # h.float().mean() hands on a bf16 gradient: one rounding more of 1 / numel
    assert ((x.grad.double() - dx).abs() <= 2. ** -8 * (dx.abs() + 1. / h.numel()) + 1e-5 * scale).all()


@pytest.mark.gpu
def test_two_streams_at_once():
    """Independent chains on two streams give what they give alone."""
    sets = [_inputs(300, 512, 4000), _inputs(33, 1024, 3000)]
    layers = [FrozenFp8Linear(s[3]) for s in sets]

    def run(i):
        x, r, w, _, t = sets[i]
        q, s, _ = rms_norm_fp8(x, w, r)
        return token_log_probs(fp8_matmul(q, s, layers[i].weight_q, layers[i].weight_scale), t, top=3)

    with torch.no_grad():
        want = [run(i) for i in range(2)]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(10):
            got = []
            for i, st in enumerate(streams):
                with torch.cuda.stream(st):
                    got.append(run(i))
            torch.cuda.synchronize()
            for a, b in zip(got, want):
                assert all(torch.equal(p, q) for p, q in zip(a, b))


def _check_alternatives(policy, inputs, logits, mask):
    actions, log_probs, entropy = policy.alternatives(inputs, 3, mask)
    use = torch.where(mask.any(-1, keepdim=True), mask, True)
    lp = torch.log_softmax(logits.float().masked_fill(~use, -torch.inf), -1)
    for i in range(mask.shape[0]):
        n = min(3, int(use[i].sum()))
        order = lp[i].argsort(descending=True, stable=True)[:n]
        assert actions[i, :n].tolist() == order.tolist() and (actions[i, n:] == -1).all()
        assert torch.allclose(log_probs[i, :n], lp[i, order], atol=1e-4)
    p = lp.exp()
    assert torch.allclose(entropy, -(p * lp.masked_fill(p == 0, 0.)).sum(-1), atol=1e-4)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_policies_name_their_alternatives(device):
    torch.manual_seed(0)
    mask = torch.rand(12, 8, device=device) < .5
    mask[0], mask[1] = False, torch.arange(8, device=device) == 4
    obs = torch.randn(12, 137, device=device)
    policy = ActorCritic(137, 8, "categorical").to(device)
    with torch.no_grad():
        _check_alternatives(policy, obs, policy(obs)[0], mask)
    with pytest.raises(ValueError):
        ActorCritic(35, 3, "continuous").to(device).alternatives(torch.randn(2, 35, device=device))
    policy = PerceptionActorCritic("residual_mlp", tensor_cores=False).to(device)
    with torch.no_grad():
        _check_alternatives(policy, {"scalars": obs}, policy({"scalars": obs})[0], mask)
