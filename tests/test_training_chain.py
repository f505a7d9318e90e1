"""Sampling, the group norm and AdamW as one training iteration uses them: a
small raster policy draws actions, is scored with a gradient, and takes a step,
each stage against 64-bit arithmetic on what the stage before it gave.

Tolerances: logits within 2^-24 times a few hundred (their layers' lengths) of
themselves; the gradient of every parameter within 1e-4 of its own norm, its
sums' lengths times 2^-24 with the norm's amplification of about ten; the step
as in test_adamw.py.
"""
import math

import pytest
import torch
from torch import nn

from autodrive_b200.meco.train import MecoConfig, train_meco
from autodrive_b200.ops.adamw import dequantize_moment
from autodrive_b200.ops.groupnorm import FusedGroupNorm, fuse_group_norms
from autodrive_b200.ops.sampling import sample_tokens
from autodrive_b200.ops.token_logprobs import token_log_probs
from autodrive_b200.train.optim import FusedAdamW
from autodrive_b200.train.sac import DiscreteSAC, make_sac_optimizers

DEVICES = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _policy(device):
    torch.manual_seed(7)
    return nn.Sequential(nn.Conv2d(6, 24, 3, padding=1), nn.GroupNorm(8, 24), nn.SiLU(), nn.AvgPool2d(4), nn.Flatten(),
                         nn.Linear(24 * 6 * 12, 8)).to(device)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("device", DEVICES)
def test_iterations(bits, device):
    with torch.backends.cudnn.flags(enabled=True, benchmark=False, deterministic=True, allow_tf32=False):
        policy = fuse_group_norms(_policy(device)).to(memory_format=torch.channels_last)
        assert isinstance(policy[1], FusedGroupNorm) and policy[1].activation == "silu"
        opt = FusedAdamW(policy.parameters(), lr=1e-2, max_grad_norm=.5, state_bits=bits, weight_decay=.01)
        moments = [[torch.zeros_like(p, dtype=torch.float64) for p in policy.parameters()] for _ in range(2)]
        for it in range(3):
            g = torch.Generator().manual_seed(it)
            x = torch.rand(40, 6, 25, 51, generator=g).to(device).contiguous(memory_format=torch.channels_last)
            mask = (torch.rand(40, 8, generator=g) < .7).to(device)
            mask[:, 0] = True
            u, adv = torch.rand(40, generator=g).to(device), torch.randn(40, generator=g).to(device)
            with torch.no_grad():
                drawn = sample_tokens(policy(x), u, mask, temperature=1., top_p=.95)
            logits = policy(x)
            scored = token_log_probs(logits, drawn.token, mask=mask)
            opt.zero_grad()
            (-(scored.log_prob * adv).mean() - .01 * scored.entropy.mean()).backward()

            # the same in 64 bits, at the parameters as they are
            exact = _policy("cpu").double()
            exact.load_state_dict({k: v.detach().cpu().double() for k, v in policy.state_dict().items()})
            z = exact(x.cpu().double())
            assert ((logits.detach().cpu().double() - z).abs() <= 1e-5 * (1 + z.abs())).all()
            lp = torch.log_softmax(z.masked_fill(~mask.cpu(), -torch.inf), -1)
            p = lp.exp()
            entropy = -(p * lp.masked_fill(~mask.cpu(), 0.)).sum(-1)
            order = p.sort(-1, descending=True).values
            least = .95 * torch.ones(40, 1, dtype=torch.float64)
            kept = ((order.cumsum(-1) - order) < least).sum(-1)
            assert (mask.cpu().gather(1, drawn.token.cpu()[:, None])).all()
            rank = (p > p.gather(1, drawn.token.cpu()[:, None]) * (1 + 1e-5)).sum(-1)
            assert (rank < kept + 1).all()
            grads = torch.autograd.grad(-(lp.gather(1, drawn.token.cpu()[:, None])[:, 0] * adv.cpu()).mean() - .01 * entropy.mean(),
                                        list(exact.parameters()))
            for a, b in zip(policy.parameters(), grads):
                assert (a.grad.cpu().double() - b).norm() <= 1e-4 * b.norm() + 1e-9

            # the step, from the gradients that were taken
            before = [q.detach().double() for q in policy.parameters()]
            gs = [q.grad.double() for q in policy.parameters()]
            opt.step()
            norm = torch.stack([t.square().sum() for t in gs]).sum().sqrt()
            assert abs(float(opt.last_norms[0]) / float(norm) - 1) <= 2. ** -22
            c = min(1., .5 / (float(norm) + 1e-6))
            for i, (q, q0, t) in enumerate(zip(policy.parameters(), before, gs)):
                m, v = moments[0][i], moments[1][i]
                m.mul_(.9).add_(.1 * c * t)
                v.mul_(.999).add_(.001 * (c * t) ** 2)
                want = q0 * (1 - 1e-4) - 1e-2 / (1 - .9 ** (it + 1)) * m / ((v / (1 - .999 ** (it + 1))).sqrt() + 1e-8)
                off = (q.detach().double() - want).abs()
                assert (off <= 40 * 2. ** -24 * 1e-2 * 10 + 1e-6 * q0.abs()).all()   # updates are at most ten times the rate
                if bits == 8:                                                      # the next step's are what is held
                    s = opt.state[q]
                    m.copy_(dequantize_moment(s["exp_avg"], s["exp_avg_scale"]))
                    v.copy_(dequantize_moment(s["exp_avg_sq"], s["exp_avg_sq_scale"]).square())


def test_trainers_take_the_options(tmp_path):
    """The commands and trainers that offer the operators run with them, and without them as they did."""
    plain = MecoConfig(track="A1", envs=2, updates=1, epochs=1, seed=1)
    assert plain.identity() == MecoConfig(track="A1", envs=2, updates=1, epochs=1, seed=1, optimizer="adam").identity()
    assert plain.identity() != MecoConfig(track="A1", envs=2, updates=1, epochs=1, seed=1, optimizer="fused").identity()
    policy, history = train_meco(MecoConfig(track="A1", envs=2, updates=1, epochs=1, seed=1, optimizer="fused8", fused_norms=True))
    assert len(history) == 1 and math.isfinite(history[0]["policy_loss"])
    assert any(isinstance(m, FusedGroupNorm) for m in policy.modules())
    other, _ = train_meco(plain)
    assert list(policy.state_dict()) == list(other.state_dict())
    agent = DiscreteSAC("baseline_mlp")
    opts = make_sac_optimizers(agent, 1e-3, "fused")
    assert all(isinstance(o, FusedAdamW) for o in opts.values())
    assert all(type(o) is torch.optim.Adam for o in make_sac_optimizers(agent, 1e-3).values())


@pytest.mark.gpu
def test_training_command_on_a_gpu():
    policy, history = train_meco(MecoConfig(track="A1", envs=4, updates=1, epochs=1, seed=1, device="cuda", optimizer="fused",
                                            fused_norms=True))
    assert math.isfinite(history[-1]["policy_loss"]) and all(p.isfinite().all() for p in policy.parameters())
