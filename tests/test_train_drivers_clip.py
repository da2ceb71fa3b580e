"""The train drivers with an optimizer that clips: what a replayed step makes of weights and moments, and a limit that changes after the capture."""
import math

import pytest
import torch

from dm_amd.losses.ELBO import ELBOLoss
from dm_amd.neural_nets.denoise_models import ddpm as dm_ddpm, unets as dm_unets
from dm_amd.optimizer import FusedAdam
from dm_amd.runtime.graphs import GraphedTrainStep, PipelinedTrainStep
from oracle import ref_cpu as O
from oracle.noise import hash_normal, hash_uniform

DRIVERS = {"single graph": GraphedTrainStep, "pipelined": PipelinedTrainStep}


def driver(kind, dev, limit):
    kw = dict(stages_channels=[32, 64, 128, 256], expand_factor=2, drop_p=0.0, T=120, beta=0.25, t_embed_dim=32, activation="gelu",
              base_groups_norm=4, initializer="he_normal", dtype=None)
    m = dm_ddpm.DDPM(dm_unets.BaseUNet, **kw, is_conditional=False, img_channels=1, reconstruction_method="mse", latent_dim=512, device=dev).to(dev)
    m.load_state_dict(O.hash_params(O.UNetCfg(img_channels=1, drop_p=0.0), head_gain=0.3))
    x0 = (hash_uniform((4, 1, 32, 32), 1) * 2 - 1).to(dev)
    fixed = dict(t=torch.tensor([5, 90, 30, 119], device=dev), noise=hash_normal((4, 1, 32, 32), 2).to(dev)) if kind == "pipelined" else {}
    opt = FusedAdam(m.parameters(), lr=1e-3, max_grad_norm=limit)
    return m, opt, DRIVERS[kind](m, ELBOLoss("mse"), opt, x0, **fixed)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(DRIVERS))
@pytest.mark.parametrize("limit", [1e-9, 1e6])             # (gradients of random timesteps differ by orders of magnitude)
def test_replayed_steps_take_clipped_gradients(dev, kind, limit):
    """weights and first moments after each replay against float64 Adam on gradients times min(1, limit / (norm + 1e-6)), from the state before.
    m' = b1 m + (1 - b1) c g in fp32: 16 roundings (b1, 1 - b1, c and its norm, products, sum).  The weights as in test_grad_clip.py: an update's
    fp32 error is held to 1e-5 lr / sqrt(1 - b2), the weight's own rounding is 2^-24."""
    m, opt, step = driver(kind, dev, limit)
    lr, b1, b2, eps = 1e-3, 0.9, 0.999, 1e-8
    for _ in range(3):
        state = opt.state_dict()["state"]
        before = [(p.detach().double(), state[i]["exp_avg"].double(), state[i]["exp_avg_sq"].double()) for i, p in enumerate(m.parameters())]
        count = int(state[0]["step"].item()) + 1
        step.replay()
        torch.cuda.synchronize()
        grads = [p.grad.double() for p in m.parameters()]
        norm = math.sqrt(sum(g.square().sum().item() for g in grads))
        assert (norm > limit) == (limit < 1) and abs(opt.grad_norm.item() - norm) <= 2.0 ** -23 * norm
        c, state = min(1.0, limit / (norm + 1e-6)), opt.state_dict()["state"]
        for i, (p, g, (w, a, v)) in enumerate(zip(m.parameters(), grads, before)):
            first, second = b1 * a + (1 - b1) * c * g, b2 * v + (1 - b2) * (c * g).square()
            err = (state[i]["exp_avg"].double() - first).abs()
            assert (err <= 16 * 2.0 ** -24 * (b1 * a.abs() + (1 - b1) * c * g.abs()) + 1e-38).all(), i
            new = w - lr / (1 - b1 ** count) * first / ((second / (1 - b2 ** count)).sqrt() + eps)
            assert ((p.detach().double() - new).abs() <= 1e-5 * lr / math.sqrt(1 - b2) + 2.0 ** -24 * new.abs()).all(), i


@pytest.mark.gpu
@pytest.mark.parametrize("kind", sorted(DRIVERS))
@pytest.mark.parametrize("limit,other", [(0.05, 0.1), (0.05, None), (None, 0.05)])
def test_a_limit_that_changes_after_the_capture_is_refused(dev, kind, limit, other):
    """the captured step has the limit it was captured with: another one would have no effect"""
    m, opt, step = driver(kind, dev, limit)
    step.replay()
    opt.max_grad_norm = other
    torch.cuda.synchronize()
    before = [p.detach().clone() for p in m.parameters()]
    with pytest.raises(RuntimeError, match="max_grad_norm.*capture"):
        step.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, p) for a, p in zip(before, m.parameters()))
    opt.max_grad_norm = limit
    step.replay()
    torch.cuda.synchronize()
    assert any(not torch.equal(a, p) for a, p in zip(before, m.parameters()))
