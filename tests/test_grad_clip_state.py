"""What clipping leaves behind beside the clipped numbers: the gradients' versions."""
import pytest
import torch

from dm_amd.optimizer import clip_grad_norm_, grad_norm


def parameter(dev, *shape):
    p = torch.zeros(*shape, device=dev, requires_grad=True)
    p.grad = torch.randn(*shape, device=dev)
    return p


@pytest.mark.gpu
def test_clipped_gradients_count_as_modified(dev):
    """as after torch's own in-place operations: a graph that saved a gradient refuses to go on with the clipped one"""
    ps = [parameter(dev, 5), parameter(dev, 70, 3)]
    w = torch.randn(5, device=dev, requires_grad=True)
    penalty = (w * ps[0].grad).sum()                           # saves the gradient
    before = [p.grad._version for p in ps]
    grad_norm(ps)
    assert [p.grad._version for p in ps] == before             # (only read)
    clip_grad_norm_(ps, 0.1)
    assert all(p.grad._version > v for p, v in zip(ps, before))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        penalty.backward()
    with torch.inference_mode():                               # gradients without a version are clipped as well
        q = torch.empty(3, device=dev)
        q.grad = torch.full((3,), 2.0, device=dev)
    assert abs(clip_grad_norm_(q, 1.0).item() - 12 ** 0.5) < 1e-6 and abs(q.grad.norm().item() - 1) < 1e-5
