"""Forward-mode derivatives through the sequence layers: refused, not lost (a dual tensor asks for no gradient, so it looks like plain inference)."""
import pytest
import torch
from torch.autograd import forward_ad

from dm_amd.neural_nets import sequence


def duals(dev):
    """per operator: its name and, for each input that may carry a tangent, a call in which that one does"""
    x, w, b = (torch.randn(*s, device=dev) for s in ((4, 8), (8,), (8,)))
    q, k, v = (torch.randn(5, h, 16, device=dev).bfloat16() for h in (2, 1, 1))
    table, buckets = torch.randn(8, 2, device=dev), sequence.relative_position_buckets(8, 6).to(dev)
    ends = torch.tensor([0, 5], dtype=torch.int32, device=dev)
    dual = lambda t: forward_ad.make_dual(t, torch.ones_like(t))  # noqa: E731
    norm = [x, w, b]
    att = [q, k, v, table]
    for i in range(3):
        args = [dual(t) if j == i else t for j, t in enumerate(norm)]
        yield "layer_norm", lambda args=args: sequence.layer_norm(*args)
    for i in range(4):
        args = [dual(t) if j == i else t for j, t in enumerate(att)]
        yield "packed_attention", lambda args=args: sequence.packed_attention(*args[:3], ends, bias_table=args[3], bias_buckets=buckets)


def refused(dev):
    with forward_ad.dual_level():
        for name, call in duals(dev):
            with pytest.raises(NotImplementedError, match=f"{name}.*forward-mode"):
                call()


def test_tangents_are_refused_without_a_gpu():
    refused("cpu")


@pytest.mark.gpu
def test_tangents_are_refused(dev):
    refused(dev)
    x = torch.randn(4, 8, device=dev)
    with pytest.raises(NotImplementedError, match="forward-mode"):
        torch.func.jvp(sequence.layer_norm, (x,), (x,))
    with pytest.raises(NotImplementedError, match="forward-mode"), forward_ad.dual_level():       # with a reverse-mode graph as well
        sequence.layer_norm(forward_ad.make_dual(x.clone().requires_grad_(), x))


@pytest.mark.gpu
def test_calls_without_a_tangent_go_on_inside_a_level(dev):
    x = torch.randn(4, 8, device=dev)
    want = sequence.layer_norm(x)
    with forward_ad.dual_level():
        assert torch.equal(sequence.layer_norm(x), want)
        assert torch.equal(sequence.layer_norm(x.clone().requires_grad_()), want)
