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


def test_the_clipped_step_runs_on_its_parameters_device(monkeypatch):
    """parameters on another device than the current one: the norm, the update that reads it and what they allocate all go to theirs (no GPU: the launches
    are only written down)"""
    import contextlib

    from dm_amd.optimizer import FusedAdam, optimizer as module
    opt = FusedAdam([torch.zeros(4, requires_grad=True)], max_grad_norm=1.0)
    flat = torch.zeros(4)
    for name in ("_flat", "_m", "_v", "_g", "_lr", "_step", "grad_norm"):
        setattr(opt, name, flat)
    opt._ema, opt._lr_host, opt._total, opt._offs = None, 1e-3, 4, [0]
    opt._span_off, opt._span_n, opt._span_kind = (torch.zeros(1, dtype=torch.int64).numpy().astype("uint64") for _ in range(3))
    here, seen = [], []

    @contextlib.contextmanager
    def on_device_of(t):
        here.append(t)
        yield
        here.pop()

    monkeypatch.setattr(module.hip, "on_device_of", on_device_of)
    monkeypatch.setattr(module.hip, "stream", lambda *a: seen.append(("stream", list(here))) or 0)
    monkeypatch.setattr(module.hip, "call", lambda name, *a: seen.append((name, list(here))))
    monkeypatch.setattr(module.ops, "launch_grad_norm", lambda *a: seen.append(("norm", list(here))))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    opt.step()
    opt.max_grad_norm = None
    opt.step()
    opt.step_ranges([(0, 4)], True)
    assert {name for name, _ in seen} == {"norm", "stream", "ddpm_adam_step_clipped", "ddpm_adam_step", "ddpm_adam_step_range"}
    assert all(any(t is flat for t in where) for _, where in seen), seen
