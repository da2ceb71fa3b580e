"""Global gradient norm and clipping against float64 (in place, and folded into FusedAdam's step), and the refusals.

The norm is summed in float64 and rounded once: 2^-24 relative, plus the square root's and the sum's float64 error (1e-13).  A clipped
element is g * coef, coef = max / (norm + 1e-6) in fp32 (three roundings, 2^-24 each, and the norm's own), one rounding of the product
and one to the element's type: (half a step of the type + 5 * 2^-24) |g coef|.  For bf16 tensors coef is rounded to bf16 before (2^-8 relative),
as torch does with them: twice half a step, and the product's bits are compared with torch's own."""
import math

import pytest
import torch

from dm_amd.optimizer import FusedAdam, clip_grad_norm_, grad_norm
from dm_amd.runtime import hip, ops

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def params_of(grads, dev):
    out = []
    for g in grads:
        p = torch.empty(g.shape, device=dev, dtype=g.dtype)
        p.grad = g.to(dev)
        out.append(p)
    return out


def norm64(grads, kind=2.0):
    v = torch.cat([g.detach().cpu().double().reshape(-1) for g in grads])
    return v.abs().max() if kind == math.inf else v.square().sum().sqrt()


def check_clip(before, params, norm, limit, kind=2.0):
    want = norm64(before, kind)
    assert norm.shape == () and norm.dtype == torch.float32
    assert abs(norm.double().cpu() - want) <= (2.0 ** -24 + 1e-12) * want
    coef = min(1.0, limit / (want.item() + 1e-6))
    for g, p in zip(before, params):
        w = g.double() * coef
        tol = (HALF_STEP[g.dtype] * (2.01 if g.dtype == torch.bfloat16 else 1) + 5 * 2.0 ** -24) * w.abs() + torch.finfo(g.dtype).smallest_normal * torch.finfo(g.dtype).eps
        assert ((p.grad.cpu().double() - w).abs() <= tol).all(), tuple(g.shape)


def make(sizes, kinds, seed=3, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(n, generator=g) * scale * 10.0 ** (i % 4 - 2)).to(kinds[i % len(kinds)]) for i, n in enumerate(sizes)]


SIZES = {"one": [1], "few": [3, 0, 17, 1, 4096, 4097], "odd": [1, 5, 7, 1023, 33333, 8, 131073], "many": [1 + 37 * i % 501 for i in range(700)],
         "large": [5_000_003, 2, 1_234_567]}


@pytest.mark.gpu
@pytest.mark.parametrize("kinds", [(torch.float32,), (torch.bfloat16,), (torch.float16, torch.float32, torch.bfloat16)])
@pytest.mark.parametrize("sizes", sorted(SIZES))
@pytest.mark.parametrize("kind", [2.0, math.inf])
def test_clip_against_float64(dev, sizes, kinds, kind):
    before = make(SIZES[sizes], kinds)
    for limit in (0.5, 1e9, 0.0):
        ps = params_of(before, dev)
        assert torch.equal(grad_norm(ps, kind).cpu(), grad_norm(ps, kind).cpu())
        norm = clip_grad_norm_(ps, limit, kind)
        check_clip(before, ps, norm, limit, kind)


@pytest.mark.gpu
def test_clip_views_of_one_buffer(dev):
    """gradients that are views of one buffer, at odd offsets: neighbours, gaps whose contents do not count and stay, one gradient twice"""
    for t in (torch.float32, torch.bfloat16):
        buf = torch.full((20000,), float("nan"), device=dev, dtype=t)
        spans = [(1, 100), (101, 4099), (4200, 1), (4203, 8000), (12203, 5), (15000, 4999)]
        params = []
        for i, (o, n) in enumerate(spans):
            buf[o:o + n] = torch.randn(n, device=dev, generator=torch.Generator(dev).manual_seed(i))
            p = torch.empty(n, device=dev, dtype=t)
            p.grad = buf[o:o + n]
            params.append(p)
        before = [p.grad.cpu().clone() for p in params]
        norm = clip_grad_norm_(params + [params[1]], 2.0)
        check_clip(before, params, norm, 2.0)
        inside = torch.zeros(20000, dtype=torch.bool)
        for o, n in spans:
            inside[o:o + n] = True
        assert buf.cpu()[~inside].isnan().all()


@pytest.mark.gpu
def test_clip_layouts_and_extremes(dev):
    g = torch.randn(6, 5, 4, 3).to(dev)
    for t in (g.permute(2, 0, 3, 1), g.to(memory_format=torch.channels_last)):        # dense in another order
        p = torch.empty_like(t)
        p.grad = t.clone(memory_format=torch.preserve_format)
        before = p.grad.cpu().clone()
        check_clip([before], [p], clip_grad_norm_(p, 1.0), 1.0)
    big = torch.tensor([3e38, -3e38, 1e20])                                            # squares overflow in 32 bits
    p = params_of([big], dev)
    norm = clip_grad_norm_(p, 1.0)
    check_clip([big], p, norm, 1.0) if math.isfinite(norm.item()) else None
    assert math.isinf(norm.item()) == bool(torch.isinf(norm64([big]).float()))
    p = params_of([torch.tensor([1e30, 2e30])], dev)
    check_clip([torch.tensor([1e30, 2e30])], p, clip_grad_norm_(p, 1.0), 1.0)
    tiny = torch.tensor([1e-30, 1e-38])                                                # squares underflow in 32 bits
    assert abs(grad_norm(params_of([tiny], dev)).item() - 1e-30) < 1e-36
    for bad in (float("nan"), float("inf")):
        for kind in (2.0, math.inf):
            p = params_of([torch.tensor([1.0, bad, 2.0]), torch.ones(2)], dev)
            want = torch.nn.utils.clip_grad_norm_(q := params_of([torch.tensor([1.0, bad, 2.0]), torch.ones(2)], "cpu"), 1.0, kind)
            got = clip_grad_norm_(p, 1.0, kind)
            assert torch.equal(torch.isnan(got.cpu()), torch.isnan(want)) and torch.equal(torch.isinf(got.cpu()), torch.isinf(want))
            for a, b in zip(p, q):
                assert torch.equal(a.grad.cpu().isnan(), b.grad.isnan()) and torch.equal(a.grad.cpu().nan_to_num(7), b.grad.nan_to_num(7))
            p = params_of([torch.tensor([1.0, bad, 2.0])], dev)
            with pytest.raises(RuntimeError, match="non-finite"):
                clip_grad_norm_(p, 1.0, kind, error_if_nonfinite=True)
            assert p[0].grad[0].item() == 1.0
    assert clip_grad_norm_([torch.empty(3, device=dev)], 1.0).item() == 0.0           # no gradients
    p = torch.empty(0, device=dev)
    p.grad = torch.empty(0, device=dev)
    assert clip_grad_norm_([p], 1.0).item() == 0.0                                     # an empty one


@pytest.mark.gpu
def test_clip_multiplies_as_torch_does(dev):
    """fp32 and bf16 gradients, clipped twice in a row: given the norm, the same bits as torch's tensor.mul_(factor on the device).  (The norm's own
    bits are not torch's, which rounds every tensor's norm before it takes the norm of those.)"""
    for t in (torch.float32, torch.bfloat16):
        ps = params_of(make([64, 33, 4097], (t,)), dev)
        for limit in (0.37, 0.1):
            before = [p.grad.clone() for p in ps]
            factor = (limit / (clip_grad_norm_(ps, limit) + 1e-6)).clamp(max=1.0)
            for p, x in zip(ps, before):
                assert torch.equal(p.grad, x.mul_(factor))


@pytest.mark.gpu
def test_clip_captured(dev):
    src = [t.to(dev) for t in make([100, 4097, 3], (torch.float32, torch.bfloat16))]
    ps = params_of(src, dev)
    grad_norm(ps)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        norm = clip_grad_norm_(ps, 0.7)
    for k in range(4):
        fresh = [t * (k + 1) for t in src]
        for p, t in zip(ps, fresh):
            p.grad.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        check_clip([t.cpu() for t in fresh], ps, norm, 0.7)


def adam64(p, g, m, v, step, lr, b1, b2, eps, wd):
    g = g + wd * p
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p - lr / (1 - b1 ** step) * m / ((v / (1 - b2 ** step)).sqrt() + eps), m, v


@pytest.mark.gpu
@pytest.mark.parametrize("flat", [False, True])
@pytest.mark.parametrize("limit,grad_scale", [(0.3, 1.0), (1e6, 1.0), (0.3, 0.25)])
def test_fused_adam_clips(dev, flat, limit, grad_scale):
    """three steps against float64 Adam on clipped gradients; .grad is left alone, grad_norm is the norm before clipping.  An update is
    lr times a quotient below 1 / sqrt(1 - b2): its fp32 error, 32 roundings of 2^-24 and powf's, is held to 1e-5 lr, the weights' own
    rounding is 2^-24 each step."""
    sizes = [7, 64, 1001, 3, 4096]
    g = torch.Generator().manual_seed(9)
    ps = [torch.randn(n, generator=g).to(dev).requires_grad_() for n in sizes]
    offs, total = [], 0
    for n in sizes:
        offs.append(total)
        total += (n + 3) // 4 * 4
    lr, b1, b2, eps, wd = 1e-2, 0.9, 0.999, 1e-8, 0.01
    opt = FusedAdam(ps, lr=lr, weight_decay=wd, max_grad_norm=limit)
    want = [(p.detach().cpu().double(), torch.zeros(n).double(), torch.zeros(n).double()) for p, n in zip(ps, sizes)]
    for step in (1, 2, 3):
        grads = [torch.randn(n, generator=g) * (i + 1) for i, n in enumerate(sizes)]
        store = torch.full((total,), float("nan"), device=dev) if flat else None     # what lies between the gradients does not count
        if flat:
            for o, n in zip(offs, sizes):
                store[o + n:o + (n + 3) // 4 * 4] = 123.0
        for p, t, o in zip(ps, grads, offs):
            p.grad = store[o:o + t.numel()].copy_(t) if flat else t.to(dev)
        opt.step(grad_scale=grad_scale)
        norm = norm64(grads)
        assert abs(opt.grad_norm.item() - norm) <= 2.0 ** -23 * norm
        coef = min(1.0, limit / (norm.item() * grad_scale + 1e-6)) * grad_scale
        want = [adam64(p, t.double() * coef, m, v, step, lr, b1, b2, eps, wd) for (p, m, v), t in zip(want, grads)]
        for p, t, w in zip(ps, grads, want):
            assert torch.equal(p.grad.cpu(), t)
            tol = 1e-5 * lr * step * (1 / math.sqrt(1 - b2)) + step * 2.0 ** -24 * w[0].abs()
            assert ((p.detach().cpu().double() - w[0]).abs() <= tol).all(), step


@pytest.mark.gpu
def test_train_drivers_clip(dev):
    """the pipelined step (whose optimizer step is otherwise taken in two pieces) and the single-graph step with max_grad_norm: the same
    weights, the norm of the gradients they step on, and a weight change that clipping bounds"""
    from dm_amd.losses.ELBO import ELBOLoss
    from dm_amd.neural_nets.denoise_models import ddpm as dm_ddpm, unets as dm_unets
    from dm_amd.runtime.graphs import PipelinedTrainStep
    from oracle import ref_cpu as O
    from oracle.noise import hash_normal, hash_uniform
    kw = dict(stages_channels=[32, 64, 128, 256], expand_factor=2, drop_p=0.0, T=120, beta=0.25, t_embed_dim=32, activation="gelu",
              base_groups_norm=4, initializer="he_normal", dtype=None)
    m = dm_ddpm.DDPM(dm_unets.BaseUNet, **kw, is_conditional=False, img_channels=1, reconstruction_method="mse", latent_dim=512, device=dev).to(dev)
    m.load_state_dict(O.hash_params(O.UNetCfg(img_channels=1, drop_p=0.0), head_gain=0.3))
    x0 = (hash_uniform((4, 1, 32, 32), 1) * 2 - 1).to(dev)
    t, noise = torch.tensor([5, 90, 30, 119], device=dev), hash_normal((4, 1, 32, 32), 2).to(dev)
    opt = FusedAdam(m.parameters(), lr=1e-3, max_grad_norm=0.05)
    step = PipelinedTrainStep(m, ELBOLoss("mse"), opt, x0, t=t, noise=noise)
    with pytest.raises(RuntimeError, match="step in pieces"):
        opt.step_ranges([(0, 4)], True)
    for _ in range(3):
        before = [p.detach().clone() for p in m.parameters()]
        step.replay()
        torch.cuda.synchronize()
        grads = [p.grad.cpu() for p in m.parameters()]
        want = norm64(grads)
        assert want > 0.05 and abs(opt.grad_norm.item() - want) <= 2.0 ** -23 * want
        assert any(not torch.equal(a, p.detach()) for a, p in zip(before, m.parameters()))


def test_clip_refusals_without_a_gpu():
    import ctypes
    p = torch.zeros(3)
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="HIP kernels only"):
        clip_grad_norm_([p], 1.0)
    with pytest.raises(ValueError, match="norm_type"):
        clip_grad_norm_([p], 1.0, norm_type=1.0)
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            clip_grad_norm_([p], bad)
        with pytest.raises(ValueError, match="max_grad_norm"):
            FusedAdam([p], max_grad_norm=bad)
    import numpy as np
    k = np.array([2, 2], dtype=np.uint8)
    with pytest.raises(ValueError, match="overlap"):
        ops._merge_spans(np.array([4096, 4104], dtype=np.uint64), np.array([4, 4]), k)
    at, n, kind = ops._merge_spans(np.array([4112, 4096, 4096, 8192], dtype=np.uint64), np.array([4, 4, 4, 0]), np.array([2, 2, 2, 0], dtype=np.uint8))
    assert at.tolist() == [4096] and n.tolist() == [8] and kind.tolist() == [2]
    f, buf = hip.lib().ddpm_grad_norm, ctypes.c_void_p(4096)
    arr = lambda a, t: np.array(a, dtype=t).ctypes.data_as(ctypes.c_void_p)  # noqa: E731
    good = dict(ptr=[4096], n=[4], k=[2], norm=0, clip=1, limit=1.0, out=buf, work=buf)
    for bad, why in ((dict(ptr=[4098]), b"aligned"), (dict(ptr=[0]), b"not there"), (dict(n=[-1]), b"not there"), (dict(k=[3]), b"element type"), (dict(norm=2), b"norm"),
                     (dict(limit=-1.0), b"max_norm"), (dict(limit=float("nan")), b"max_norm"), (dict(out=None), b"null"), (dict(work=None), b"null")):
        a = dict(good, **bad)
        rc = f(arr(a["ptr"], np.uint64), arr(a["n"], np.int64), arr(a["k"], np.uint8), 1, a["norm"], a["clip"], a["limit"], a["out"], a["work"], None)
        assert rc != 0 and why in hip.lib().ddpm_last_error(), bad
    assert f(None, None, None, 1, 0, 0, 0.0, buf, buf, None) != 0
