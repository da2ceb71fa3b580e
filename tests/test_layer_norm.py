"""Layer norm (forward, backward, the parameters' gradients) against float64, and its refusals.

Tolerances, per element, u = half a step of the output's type relative to the value (2^-8 bf16, 2^-11 fp16, 2^-24 fp32):
  y = xhat * w + b: one final rounding, u * |y|, and the fp32 evaluation before it.  The mean of C numbers, summed in at most 32
  dependent steps, is off by at most 40 * 2^-24 * mean|x|, which xhat = (x - mean) * rstd carries times rstd; the deviations'
  relative errors add 2^-24 * 50 to |xhat|.  Together: u |y| + 2^-18 * |w| * (|xhat| + rstd * mean|x|).
  dx: u |dx| + 2^-17 * rstd * (1 + rstd * mean|x|) * (max|g| + max|xhat| * mean|g xhat|), the same errors through g - c1 - xhat c2.
  dw, db: sums of n terms in fp32, partial sums of at most n / 16 + 64 dependent steps: bounded by 2^-24 * n * sum|terms| in the worst
  case and, rounding errors being of either sign, by 2^-24 * 4 * sqrt(n) * ... in practice; used here: 2^-24 * (n + 64) * mean of
  |terms| * sqrt(n) + the error of xhat (2^-18 (|xhat| + rstd mean|x|)) summed over |dy|."""
import pytest
import torch

from dm_amd.neural_nets import sequence
from dm_amd.runtime import hip, ops

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}


def inputs(rows, c, dtype, seed=1, pad=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    store = torch.zeros(rows, c + pad, dtype=dtype)
    store[:, :c] = n(rows, c) * (n(rows, 1).abs() + 0.1) + 2 * n(rows, 1)
    return store, 1 + 0.2 * n(c), 0.3 * n(c), n(rows, c).to(dtype)


def reference(x, w, b, dy, eps=1e-5):
    x, dy = x.double(), dy.double()
    w, b = (torch.ones(x.shape[1]) if w is None else w).double(), (torch.zeros(x.shape[1]) if b is None else b).double()
    mean = x.mean(1, keepdim=True)
    rstd = ((x - mean).square().mean(1, keepdim=True) + eps).rsqrt()
    h = (x - mean) * rstd
    g = dy * w
    c2 = (g * h).mean(1, keepdim=True)
    dx = rstd * (g - g.mean(1, keepdim=True) - h * c2)
    err_h = 2.0 ** -18 * (h.abs() + rstd * x.abs().mean(1, keepdim=True))
    n = max(1, x.shape[0])
    acc = lambda t: 2.0 ** -24 * (n + 64) / n * t.abs().sum(0) * n ** 0.5  # noqa: E731
    amax = lambda t: t.abs().amax(1, keepdim=True)  # noqa: E731
    tol_dx = 2.0 ** -17 * rstd * (1 + rstd * x.abs().mean(1, keepdim=True)) * (amax(g) + amax(h) * (g * h).abs().mean(1, keepdim=True)) if x.shape[0] else dx
    return dict(y=h * w + b, dx=dx, dw=(dy * h).sum(0), db=dy.sum(0)), dict(
        y=err_h * w.abs() + 2.0 ** -22 * b.abs(), dx=tol_dx, dw=acc(dy * h) + (dy.abs() * err_h).sum(0), db=acc(dy))


def check(got, want, tol, dtype):
    got, err = got.detach().cpu().double(), HALF_STEP[dtype] * want.abs() * 1.0001 + tol
    if dtype != torch.float32:
        err = err + torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps        # (a result below the normal range: half its spacing)
    bad = (got - want).abs() > err
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / err).max():.3g} of the tolerance"


# one element, less than a vector, each lane-group width, its borders, workgroup rows, odd widths, the largest
WIDTHS = [1, 2, 3, 8, 31, 32, 64, 72, 255, 256, 500, 512, 1000, 1001, 1024, 1025, 1032, 2048, 2056, 4096, 4097, 5000, 8192]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("c", WIDTHS)
@pytest.mark.parametrize("rows,pad", [(1, 0), (37, 3), (2500, 8)])
def test_layer_norm_against_float64(dev, dtype, c, rows, pad):
    if rows == 2500 and c > 1100:
        rows = 1100
    store, w, b, dy = inputs(rows, c, dtype, seed=c, pad=pad)
    want, tol = reference(store[:, :c], w, b, dy)
    x = store.to(dev)[:, :c].requires_grad_()
    wd, bd = w.to(dev).requires_grad_(), b.to(dev).requires_grad_()
    y = sequence.layer_norm(x, wd, bd)
    assert y.dtype == dtype and y.shape == x.shape
    check(y, want["y"], tol["y"], dtype)
    dx, dw, db = torch.autograd.grad(y, [x, wd, bd], dy.to(dev))
    check(dx, want["dx"], tol["dx"], dtype)
    check(dw, want["dw"], tol["dw"], torch.float32)
    check(db, want["db"], tol["db"], torch.float32)
    again = torch.autograd.grad(sequence.layer_norm(x, wd, bd), [x, wd, bd], dy.to(dev))
    assert all(torch.equal(a, g) for a, g in zip(again, (dx, dw, db)))              # a fixed order of summation


@pytest.mark.gpu
def test_layer_norm_gradient_is_the_derivative(dev):
    """central differences of a float64 evaluation, at the gradient's direction: (f(x + h d) - f(x - h d)) / 2h"""
    store, w, b, dy = inputs(6, 40, torch.float32)
    f = lambda x, w, b: (reference(x, w, b, dy)[0]["y"] * dy.double()).sum()  # noqa: E731
    leaves = [t.to(dev).requires_grad_() for t in (store, w, b)]
    grads = [g.cpu().double() for g in torch.autograd.grad(sequence.layer_norm(*leaves), leaves, dy.to(dev))]
    base, h = [store.double(), w.double(), b.double()], 1e-4
    for i, g in enumerate(grads):
        d = g / g.norm()
        up, down = ([t + (s * h * d if j == i else 0) for j, t in enumerate(base)] for s in (1, -1))
        slope = (f(*up) - f(*down)) / (2 * h)
        assert abs(slope - g.norm()) <= 1e-5 * g.norm()          # (differences: h^2 / 6 of a third derivative of order one, ~1e-8; fp32 gradients 1e-6)


@pytest.mark.gpu
def test_layer_norm_hard_rows(dev):
    """rows without variance, a row far from zero, a row with an infinity or a NaN, which must not reach its neighbours"""
    x = torch.randn(6, 300, generator=torch.Generator().manual_seed(2))
    x[1] = 3.0
    x[2] += 1e4
    x[3, 7], x[4, 0] = float("inf"), float("nan")
    y = sequence.layer_norm(x.to(dev)).cpu()
    assert y[3].isnan().all() and y[4].isnan().all()
    want, tol = reference(x, None, None, torch.zeros_like(x))
    for r in (0, 1, 2, 5):
        check(y[r], want["y"][r], tol["y"][r], torch.float32)


@pytest.mark.gpu
def test_layer_norm_shapes_and_absent_parts(dev):
    x = torch.randn(2, 5, 48, device=dev, dtype=torch.bfloat16)
    w = torch.randn(48, device=dev)
    assert torch.equal(sequence.layer_norm(x, w).view(10, 48), sequence.layer_norm(x.reshape(10, 48), w, torch.zeros(48, device=dev)))
    t = x.transpose(0, 1)                                       # rows in another order
    assert torch.equal(sequence.layer_norm(t), sequence.layer_norm(t.contiguous()))
    s = x.transpose(1, 2)                                       # rows that are not contiguous
    assert torch.equal(sequence.layer_norm(s), sequence.layer_norm(s.contiguous()))
    e = x[:, :1].expand(2, 5, 48)                               # rows that lie on each other
    assert torch.equal(sequence.layer_norm(e), sequence.layer_norm(e.contiguous()))
    leaf = x.float().requires_grad_()
    sequence.layer_norm(leaf, w).sum().backward()               # an expanded gradient
    want = torch.autograd.grad(sequence.layer_norm(leaf, w), leaf, torch.ones(2, 5, 48, device=dev))[0]
    assert torch.equal(leaf.grad, want)
    wl = w.clone().requires_grad_()                             # only the weight's gradient
    y = sequence.layer_norm(torch.zeros(0, 48, device=dev), wl)
    assert y.shape == (0, 48)
    y.sum().backward()
    assert torch.equal(wl.grad, torch.zeros_like(wl))           # no rows: a zero gradient, written
    odd = torch.randn(64 * 49 + 1, device=dev)[1:].view(64, 49)[:, :48]               # rows that start off the vector alignment
    # (moved element by element: another order of summation than the aligned copy's, so the bits may differ; both within the bound above)
    want, tol = reference(odd.cpu(), None, None, torch.zeros(64, 48))
    check(sequence.layer_norm(odd), want["y"], tol["y"], torch.float32)
    check(sequence.layer_norm(odd.contiguous()), want["y"], tol["y"], torch.float32)


@pytest.mark.gpu
def test_layer_norm_module_and_graph(dev):
    """the module's parameters under nn.LayerNorm's names; forward and backward captured together and replayed on new inputs"""
    m = sequence.LayerNorm(96, device=dev)
    ref = torch.nn.LayerNorm(96)
    with torch.no_grad():
        ref.weight.normal_(1, 0.2)
        ref.bias.normal_(0, 0.2)
    m.load_state_dict(ref.state_dict())
    x, dy = (torch.randn(33, 96, device=dev, dtype=torch.bfloat16) for _ in range(2))

    def body():
        leaf = x.detach().requires_grad_()
        y = m(leaf)
        return [y.detach()] + list(torch.autograd.grad(y, [leaf, m.weight, m.bias], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = body()
    for k in range(4):
        x.normal_()
        dy.normal_()
        g.replay()
        torch.cuda.synchronize()
        for a, b in zip(out, body()):
            assert torch.equal(a, b), k


@pytest.mark.gpu
def test_capture_beside_a_living_graph_is_refused(dev):
    """a graph of the same parameters that an eager call on the default stream made and that is still alive: a captured backward pass would
    make the default stream wait for the capture.  It is refused before that; without the graph it goes through"""
    m = sequence.LayerNorm(64, device=dev)
    x = torch.randn(8, 64, device=dev)
    old = m(x)
    assert not torch.cuda.is_current_stream_capturing()
    with torch.no_grad():                                                         # (a capture without a backward pass is free to go on)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            m(x)
    with pytest.raises(RuntimeError, match="is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(m(x), [m.weight, m.bias], x)
    torch.cuda.synchronize()
    want = torch.autograd.grad(old, [m.weight, m.bias], x)
    del old
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = torch.autograd.grad(m(x), [m.weight, m.bias], x)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_layer_norm_refusals_without_a_gpu():
    with pytest.raises(RuntimeError, match="HIP kernels only"):
        sequence.layer_norm(torch.zeros(2, 8))
    with pytest.raises(ValueError, match="last axis"):
        sequence.layer_norm(torch.zeros(2, 0))
    with pytest.raises(ValueError, match="last axis"):
        sequence.LayerNorm(8)(torch.zeros(2, 9))
    x, d = torch.zeros(4, 8), torch.zeros(4, 2)
    with pytest.raises(ValueError, match="type torch.int32"):
        ops.layer_norm_forward(x.int(), None, None)
    for w in (torch.ones(7), torch.ones(8).double(), torch.ones(16)[::2]):
        with pytest.raises(ValueError, match="contiguous float32 tensors of 8"):
            ops.layer_norm_forward(x, w, None)
    run = hip.lib().ddpm_layer_norm_forward
    desc = lambda **k: hip.LayerNormDesc(**dict(dict(x=x.data_ptr(), y=x.data_ptr(), rows=4, C=8, ldx=8, ldy=8, dtype=2, eps=1e-5), **k))  # noqa: E731
    import ctypes
    for bad, why in ((dict(C=8193), b"8193"), (dict(C=0), b"0 elements"), (dict(rows=-1), b"-1 rows"), (dict(ldx=7), b"row stride"), (dict(ldy=0), b"row stride"),
                     (dict(dtype=3), b"element type"), (dict(x=None), b"null"), (dict(y=None), b"null"), (dict(eps=-1.0), b"eps")):
        assert run(ctypes.byref(desc(**bad)), None) != 0 and why in hip.lib().ddpm_last_error(), bad
    assert run(None, None) != 0
    back = desc(dy=x.data_ptr(), lddy=8, stats=d.data_ptr(), dw=x.data_ptr())
    assert hip.lib().ddpm_layer_norm_backward(ctypes.byref(back), None) != 0 and b"part" in hip.lib().ddpm_last_error()
    assert hip.lib().ddpm_layer_norm_part_rows(ctypes.byref(desc(dy=None))) == -1
