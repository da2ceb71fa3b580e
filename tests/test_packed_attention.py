"""Attention over packed sequences, forward and backward, with and without the relative position bias, against float64, and its refusals.

Tolerances, per element, from worst cases of every rounding (u = half a step of the 16-bit type: 2^-8 bf16, 2^-11 fp16):
  score: a product of `width` terms and a scale in fp32, off by at most e = (width + 8) 2^-24 scale sum|q k| + 2^-22 |score|; a
  probability (numerator and normaliser) then by 2 e + 2^-19 relative.
  o: p rounded to 16 bits (u; fp16 also half its smallest spacing, 2^-25, on numbers whose maximum is at least 1), a sum of n terms in
  fp32 (n 2^-24) and the result's rounding:  u |o| + sum_j (p (u + 2 e + 2^-19 + n 2^-24) + 2^-25 [fp16]) |v|.
  ds = p (do.v - D): relative 2 e + 2^-19 of itself, p times the errors of do.v ((width + 8) 2^-24 |do|.|v|) and of D (|do| times o's error), its
  own rounding u |ds| (+ 2^-25 in fp16); dq, dk, dv: those errors times |k|, |q|, |do|, summed, plus n 2^-24 of the terms, plus u of the result.
  A result in fp16 below 2^-14 is a multiple of 2^-24: its rounding is 2^-25 then, not u of it (dv = -1.1177008771e-05 of one case is
  2.87e-08 from the nearest fp16 number, by the format alone).
  Rows of at most 128 keys, keys of at most 128 queries (two=True): p and ds of the backward products in two parts, u^2 in place of u (what the first
  part leaves is exact in 32 bits), twice the terms to sum, and D as the sum of p (do.v), each with its own errors above and n 2^-24.
  dtable: the 32-bit ds, D from an output whose p had an error of u^2 instead of u; a sum of all pairs of a bucket, m 2^-24 at most for the
  m terms of one row of tiles (64 of them per step, then steps, waves and slots in turn: 2^-24 (64 + 512) used)."""
import ctypes
import math

import pytest
import torch

from dm_amd.neural_nets import sequence
from dm_amd.runtime import hip, ops

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(lens_q, lens_k, heads, kv, width, dtype, seed=0, tail=0, lead=0, table=None):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    tq, tk = lead + sum(lens_q) + tail, lead + sum(lens_k) + tail
    d = dict(q=n(tq, heads, width), k=n(tk, kv, width), v=n(tk, kv, width), do=n(tq, heads, width))
    d["eq"] = torch.tensor([lead] + [lead + sum(lens_q[:i + 1]) for i in range(len(lens_q))], dtype=torch.int32)
    d["ek"] = torch.tensor([lead] + [lead + sum(lens_k[:i + 1]) for i in range(len(lens_k))], dtype=torch.int32)
    if table is not None:
        buckets, far, both = table
        d["buckets"] = sequence.relative_position_buckets(buckets, far, both)
        d["table"] = torch.randn(buckets, heads, generator=g)
    return d


def reference(d, causal, scale=None, two=False):
    """results and tolerances in float64, sequence by sequence"""
    dtype, heads, kv, width = d["q"].dtype, d["q"].shape[1], d["k"].shape[1], d["q"].shape[2]
    u, floor = HALF_STEP[dtype], (2.0 ** -25 if dtype == torch.float16 else 0.0)
    scale = width ** -0.5 if scale is None else scale
    out = {n: torch.zeros(d[s].shape, dtype=torch.float64) for n, s in (("o", "q"), ("dq", "q"), ("dk", "k"), ("dv", "v"))}
    tol = {n: torch.zeros_like(t) for n, t in out.items()}
    if "table" in d:
        out["dtable"] = torch.zeros(d["table"].shape, dtype=torch.float64)
        tol["dtable"] = torch.zeros_like(out["dtable"])
    q, k, v, do = (d[n].double().permute(1, 0, 2) for n in ("q", "k", "v", "do"))
    k, v = k.repeat_interleave(heads // kv, 0), v.repeat_interleave(heads // kv, 0)
    share = lambda x: x.view(kv, heads // kv, *x.shape[1:]).sum(1).permute(1, 0, 2)  # noqa: E731
    for b in range(len(d["eq"]) - 1):
        rq, rk = slice(int(d["eq"][b]), int(d["eq"][b + 1])), slice(int(d["ek"][b]), int(d["ek"][b + 1]))
        nq, nk = rq.stop - rq.start, rk.stop - rk.start
        if nq == 0 or nk == 0:
            continue
        Q, K, V, dO = q[:, rq], k[:, rk], v[:, rk], do[:, rq]
        off = nk - nq if causal else 0
        dist = torch.arange(nk)[None, :] - (torch.arange(nq)[:, None] + off)
        s = scale * Q @ K.transpose(1, 2)
        e = (width + 8) * 2.0 ** -24 * scale * Q.abs() @ K.abs().transpose(1, 2)
        if "table" in d:
            far = len(d["buckets"]) // 2
            which = d["buckets"].long()[dist.clamp(-far, far) + far]
            s = s + d["table"].double()[which].permute(2, 0, 1)
        e = e + 2.0 ** -22 * s.abs()
        seen = dist <= 0 if causal else torch.ones(nq, nk, dtype=torch.bool)
        s = s.masked_fill(~seen, -math.inf)
        p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0) * seen                       # (a row that sees nothing: zeros)
        ep = 2 * (e * seen).amax(-1, keepdim=True) + 2.0 ** -19
        o = p @ V
        base = ep + nk * 2.0 ** -24
        terms = p @ V.abs()
        miss = floor * seen.double() @ V.abs()
        to = (u + base) * terms + miss
        dp = dO @ V.transpose(1, 2)
        D = (dO * o).sum(-1, keepdim=True)
        ds = p * (dp - D)
        err_dp = (width + 8) * 2.0 ** -24 * dO.abs() @ V.abs().transpose(1, 2)
        err_d = lambda t: (dO.abs() * t).sum(-1, keepdim=True)  # noqa: E731
        eds32 = ds.abs() * ep + p * (err_dp + err_d((u * u + base) * terms + miss * u + 2.0 ** -23 * o.abs()))
        eds = ds.abs() * (ep + u) + p * (err_dp + err_d(to + u * o.abs())) + floor * seen
        ep16 = p * (u + ep) + floor * seen
        if two:
            e_d = (p * (dp.abs() * (ep + nk * 2.0 ** -24) + err_dp)).sum(-1, keepdim=True)
            eds = ds.abs() * (ep + u * u + (nk + nq * heads // kv) * 2.0 ** -24) + p * (err_dp + e_d) + floor * seen
            ep16 = p * (u * u + ep + nq * heads // kv * 2.0 ** -24) + floor * seen
        add = lambda name, rows, x, t: (out[name][rows].add_(x), tol[name][rows].add_(t))  # noqa: E731
        add("o", rq, o.permute(1, 0, 2), (to + u * o.abs() + floor).permute(1, 0, 2))
        add("dq", rq, (scale * ds @ K).permute(1, 0, 2), (scale * ((eds + nk * 2.0 ** -24 * ds.abs()) @ K.abs()) + u * (scale * ds @ K).abs() + floor).permute(1, 0, 2))
        total = nq * heads // kv * 2.0 ** -24
        dk, dv = share(scale * ds.transpose(1, 2) @ Q), share(p.transpose(1, 2) @ dO)
        add("dk", rk, dk, scale * share((eds + total * ds.abs()).transpose(1, 2) @ Q.abs()) + u * dk.abs() + floor)
        add("dv", rk, dv, share((ep16 + total * p).transpose(1, 2) @ dO.abs()) + u * dv.abs() + floor)
        if "table" in d:
            for x, dst in ((ds, out["dtable"]), (eds32 + 576 * 2.0 ** -24 * ds.abs(), tol["dtable"])):
                dst.index_add_(0, which.reshape(-1), (x * seen).permute(1, 2, 0).reshape(-1, heads))
    return out, tol


def check(name, got, want, tol):
    got = got.detach().cpu().double()
    bad = ~((got - want).abs() <= tol * 1.0001 + 1e-30)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {((got - want).abs() / (tol + 1e-30)).max():.3g} of the tolerance"


def run(d, dev, causal, cross=True, scale=None):
    x = {n: d[n].to(dev).requires_grad_() for n in ("q", "k", "v")}
    table = d["table"].to(dev).requires_grad_() if "table" in d else None
    o = sequence.packed_attention(x["q"], x["k"], x["v"], d["eq"].to(dev), ends_k=d["ek"].to(dev) if cross else None, causal=causal, scale=scale, bias_table=table,
                                  bias_buckets=d["buckets"].to(dev) if table is not None else None)
    grads = torch.autograd.grad(o, [x["q"], x["k"], x["v"]] + ([table] if table is not None else []), d["do"].to(dev))
    return dict(zip(["o", "dq", "dk", "dv", "dtable"], [o.detach()] + list(grads)))


def compare(d, dev, causal, **kw):
    got = run(d, dev, causal, **kw)
    want, tol = reference(d, causal, kw.get("scale"))
    for n in want:
        check(n, got[n], want[n], tol[n])
    return got


# lengths from zero and one to several tiles, around the tile sizes
LENS = {"one": [1], "short": [3, 1, 0, 17, 2], "tiles": [64, 32, 128, 31, 33, 63, 65, 127, 129], "long": [700, 1, 333], "empty": [0, 0]}


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", sorted(LENS))
@pytest.mark.parametrize("heads,kv,width", [(2, 2, 64), (4, 1, 128), (6, 2, 32), (2, 1, 8), (3, 3, 40), (2, 2, 96)])
def test_against_float64(dev, dtype, causal, lens, heads, kv, width):
    d = make(LENS[lens], LENS[lens], heads, kv, width, dtype, seed=width, tail=5)
    compare(d, dev, causal, cross=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv,width", [(2, 2, 64), (4, 1, 128), (2, 1, 8), (3, 3, 40)])
def test_gradients_of_short_sequences_have_one_rounding(dev, dtype, causal, heads, kv, width):
    d = make([2, 1, 5, 17, 64, 100, 128, 3], [2, 1, 5, 17, 64, 100, 128, 3], heads, kv, width, dtype, seed=19)
    got = run(d, dev, causal)
    want, tol = reference(d, causal, two=True)
    for n in ("dq", "dk", "dv"):
        check(n, got[n], want[n], tol[n])


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lens", ["one", "short", "tiles", "long"])
@pytest.mark.parametrize("heads,kv,width,table", [(2, 2, 64, (32, 128, True)), (4, 2, 128, (16, 40, False)), (2, 1, 32, (8, 5, True)), (2, 2, 40, (32, 1024, True))])
def test_bias_against_float64(dev, causal, lens, heads, kv, width, table):
    d = make(LENS[lens], LENS[lens], heads, kv, width, torch.bfloat16, seed=width, tail=3, table=table)
    compare(d, dev, causal, cross=False)


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("table", [None, (32, 64, True)])
def test_queries_and_keys_of_different_lengths(dev, causal, table):
    """one query on many keys, more queries than keys (causal: the first see nothing), sequences without keys or without queries"""
    lq, lk = [1, 70, 200, 5, 0, 130], [300, 20, 65, 0, 9, 131]
    d = make(lq, lk, 4, 2, 64, torch.float16, seed=5, tail=4, lead=3, table=table)
    got = compare(d, dev, causal)
    for n in ("o", "dq"):
        assert (got[n][:3] == 0).all() and (got[n][-4:] == 0).all() and (got[n][3 + 271:3 + 276] == 0).all()
    if causal:
        assert (got["o"][3 + 1:3 + 51] == 0).all() and (got["o"][3 + 71:3 + 71 + 135] == 0).all()


@pytest.mark.gpu
def test_large_scores_and_bias(dev):
    """a softmax that is nearly one-hot, scores far from zero, a row whose maximum grows late, a bias of -inf (a bucket that is masked)"""
    d = make([200], [200], 2, 2, 64, torch.bfloat16, seed=8, table=(8, 16, True))
    d["q"] = (d["q"].float() * 4).to(torch.bfloat16)
    d["k"][150] = d["k"][150] * 8
    compare(d, dev, True, cross=False)
    d["table"][3] = -200.0
    compare(d, dev, False, cross=False)
    d["table"][3] = -math.inf
    want, _ = reference(dict(d, table=torch.where(d["table"].isinf(), -1e9, d["table"])), False)
    got = run(d, dev, False, cross=False)
    assert all(torch.isfinite(t).all() for t in got.values())
    assert (got["dtable"][3] == 0).all() and (got["o"].cpu().double() - want["o"]).norm() < 2.0 ** -7 * want["o"].norm()


@pytest.mark.gpu
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("heads,kv,width,table", [(2, 1, 64, (8, 16, True)), (2, 2, 128, (32, 1024, True))])
def test_a_bias_of_the_lowest_value(dev, causal, heads, kv, width, table):
    """float32's lowest value, -1e9 and 1e6 as biases, for one bucket and for all of them (the rows' keys are then masked alike and keep their
    scores): as biases of +-8192 / log2(e), which is where the kernels limit them"""
    limit = 8192 * math.log(2.0)
    for low in (torch.finfo(torch.float32).min, -1e9):
        for rows in (slice(0, 1), slice(2, 5), slice(None)):
            d = make([200, 1, 70], [200, 1, 70], heads, kv, width, torch.bfloat16, seed=18, table=table)
            d["table"][rows] = low
            got = run(d, dev, causal, cross=False)
            d["table"].clamp_(-limit, limit)
            want, tol = reference(d, causal)
            for n in want:
                check(n, got[n], want[n], tol[n])
    d["table"][:] = 1e6
    got = run(d, dev, causal, cross=False)
    d["table"][:] = limit
    want, tol = reference(d, causal)
    for n in want:
        check(n, got[n], want[n], tol[n])


@pytest.mark.gpu
def test_infinities_and_nan_outside_stay_there(dev):
    """NaN in rows of no sequence and in another sequence; -inf and inf where the mask hides them"""
    d = make([40, 90], [40, 90], 2, 1, 64, torch.bfloat16, seed=9, tail=6)
    clean = run(d, dev, False, cross=False)
    for n in ("q", "k", "v", "do"):
        d[n][-6:] = math.nan
    got = run(d, dev, False, cross=False)
    for n in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[n], clean[n]), n
        assert (got[n][-6:] == 0).all()
    for n in ("q", "k", "v", "do"):
        d[n][40:130] = math.nan
    got = run(d, dev, False, cross=False)
    for n in ("o", "dq", "dk", "dv"):
        assert torch.equal(got[n][:40], clean[n][:40]), n


@pytest.mark.gpu
@pytest.mark.parametrize("width", [8, 32, 64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_a_tile_ends_where_its_sequence_does(dev, width, causal):
    """NaN in every row behind a sequence that ends inside a tile, at every load of the tile: nothing of it arrives, not even times zero"""
    for n in (1, 3, 5, 9, 17, 31, 33, 50, 63, 65, 100):
        d = make([n, 140], [n, 140], 4, 2, width, torch.bfloat16, seed=n)
        clean = run(d, dev, causal, cross=False)
        for name in ("q", "k", "v", "do"):
            d[name][n:] = math.nan
        got = run(d, dev, causal, cross=False)
        for name in ("o", "dq", "dk", "dv"):
            assert torch.equal(got[name][:n], clean[name][:n]), (n, name)


@pytest.mark.gpu
def test_strides_and_views(dev):
    """q, k, v as views of one packed projection; other layouts; results and gradients into views, rows outside left as they were"""
    d = make([50, 77], [50, 77], 4, 2, 64, torch.bfloat16, seed=10, tail=9)
    want = run(d, dev, True, cross=False)
    packed = torch.cat([d["q"], d["k"], d["v"]], 1).to(dev).requires_grad_()
    q, k, v = packed.split([4, 2, 2], 1)
    o = sequence.packed_attention(q, k, v, d["eq"].to(dev), causal=True)
    assert torch.equal(o, want["o"])
    g, = torch.autograd.grad(o, packed, d["do"].to(dev))
    assert torch.equal(g, torch.cat([want["dq"], want["dk"], want["dv"]], 1))
    heads_first = lambda t: t.to(dev).permute(1, 0, 2).contiguous().permute(1, 0, 2)  # noqa: E731
    strided = lambda t: torch.stack([t, t], 2).flatten(2).to(dev)[:, :, :64]  # noqa: E731
    unaligned = lambda t: torch.cat([t.reshape(-1)[:1], t.reshape(-1)]).to(dev)[1:].view(t.shape)  # noqa: E731
    inner = lambda t: t.to(dev).transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    for f in (heads_first, strided, unaligned, inner):
        assert torch.equal(sequence.packed_attention(f(d["q"]), f(d["k"]), f(d["v"]), d["eq"].to(dev), causal=True), want["o"])
    one = d["k"][:, :1].to(dev)
    assert torch.equal(sequence.packed_attention(d["q"].to(dev), one.expand(-1, 2, -1), one.expand(-1, 2, -1), d["eq"].to(dev)),
                       sequence.packed_attention(d["q"].to(dev), one, one, d["eq"].to(dev)))
    out = torch.full((136, 4, 64), 7.0, device=dev, dtype=torch.bfloat16)
    o, lse, _ = ops.packed_attention_forward(q.detach(), k.detach(), v.detach(), d["eq"].to(dev), causal=True, out=out)
    assert torch.equal(out[:127], want["o"][:127]) and (out[127:] == 7).all()
    store = torch.full((136, 8, 64), 5.0, device=dev, dtype=torch.bfloat16)
    ops.packed_attention_backward(q.detach(), k.detach(), v.detach(), out, lse, d["do"].to(dev), d["eq"].to(dev), causal=True, grads=store.split([4, 2, 2], 1))
    assert torch.equal(store[:127], g[:127]) and (store[127:] == 5).all()


@pytest.mark.gpu
def test_gradients_are_derivatives(dev):
    """central differences of the float64 forward pass along each gradient's own direction.  The slope along g / |g| is |g|; the kernel's
    gradient is off by at most its tolerance, and the differences by h^2: the bound is the tolerance's norm plus 1e-4 |g|."""
    d = make([9, 20], [9, 20], 2, 1, 32, torch.float16, seed=11, table=(8, 6, True))
    got = run(d, dev, True, cross=False)
    _, tol = reference(d, True)
    f = lambda e: (reference(e, True)[0]["o"] * d["do"].double()).sum()  # noqa: E731
    for name, key in (("q", "dq"), ("k", "dk"), ("v", "dv"), ("table", "dtable")):
        g = got[key].cpu().double()
        h = 1e-3
        up, down = (f(dict(d, **{name: Exact(d[name].double() + s * h * g / g.norm(), d[name].dtype)})) for s in (1, -1))
        assert abs((up - down) / (2 * h) - g.norm()) <= tol[key].norm() + 1e-4 * g.norm(), name


def Exact(t, dtype):
    """float64 values for reference(), which asks an input only for its shape, its type and .double()"""
    class Wrapped:
        shape, double = t.shape, lambda self: t
    w = Wrapped()
    w.dtype = dtype
    return w


@pytest.mark.gpu
def test_same_bits_every_time_and_one_head_at_a_time(dev):
    d = make([300, 41, 129], [300, 41, 129], 4, 2, 64, torch.bfloat16, seed=12, table=(32, 64, True))
    a, b = run(d, dev, True, cross=False), run(d, dev, True, cross=False)
    for n in a:
        assert torch.equal(a[n], b[n]), n


@pytest.mark.gpu
def test_boundaries_that_are_wrong_stay_inside(dev):
    """boundaries out of order or out of range are clamped on the device: no access outside of the tensors, and whole sequences in front of
    them come out right"""
    d = make([30, 40], [30, 40], 2, 2, 64, torch.bfloat16, seed=13)
    want = run(d, dev, False, cross=False)
    bad = dict(d, eq=torch.tensor([0, 30, 1000], dtype=torch.int32))
    assert torch.equal(run(bad, dev, False, cross=False)["o"], want["o"])
    for ends in ([0, 50, 20, 70], [-5, 30, 70], [0, 70, -1], [2 ** 31 - 1, 0, 30]):
        got = run(dict(d, eq=torch.tensor(ends, dtype=torch.int32)), dev, True, cross=False)
        torch.cuda.synchronize()
        assert got["o"].shape == want["o"].shape


@pytest.mark.gpu
def test_captured_and_on_another_stream(dev):
    d = make([33, 100], [33, 100], 2, 2, 64, torch.bfloat16, seed=14, table=(16, 32, True))
    x = {n: d[n].to(dev) for n in ("q", "k", "v", "do", "table")}
    ends, buckets = d["eq"].to(dev), d["buckets"].to(dev)

    def body():
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v", "table")]
        o = sequence.packed_attention(*leaves[:3], ends, causal=True, bias_table=leaves[3], bias_buckets=buckets)
        return [o.detach()] + list(torch.autograd.grad(o, leaves, x["do"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = body()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(other, body()))
    graphs = []
    for _ in range(2):                                           # two graphs: workspaces of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = body()
        graphs.append((g, out))
    for k in range(4):
        for n in ("q", "k", "v", "do", "table"):
            x[n].normal_()
        ends.copy_(torch.tensor([0, 20 + k, 133 - k], dtype=torch.int32))         # other lengths, the same launch
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        want = body()
        for _, out in graphs:
            assert all(torch.equal(a, b) for a, b in zip(out, want)), k


@pytest.mark.gpu
def test_capture_beside_a_living_graph_is_refused(dev):
    d = make([9, 20], [9, 20], 2, 1, 32, torch.bfloat16, seed=20, table=(8, 6, True))
    q, k, v, ends, do = (d[n].to(dev) for n in ("q", "k", "v", "eq", "do"))
    table, how = d["table"].to(dev).requires_grad_(), dict(bias_buckets=d["buckets"].to(dev))
    old = sequence.packed_attention(q, k, v, ends, bias_table=table, **how)
    with pytest.raises(RuntimeError, match="packed_attention.*is alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            torch.autograd.grad(sequence.packed_attention(q, k, v, ends, bias_table=table, **how), table, do)
    torch.cuda.synchronize()
    want, = torch.autograd.grad(old, table, do)
    del old
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got, = torch.autograd.grad(sequence.packed_attention(q, k, v, ends, bias_table=table, **how), table, do)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)


@pytest.mark.gpu
def test_many_sequences(dev):
    """more sequences than a wave has lanes, most of them shorter than a tile"""
    g = torch.Generator().manual_seed(15)
    lens = torch.randint(0, 20, (300,), generator=g).tolist() + [200]
    compare(make(lens, lens, 2, 1, 32, torch.bfloat16, seed=15), dev, True, cross=False)


@pytest.mark.gpu
def test_an_encoder_layer(dev):
    """layer norm, packed attention with bias, and the clipped optimizer step as a conditioning encoder uses them: two steps, gradients of all
    parameters against the same layer in plain float32 operations.  Bound: the layer's activations are bf16 (half a step 2^-8 each; at most ten
    roundings lie between a parameter and the loss, and they add up as independent errors do): 2^-8 * sqrt(10) * 4 of a gradient's norm."""
    from dm_amd.optimizer import FusedAdam
    torch.manual_seed(3)
    c, heads, lens = 128, 4, [40, 7, 81]
    ends = torch.tensor([0, 40, 47, 128], dtype=torch.int32, device=dev)
    norm, bias = sequence.LayerNorm(c, device=dev), sequence.RelativePositionBias(16, heads, 20, device=dev)
    with torch.no_grad():
        bias.weight.normal_()
        norm.weight.normal_(1, 0.2)
    w_qkv, w_o = ((torch.randn(n, c, device=dev) / c ** 0.5).requires_grad_() for n in (3 * c, c))
    params = [norm.weight, norm.bias, bias.weight, w_qkv, w_o]
    x, target = torch.randn(128, c, device=dev), torch.randn(128, c, device=dev)

    def layer(plain):
        if plain:
            y = torch.nn.functional.layer_norm(x, (c,), norm.weight, norm.bias)
            q, k, v = (y @ w_qkv.t()).view(128, 3, heads, 32).unbind(1)
            parts, at = [], 0
            for n in lens:
                dist = torch.arange(n, device=dev)[None, :] - torch.arange(n, device=dev)[:, None]
                far = len(bias.buckets) // 2
                b = bias.weight[bias.buckets.long()[dist.clamp(-far, far) + far]].permute(2, 0, 1)
                s = torch.stack([q[at:at + n, i] @ k[at:at + n, i].t() for i in range(heads)]) * 32 ** -0.5 + b
                p = torch.softmax(s, -1)
                parts.append(torch.stack([p[i] @ v[at:at + n, i] for i in range(heads)], 1))
                at += n
            return x + torch.cat(parts).reshape(128, c) @ w_o.t()
        y = norm(x.bfloat16())
        q, k, v = (y @ w_qkv.bfloat16().t()).view(128, 3 * heads, 32).split([heads, heads, heads], 1)
        o = sequence.packed_attention(q, k, v, ends, **bias())
        return x + (o.reshape(128, c) @ w_o.bfloat16().t()).float()

    opt = FusedAdam(params, lr=1e-3, max_grad_norm=0.1)
    for _ in range(2):
        want = torch.autograd.grad((layer(True) - target).square().mean(), params)
        opt.zero_grad()
        (layer(False) - target).square().mean().backward()
        for p, g in zip(params, want):
            assert (p.grad - g).norm() <= 2.0 ** -8 * 10 ** 0.5 * 4 * g.norm()
        opt.step()
        total = torch.cat([p.grad.double().reshape(-1) for p in params]).norm()
        assert abs(opt.grad_norm.item() - total.item()) <= 2.0 ** -23 * total.item()


def test_buckets():
    far = lambda t: len(t) // 2  # noqa: E731
    both = sequence.relative_position_buckets(32, 128)
    f = far(both)
    assert both[f].item() == 0 and [both[f - n].item() for n in range(1, 8)] == list(range(1, 8)) and [both[f + n].item() for n in range(1, 8)] == list(range(17, 24))
    # borders that are whole numbers: 8 * 16^(t / 8) at t = 2, 4, 6 is 11.3.., 32, 64 -> 16 (t = 2: 8 * 2), 32 (t = 4), 64 (t = 6)
    assert [both[f - n].item() for n in (15, 16, 31, 32, 63, 64, 90, 91)] == [9, 10, 11, 12, 13, 14, 14, 15] and f == 91
    one = sequence.relative_position_buckets(32, 128, bidirectional=False)
    f = far(one)
    assert (one[f:] == 0).all() and one[f - 15].item() == 15 and one[0].item() == 31
    for bad in ((3, 128, True), (2, 128, True), (1, 16, False), (32, 8, True), (32, 1025, True)):
        with pytest.raises(ValueError):
            sequence.relative_position_buckets(*bad)


def test_refusals_without_a_gpu():
    h = torch.bfloat16
    q, k, e = torch.zeros(4, 4, 64, dtype=h), torch.zeros(4, 2, 64, dtype=h), torch.tensor([0, 4], dtype=torch.int32)
    table, buckets = torch.zeros(8, 4), torch.zeros(17, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="HIP kernels only"):
        sequence.packed_attention(q, k, k, e)
    with pytest.raises(ValueError, match="not \\[tokens, heads, width\\]"):
        sequence.packed_attention(q.view(4, -1), k, k, e)
    f = ops.packed_attention_forward
    for args, kw, why in (((q, k[:, :, :32], k[:, :, :32], e), {}, "whole groups"), ((q, k, k[:3], e), {}, "whole groups"), ((q, k.repeat(1, 2, 1)[:, :3], k.repeat(1, 2, 1)[:, :3], e), {}, "whole groups"),
                          ((q.float(), k.float(), k.float(), e), {}, "types"), ((q, k.half(), k, e), {}, "types"), ((q, k, k, e.long()), {}, "int32"),
                          ((q, k, k, e.view(1, 2)), {}, "int32"), ((q, k, k, e, torch.zeros(3, dtype=torch.int32)), {}, "int32"), ((q, k, k, e), dict(table=table), "both"),
                          ((q, k, k, e), dict(table=table.double(), bucket_of=buckets), "bias table"), ((q, k, k, e), dict(table=table[:, :3], bucket_of=buckets), "bias table"),
                          ((q, k, k, e), dict(table=table, bucket_of=buckets[:16]), "2 far"), ((q, k, k, e), dict(table=table, bucket_of=buckets.long()), "2 far")):
        with pytest.raises(ValueError, match=why):
            f(*args, **kw)
    at = q.data_ptr() // 16 * 16
    good = dict({f"{n}": at for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv", "ends_q", "ends_k", "lse", "dsum")}, Tq=4, Tk=4, B=1, H=4, Hk=2, dh=64, dtype=0, scale=0.1,
                **{f"{n}_row": 256 for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv")}, **{f"{n}_head": 64 for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv")})
    last = lambda: hip.lib().ddpm_last_error()  # noqa: E731
    for bad, why in ((dict(dh=60), b"head width"), (dict(dh=136), b"head width"), (dict(dh=0), b"head width"), (dict(dtype=2), b"element type"), (dict(Hk=3), b"heads"), (dict(Hk=0), b"heads"),
                     (dict(Tq=-1), b"queries"), (dict(B=-1), b"sequences"), (dict(scale=0.0), b"scale"), (dict(scale=math.nan), b"scale"), (dict(scale=math.inf), b"scale"),
                     (dict(ends_q=None), b"boundaries"), (dict(q=None), b"q is null"), (dict(v=at + 2), b"16-byte"), (dict(k_row=252), b"strides of k"), (dict(o_head=0), b"strides of o"),
                     (dict(q_row=1 << 24), b"2^24"), (dict(k_head=32), b"shorter"), (dict(table=at), b"both"), (dict(table=at, bucket_of=at, far=3, buckets=8), b"distances"),
                     (dict(table=at, bucket_of=at, far=1025, buckets=8), b"distances"), (dict(table=at, bucket_of=at, far=8, buckets=0), b"buckets"),
                     (dict(B=(1 << 24) - 1, H=1024), b"workgroups"), (dict(B=1 << 22), b"workgroups")):
        assert hip.lib().ddpm_packed_attention_forward(ctypes.byref(hip.PackedAttnDesc(**dict(good, **bad))), None) != 0 and why in last(), (bad, last())
    for bad, why in ((dict(lse=None), b"lse"), (dict(dsum=None), b"dsum"), (dict(dtable=at), b"not there"), (dict(table=at, bucket_of=at, far=8, buckets=8, dtable=at), b"dtable_part"),
                     (dict(dq=at + 8), b"dq"), (dict(dout_row=100), b"dout")):
        assert hip.lib().ddpm_packed_attention_backward(ctypes.byref(hip.PackedAttnDesc(**dict(good, **bad))), None) != 0 and why in last(), (bad, last())
    assert hip.lib().ddpm_packed_attention_forward(None, None) != 0
