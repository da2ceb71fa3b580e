"""Gradients of packed attention where a bias of -inf hides all keys of a query: zeros for that query and nothing from it anywhere else.

Tolerances as in test_packed_attention.py (worst cases of every rounding, u = half a step of the type), over the pairs that are seen: neither hidden by
the causal order nor by the bias."""
import math

import pytest
import torch

from dm_amd.neural_nets import sequence

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make(lens, heads, kv, width, dtype, table, hide, seed):
    """inputs of sequences of these lengths; the buckets in `hide` are -inf (of every head, or of (bucket, head) alone)"""
    g = torch.Generator().manual_seed(seed)
    n = lambda *s: torch.randn(*s, generator=g).to(dtype)  # noqa: E731
    total = sum(lens)
    d = dict(q=n(total, heads, width), k=n(total, kv, width), v=n(total, kv, width), do=n(total, heads, width))
    d["ends"] = torch.tensor([0] + lens, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    d["buckets"], d["table"] = sequence.relative_position_buckets(*table), torch.randn(table[0], heads, generator=g)
    for at in hide:
        d["table"][at] = -math.inf
    return d


def reference(d, causal):
    """float64 results, their tolerances, and per query and head whether it sees a key"""
    heads, kv, width = d["q"].shape[1], d["k"].shape[1], d["q"].shape[2]
    u, floor = HALF_STEP[d["q"].dtype], (2.0 ** -25 if d["q"].dtype == torch.float16 else 0.0)
    names = ("o", "dq", "dk", "dv", "dtable")
    out = {n: torch.zeros(d[s].shape, dtype=torch.float64) for n, s in zip(names, ("q", "q", "k", "v", "table"))}
    tol = {n: torch.zeros_like(t) for n, t in out.items()}
    sees, far, scale = torch.zeros(d["q"].shape[:2], dtype=torch.bool), len(d["buckets"]) // 2, width ** -0.5
    for b in range(len(d["ends"]) - 1):
        rows = slice(int(d["ends"][b]), int(d["ends"][b + 1]))
        n = rows.stop - rows.start
        dist = torch.arange(n)[None, :] - torch.arange(n)[:, None]
        which = d["buckets"].long()[dist.clamp(-far, far) + far]
        for h in range(heads):
            Q, K, V, dO = (d[x][rows, h if x in ("q", "do") else h // (heads // kv)].double() for x in ("q", "k", "v", "do"))
            bias = d["table"][:, h].double()[which]
            seen = (bias > -math.inf) & (dist <= 0 if causal else torch.ones(n, n, dtype=torch.bool))
            s = torch.where(seen, scale * Q @ K.t() + bias, -math.inf)
            e = torch.where(seen, (width + 8) * 2.0 ** -24 * scale * Q.abs() @ K.abs().t() + 2.0 ** -22 * s.abs(), 0.0)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            o, ep = p @ V, 2 * e.amax(-1, keepdim=True) + 2.0 ** -19
            dp, D = dO @ V.t(), (dO * o).sum(-1, keepdim=True)
            ds = p * (dp - D)
            base, terms, miss, live = ep + n * 2.0 ** -24, p @ V.abs(), floor * seen.double() @ V.abs(), seen.double()
            err_dp = (width + 8) * 2.0 ** -24 * dO.abs() @ V.abs().t()
            to = (u + base) * terms + miss
            err_d = lambda t: (dO.abs() * t).sum(-1, keepdim=True)  # noqa: E731
            eds32 = ds.abs() * ep + p * (err_dp + err_d((u * u + base) * terms + miss * u + 2.0 ** -23 * o.abs()))
            eds = ds.abs() * (ep + u) + p * (err_dp + err_d(to + u * o.abs())) + floor * live
            sees[rows, h] = seen.any(-1)
            g, many = h // (heads // kv), n * heads // kv * 2.0 ** -24
            for name, at, x, t in (("o", h, o, to), ("dq", h, scale * ds @ K, scale * (eds + n * 2.0 ** -24 * ds.abs()) @ K.abs()),
                                   ("dk", g, scale * ds.t() @ Q, scale * (eds + many * ds.abs()).t() @ Q.abs()),
                                   ("dv", g, p.t() @ dO, (p * (u + ep + many) + floor * live).t() @ dO.abs())):
                out[name][rows, at] += x
                tol[name][rows, at] += t
            for x, dst in ((ds, out["dtable"]), (eds32 + 576 * 2.0 ** -24 * ds.abs(), tol["dtable"])):
                dst[:, h].index_add_(0, which.reshape(-1), x.reshape(-1))
    for name in ("o", "dq", "dk", "dv"):                       # the result's own rounding; what nothing was added to is zero exactly
        tol[name] += (u * out[name].abs() + floor) * (tol[name] > 0)
    return out, tol, sees


def run(d, dev, causal):
    x = {n: d[n].to(dev).requires_grad_() for n in ("q", "k", "v", "table")}
    o = sequence.packed_attention(x["q"], x["k"], x["v"], d["ends"].to(dev), causal=causal, bias_table=x["table"], bias_buckets=d["buckets"].to(dev))
    return dict(zip(("o", "dq", "dk", "dv", "dtable"), [o.detach()] + list(torch.autograd.grad(o, list(x.values()), d["do"].to(dev)))))


# hidden for causal: the own place (the first query of a sequence sees nothing then); not causal: everything that is not beyond the far end, so that
# queries near both ends of a short sequence see nothing; all of it; all of it for one head
NEAR = [slice(0, 7), slice(8, 15)]
CASES = {"own place": (True, [0]), "near": (False, NEAR), "near, causal": (True, NEAR), "all": (False, [slice(None)]), "all, causal": (True, [slice(None)]),
         "one head": (False, [(slice(None), 1)]), "one head, causal": (True, [(slice(None), 1), (0, 0)])}


@pytest.mark.gpu
@pytest.mark.parametrize("case", sorted(CASES))
@pytest.mark.parametrize("lens", [[1, 40, 3, 7, 128, 1], [700, 129, 1, 300]], ids=["short", "long"])
@pytest.mark.parametrize("heads,kv,width,dtype", [(2, 2, 64, torch.bfloat16), (4, 2, 128, torch.bfloat16), (2, 1, 32, torch.float16)])
def test_queries_whose_keys_are_all_hidden(dev, case, lens, heads, kv, width, dtype):
    causal, hide = CASES[case]
    d = make(lens, heads, kv, width, dtype, (16, 40, True), hide, seed=width)
    want, tol, sees = reference(d, causal)
    assert not sees.all()
    got = run(d, dev, causal)
    for n, w in want.items():
        x = got[n].cpu().double()
        assert torch.isfinite(x).all(), n
        bad = ~((x - w).abs() <= tol[n] * 1.0001 + 1e-30)
        assert not bad.any(), f"{n}: {int(bad.sum())} of {bad.numel()} off, worst {((x - w).abs() / (tol[n] + 1e-30)).max():.3g} of the tolerance"
    for n in ("o", "dq"):
        assert (got[n].cpu()[~sees] == 0).all(), n
    assert (got["dtable"].cpu()[d["table"] == -math.inf] == 0).all()
