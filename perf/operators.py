"""Operators of the conditioning sequence and of the training step, as they are measured: layer norm, attention over packed
sequences, the learned relative position bias inside that attention, and the global gradient norm with clipping.

Every operator has a plain form here (elementary torch operations in 32 bits) and the calls a program makes of this package."""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-5


# ---- cases --------------------------------------------------------------------------------------------------------------------
def listed():
    ln = dict(op="layer_norm", bias=True, pad=0)
    at = dict(op="attention", causal=True, tail=0, packed=False)
    bi = dict(op="bias_attention", causal=False, tail=0, packed=False, buckets=32, max_distance=128)
    cl = dict(op="clip", norm="2", seed_sizes=1)
    return [
        # one prompt's tokens through one norm while sampling: launch latency
        dict(ln, name="layer_norm_prompt", rows=64, cols=512, dtype="bf16", train=False),
        # the widest rows a conditioning encoder of this package's kind carries, many prompts at once
        dict(ln, name="layer_norm_wide", rows=65536, cols=4096, dtype="bf16", train=False),
        # a training step's norm over the tokens of 64 images of 16x16 positions, forward and backward
        dict(ln, name="layer_norm_train", rows=16384, cols=1024, dtype="bf16", train=True),
        # odd width, padded rows, 32-bit activations, no bias
        dict(ln, name="layer_norm_odd_train", rows=5003, cols=1001, dtype="fp32", train=True, bias=False, pad=7),
        # eight short prompts with a causal encoder while sampling: launch latency
        dict(at, name="attention_prompts", lens="77 12 1 64 33 9 77 50", heads=8, kv_heads=8, dim=64, dtype="bf16", train=False, tail=13, packed=True),
        # two long documents with grouped heads: the largest case
        dict(at, name="attention_long", lens="8192 7937", heads=32, kv_heads=8, dim=128, dtype="bf16", train=False),
        # a training batch of ragged sequences with grouped heads, forward and backward
        dict(at, name="attention_train", lens="2048 1999 1501 1024 2047 777 130 1", heads=16, kv_heads=4, dim=128, dtype="bf16", train=True),
        # sixteen prompts through a bidirectional encoder with position bias while sampling
        dict(bi, name="bias_prompts", lens="77 256 31 128 200 8 255 77 100 17 90 256 64 3 141 222", heads=8, kv_heads=8, dim=64, dtype="bf16", train=False, packed=True),
        # long ragged sequences with position bias, training: the bias's gradient among the outputs
        dict(bi, name="bias_train", lens="2048 1025 1536 63 1999 512", heads=8, kv_heads=8, dim=64, dtype="bf16", train=True),
        # causal, grouped heads, half precision, the one-sided buckets
        dict(bi, name="bias_causal_train", lens="1024 1000 513 300", heads=16, kv_heads=4, dim=64, dtype="fp16", train=True, causal=True),
        # the denoiser's 350 parameter tensors: gradients as its backward pass lays them out
        dict(cl, name="clip_network", align=4, tensors=350, elements=6_857_763, dtype="fp32"),
        # a large model's gradients in two types, allocated apart
        dict(cl, name="clip_large", align=256, tensors=500, elements=400_000_000, dtype="mixed"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["layer_norm", "attention", "bias_attention", "clip"])
    if op == "layer_norm":
        cols = rng.choice([_log_int(rng, 5, 8192), 8 * _log_int(rng, 4, 1024)])
        train = rng.random() < 0.6
        rows = min(_log_int(rng, 1, 65536), (1 << 27) // cols)
        return dict(op=op, rows=rows, cols=cols, dtype=rng.choice(["bf16", "fp16", "fp32"]), train=train, bias=rng.random() < 0.7,
                    pad=rng.choice([0, 0, 8, rng.randrange(1, 20)]))
    if op == "clip":
        n = _log_int(rng, 1, 600)
        return dict(op=op, norm=rng.choice(["2", "2", "inf"]), tensors=n, elements=max(n, _log_int(rng, 100, 200_000_000)),
                    dtype=rng.choice(["fp32", "bf16", "mixed"]), seed_sizes=rng.randrange(1 << 30),
                    align=rng.choice([1, 4, 256]))
    kv = rng.choice([1, 2, 4, 8])
    heads = kv * rng.choice([1, 1, 2, 4])
    dim = rng.choice([8, 32, 40, 64, 64, 96, 128, 128])
    train = rng.random() < 0.6
    n = _log_int(rng, 1, 16)
    longest = _log_int(rng, 2, 4096 if op == "attention" else 2048)
    while n > 1 and n * heads * longest * longest > (1 << 30):
        n -= 1
    lens = [longest] + [rng.choice([rng.randrange(1, longest + 1), _log_int(rng, 1, longest)]) for _ in range(n - 1)]
    rng.shuffle(lens)
    case = dict(op=op, lens=" ".join(map(str, lens)), heads=heads, kv_heads=kv, dim=dim, dtype=rng.choice(["bf16", "bf16", "fp16"]), train=train,
                causal=rng.random() < 0.5, tail=rng.choice([0, 0, rng.randrange(1, 100)]), packed=rng.random() < 0.5)
    if op == "bias_attention":
        case |= dict(buckets=rng.choice([8, 16, 32, 64]), max_distance=rng.choice([64, 100, 128, 256]))
    return case


# ---- inputs -------------------------------------------------------------------------------------------------------------------
def _lens(case):
    return [int(n) for n in case["lens"].split()]


def _bucket_of(case):
    """Bucket of every distance key - query from -max_distance to max_distance.  Half of the buckets (all of them when causal, where
    keys never follow the query) hold single distances, the others ranges whose borders grow geometrically up to max_distance;
    bucket e + t begins at the first n with (n / e)^k >= (max_distance / e)^t, compared in whole numbers."""
    far, half = case["max_distance"], case["buckets"] if case["causal"] else case["buckets"] // 2
    e = half // 2
    k = half - e
    one_side = [n if n < e else e + min(k - 1, sum(n ** k * e ** t >= far ** t * e ** k for t in range(1, k))) for n in range(far + 1)]
    after = [0 if case["causal"] else half + b for b in one_side]
    return one_side[:0:-1] + [one_side[0]] + after[1:]


def _sizes(case):
    """Element counts of the tensors: spread over a factor of thousands, with the total of the case"""
    g = torch.Generator().manual_seed(case["seed_sizes"])
    share = torch.exp(torch.rand(case["tensors"], generator=g, dtype=torch.float64) * 8)
    return [max(1, int(s)) for s in share / share.sum() * case["elements"]]


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(dev).manual_seed(seed)
    rand = lambda *shape: torch.randn(*shape, generator=g, device=dev)  # noqa: E731
    state = {"case": case}
    if case["op"] == "layer_norm":
        t, rows, cols = DTYPES[case["dtype"]], case["rows"], case["cols"]
        store = torch.zeros(rows, cols + case["pad"], device=dev, dtype=t)
        x = store[:, :cols]
        x.copy_(rand(rows, cols) * (rand(rows, 1).abs() + 0.1) + rand(rows, 1))
        state |= dict(x=x.requires_grad_(case["train"]), weight=(1 + 0.2 * rand(cols)).requires_grad_(case["train"]),
                      bias=(0.2 * rand(cols)).requires_grad_(case["train"]) if case["bias"] else None, dy=rand(rows, cols).to(t) if case["train"] else None)
    elif case["op"] == "clip":
        kinds = {"fp32": [torch.float32], "bf16": [torch.bfloat16], "mixed": [torch.float32, torch.bfloat16, torch.bfloat16]}[case["dtype"]]
        sizes, ends = _sizes(case), {t: 0 for t in kinds}
        state["params"] = []
        for i, n in enumerate(sizes):                          # one buffer of gradients for each type, every gradient a view of it
            ends[kinds[i % len(kinds)]] += -(-n // case["align"]) * case["align"]
        state["buffers"] = {t: torch.zeros(n, device=dev, dtype=t) for t, n in ends.items()}
        ends = {t: 0 for t in kinds}
        for i, n in enumerate(sizes):
            t = kinds[i % len(kinds)]
            p = torch.empty(n, device=dev, dtype=t)
            p.grad = state["buffers"][t][ends[t]:ends[t] + n].copy_(rand(n) * 10.0 ** (i % 5 - 3))
            ends[t] += -(-n // case["align"]) * case["align"]
            state["params"].append(p)
    else:
        t, h, hk, d, lens = DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"], _lens(case)
        total = sum(lens) + case["tail"]
        if case["packed"]:                                     # one projection's output, cut into heads
            q, k, v = rand(total, h + 2 * hk, d).to(t).split([h, hk, hk], 1)
        else:
            q, k, v = (rand(total, n, d).to(t) for n in (h, hk, hk))
        ends = torch.tensor([0] + lens).cumsum(0).to(dev, torch.int32)
        state |= {n: x.detach().requires_grad_(case["train"]) for n, x in (("q", q), ("k", k), ("v", v))}
        state |= dict(ends=ends, longest=max(lens), do=rand(total, h, d).to(t) if case["train"] else None, table=None, bucket_of=None)
        if case["op"] == "bias_attention":
            state["table"] = rand(case["buckets"], h).requires_grad_(case["train"])
            state["bucket_of"] = torch.tensor(_bucket_of(case), dtype=torch.int32, device=dev)
    return state


# ---- one pass -----------------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    return {"layer_norm": _layer_norm, "clip": _clip, "attention": _attention, "bias_attention": _attention}[state["case"]["op"]](state)


def _run_own(s):
    import dm_amd_bootstrap  # noqa: F401
    case = s["case"]
    if case["op"] == "clip":
        from dm_amd.optimizer import clip_grad_norm_
        norm = clip_grad_norm_(s["params"], 1.0, norm_type=float(case["norm"]))
        return {"norm": norm, "buffers": list(s["buffers"].values())}
    from dm_amd.neural_nets import sequence
    if case["op"] == "layer_norm":
        y = sequence.layer_norm(s["x"], s["weight"], s["bias"], EPS)
        leaves, dy = [s["x"], s["weight"]] + ([s["bias"]] if s["bias"] is not None else []), s["dy"]
    else:
        y = sequence.packed_attention(s["q"], s["k"], s["v"], s["ends"], causal=case["causal"], bias_table=s["table"], bias_buckets=s["bucket_of"])
        leaves, dy = [s["q"], s["k"], s["v"]] + ([s["table"]] if s["table"] is not None else []), s["do"]
    if not case["train"]:
        return {"y": y}
    return {"y": y.detach(), "grads": list(torch.autograd.grad(y, leaves, dy))}


@torch.no_grad()
def _layer_norm(s):
    x, w = s["x"].float(), s["weight"]
    c = x - x.mean(-1, keepdim=True)
    rstd = (c.square().mean(-1, keepdim=True) + EPS).rsqrt()
    xhat = c * rstd
    y = xhat * w if s["bias"] is None else xhat * w + s["bias"]
    y = y.to(s["x"].dtype)
    if not s["case"]["train"]:
        return {"y": y}
    dy = s["dy"].float()
    g = dy * w
    dx = rstd * (g - g.mean(-1, keepdim=True) - xhat * (g * xhat).mean(-1, keepdim=True))
    grads = [dx.to(s["x"].dtype), (dy * xhat).sum(0)]
    return {"y": y, "grads": grads if s["bias"] is None else grads + [dy.sum(0)]}


@torch.no_grad()
def _clip(s):
    grads = [p.grad for p in s["params"]]
    flat = torch.cat([g.reshape(-1).float() for g in grads])
    norm = (flat.abs().amax() if s["case"]["norm"] == "inf" else flat.double().square().sum().sqrt()).float()
    torch._foreach_mul_(grads, (1.0 / (norm + 1e-6)).clamp(max=1.0))
    return {"norm": norm, "buffers": list(s["buffers"].values())}


@torch.no_grad()
def _attention(s):
    """On a padded batch: [sequence, head, query, key] in 32 bits, key rows past a sequence's end masked"""
    case, q, ends, n = s["case"], s["q"], s["ends"].long(), s["longest"]
    (total, h, d), b, group = q.shape, len(ends) - 1, case["heads"] // case["kv_heads"]
    at, tok = torch.arange(n, device=q.device), torch.arange(total, device=q.device)
    inside = at < (ends[1:] - ends[:-1])[:, None]
    row = (ends[:-1, None] + at).clamp(max=total - 1)                     # token of each place of the padded batch
    seq = torch.searchsorted(ends[1:], tok, right=True).clamp(max=b - 1)
    place = (seq * n + tok - ends[seq]).clamp(max=b * n - 1)              # and back
    real = (tok < ends[-1])[:, None, None]
    spread = lambda x: (x.float()[row] * inside[..., None, None]).transpose(1, 2)  # noqa: E731
    back = lambda x: x.transpose(1, 2).reshape(b * n, -1, d)[place] * real  # noqa: E731
    qp, kp, vp = spread(q), spread(s["k"]).repeat_interleave(group, 1), spread(s["v"]).repeat_interleave(group, 1)
    scale = 1 / math.sqrt(d)
    p = qp @ kp.transpose(-1, -2) * scale
    far = case.get("max_distance", 0)
    if s["table"] is not None:
        bucket = s["bucket_of"].long()[(at[None, :] - at[:, None]).clamp(-far, far) + far]
        p += s["table"][bucket].permute(2, 0, 1)
    seen = inside[:, None, None, :] & (at[None, :] <= at[:, None] if case["causal"] else torch.ones(n, n, dtype=torch.bool, device=q.device))
    p.masked_fill_(~seen, -math.inf)
    p = (p - p.amax(-1, keepdim=True)).exp()
    p = p / p.sum(-1, keepdim=True)
    o = p @ vp
    y = back(o).to(q.dtype)
    if not case["train"]:
        return {"y": y}
    do = spread(s["do"])
    dv = p.transpose(-1, -2) @ do
    ds = p * (do @ vp.transpose(-1, -2) - (do * o).sum(-1, keepdim=True))
    dq, dk = ds @ kp * scale, ds.transpose(-1, -2) @ qp * scale
    shared = lambda x: back(x.view(b, -1, group, n, d).sum(2))  # noqa: E731
    grads = [back(dq).to(q.dtype), shared(dk).to(q.dtype), shared(dv).to(q.dtype)]
    if s["table"] is not None:
        # sums along the diagonals key - query: rows in reverse order, each shifted by one more, so that a distance is a column
        e = torch.nn.functional.pad(ds.sum(0).flip(1), (0, n)).reshape(h, -1)[:, :n * (2 * n - 1)].view(h, n, 2 * n - 1).sum(1)
        which = s["bucket_of"].long()[torch.arange(1 - n, n, device=q.device).clamp(-far, far) + far]
        grads.append(torch.zeros_like(s["table"]).index_add_(0, which, e.t().contiguous()))
    return {"y": y, "grads": grads}


# ---- cost and definition ------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "layer_norm":
        n, size = case["rows"] * case["cols"], DTYPES[case["dtype"]].itemsize
        return {"bytes": (4 if case["train"] else 2) * n * size + 16 * case["cols"], "flops": (20 if case["train"] else 8) * n}
    if case["op"] == "clip":
        sizes = _sizes(case)
        wide = {"fp32": sum(sizes), "bf16": 0, "mixed": sum(sizes[::3])}[case["dtype"]]
        return {"bytes": 2 * (4 * wide + 2 * (sum(sizes) - wide)), "flops": 3 * sum(sizes)}
    lens, h, hk, d = _lens(case), case["heads"], case["kv_heads"], case["dim"]
    pairs = sum(n * (n + 1) // 2 if case["causal"] else n * n for n in lens)
    size = 2 * sum(lens) * d                                   # one head of one tensor, 16-bit
    return {"bytes": size * ((4 * h + 4 * hk) if case["train"] else (2 * h + 2 * hk)), "flops": (14 if case["train"] else 4) * pairs * h * d}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layer_norm":
        leaves = [x.detach().double().requires_grad_(case["train"]) for x in (s["x"], s["weight"], s["bias"]) if x is not None]
        x, w = leaves[:2]
        var, mean = torch.var_mean(x, -1, correction=0, keepdim=True)
        y = (x - mean) / torch.sqrt(var + EPS) * w + (leaves[2] if case["bias"] else 0)
        return {"y": y.detach(), "grads": list(torch.autograd.grad(y, leaves, s["dy"].double()))} if case["train"] else {"y": y}
    if case["op"] == "clip":
        grads = [p.grad.double() for p in s["params"]]
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(g, float(case["norm"])) for g in grads]), float(case["norm"]))
        return {"norm": norm, "buffers": [b.double() * min(1.0, 1.0 / (norm.item() + 1e-6)) for b in s["buffers"].values()]}
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    y = torch.zeros(s["q"].shape, device="cuda", dtype=torch.float64)
    names = ["q", "k", "v"] + (["table"] if s["table"] is not None else [])
    grads = {n: torch.zeros(s[n].shape, device="cuda", dtype=torch.float64) for n in names}
    begin = 0
    for n in _lens(case):
        if case["op"] == "bias_attention":
            far = case["max_distance"]
            offset = torch.arange(n, device="cuda").view(1, n) - torch.arange(n, device="cuda").view(n, 1)
            kind = torch.tensor(_bucket_of(case), device="cuda")[offset.clamp(min=-far, max=far) + far]
        for i in range(h):
            part = slice(begin, begin + n)
            j = i // (h // hk)
            a, b, c = (x.detach()[part, m].double().requires_grad_(case["train"]) for x, m in ((s["q"], i), (s["k"], j), (s["v"], j)))
            score = a @ b.T / d ** 0.5
            leaves = [a, b, c]
            if case["op"] == "bias_attention":
                leaves.append(s["table"].detach()[:, i].double().requires_grad_(case["train"]))
                score = score + leaves[3][kind]
            if case["causal"]:
                score = score.masked_fill(torch.ones(n, n, dtype=torch.bool, device="cuda").triu(1), -math.inf)
            o = torch.softmax(score, -1) @ c
            y[part, i] = o.detach()
            if case["train"]:
                found = torch.autograd.grad(o, leaves, s["do"][part, i].double())
                grads["q"][part, i] = found[0]
                grads["k"][part, j] += found[1]
                grads["v"][part, j] += found[2]
                if len(found) > 3:
                    grads["table"][:, i] += found[3]
        begin += n
    return {"y": y, "grads": [grads[n] for n in names]} if case["train"] else {"y": y}
