"""Layers of an encoder of token sequences: layer norm over the channels of each token, and attention over packed sequences of different
lengths (causal or not, grouped heads, learned relative position bias), as autograd functions and modules on the HIP kernels.  Prompts of one
length come out of such an encoder as ConditionalModule's key sequence, x.view(prompts, length, width).  ConditionalModule has no mask: prompts of
different lengths would have to be padded for it, and it would attend to the padding.  Activations are bf16, fp16 or (layer norm) fp32; parameters are fp32, as
everywhere in this package.  The reference has no such encoder; its ConditionalModule takes the sequence from outside
(constituent_blocks.py:402-437 there)."""
from __future__ import annotations

import threading
import weakref
from typing import Optional

import torch
from torch import Tensor, nn
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from ..runtime import hip, ops


def _need_gpu(what: str, *tensors) -> None:
    dev = tensors[0].device
    if dev.type != "cuda":
        raise RuntimeError(f"{what} runs on the HIP kernels only: tensors must live on an MI355X (cuda) device")
    for t in tensors[1:]:
        if t is not None and t.device != dev:
            raise ValueError(f"{what}: tensors on {dev} and {t.device}")


def _no_tangents(what: str, *tensors) -> None:
    """A dual tensor need not ask for a gradient: past the autograd function its tangent would be lost without a word"""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise NotImplementedError(f"{what}: forward-mode derivatives (jvp) are not there")


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _rows(t: Tensor, c: int) -> Tensor:
    """t as [rows, c] with contiguous rows that do not overlap (an expanded or transposed tensor is copied)"""
    r = t.reshape(-1, c)
    if r.stride(1) != 1 or (r.shape[0] > 1 and r.stride(0) < c):
        r = r.contiguous()
    return r if r.stride(1) == 1 else r.as_strided(r.shape, (1, 1))         # (c = 1: torch leaves such a stride as it was)


_graphs: list = []                   # weak references to the nodes of this module's autograd graphs, dead ones swept now and then
_sweep_at = 4096                     # length of that list at which the next sweep is due
_graphs_lock = threading.RLock()     # (held by sweeps and notes: a node noted between a sweep's look and its end would be lost)


def _capturing(t: Tensor) -> bool:
    with hip.on_device_of(t):
        return torch.cuda.is_current_stream_capturing()


def _note_graph(ctx, *inputs) -> None:
    """All graphs of a leaf share the node that receives its gradient, and that node stays with the stream of the graph that made it.  If that is
    the default stream, autograd makes it wait for a captured backward pass, which no capture survives (nor does the process): so
    the backward pass of a captured graph looks for such a graph, and refuses in time."""
    global _sweep_at
    ctx.stream, ctx.stale = hip.stream(inputs[0].get_device()), False        # (of the inputs' device, which need not be the current one)
    if ctx.stream == 0:
        with _graphs_lock:
            _graphs.append(weakref.ref(ctx))
            if len(_graphs) >= _sweep_at:
                _graphs[:] = [r for r in _graphs if r() is not None]
                _sweep_at = max(4096, 2 * len(_graphs))
    elif _capturing(inputs[0]):
        leaves = [t for t in inputs if t is not None and t.requires_grad and t.is_leaf]
        with _graphs_lock:
            noted = list(_graphs)
        held = [getattr(node, "variable", None) for r in noted if (graph := r()) is not None for node, _ in graph.next_functions]
        ctx.stale = any(h is t for h in held if h is not None for t in leaves)


def _refuse_stale(ctx, what: str) -> None:
    if ctx.stale and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what}: this backward pass is being captured while an earlier graph of the same parameters or inputs, made on the default "
                           "stream, is alive; delete its results (or make it on a side stream) before the capture")


class _LayerNormFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: Tensor, weight: Optional[Tensor], bias: Optional[Tensor], eps: float):
        rows = _rows(x, x.shape[-1])
        y, stats = ops.layer_norm_forward(rows, weight, bias, eps, want_stats=any(ctx.needs_input_grad))
        _note_graph(ctx, x, weight, bias)
        ctx.save_for_backward(rows, weight, stats)
        return y.view(x.shape)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy: Tensor):
        _refuse_stale(ctx, "layer_norm")
        rows, weight, stats = ctx.saved_tensors
        nx, nw, nb, _ = ctx.needs_input_grad
        dx, dw, db = ops.layer_norm_backward(rows, _rows(dy, rows.shape[1]), weight, stats, want_dx=nx, want_dw=nw, want_db=nb)
        return dx.view(dy.shape) if nx else None, dw, db, None


def layer_norm(x: Tensor, weight: Optional[Tensor] = None, bias: Optional[Tensor] = None, eps: float = 1e-5) -> Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis (1 to 8192 elements, var over n), statistics in fp32, the
    result in x's type.  weight, bias: fp32 [C] or None.  Differentiable once in x, weight and bias (in reverse mode)."""
    if x.dim() < 1 or x.shape[-1] < 1:
        raise ValueError(f"layer_norm: x of shape {tuple(x.shape)} has no last axis to normalise")
    _no_tangents("layer_norm", x, weight, bias)
    _need_gpu("layer_norm", x, weight, bias)
    if not _wants_grad(x, weight, bias):                  # (a graph node costs a third of a short call's host time)
        return ops.layer_norm_forward(_rows(x, x.shape[-1]), weight, bias, float(eps), want_stats=False)[0].view(x.shape)
    return _LayerNormFn.apply(x, weight, bias, float(eps))


class LayerNorm(nn.Module):
    """nn.LayerNorm over the last axis on the HIP kernels: the same state_dict keys; normalized_shape is one number, parameters are fp32"""

    def __init__(self, normalized_shape: int, eps: float = 1e-5, elementwise_affine: bool = True, bias: bool = True, device=None):
        super().__init__()
        self.normalized_shape, self.eps = (int(normalized_shape),), float(eps)
        c = self.normalized_shape[0]
        self.weight = nn.Parameter(torch.ones(c, device=device)) if elementwise_affine else None
        self.bias = nn.Parameter(torch.zeros(c, device=device)) if elementwise_affine and bias else None

    def forward(self, x: Tensor) -> Tensor:
        if x.shape[-1:] != self.normalized_shape:
            raise ValueError(f"LayerNorm({self.normalized_shape[0]}): last axis of {tuple(x.shape)}")
        return layer_norm(x, self.weight, self.bias, self.eps)


# ---- attention over packed sequences ----------------------------------------------------------------------------------------
def _heads(t: Tensor) -> Tensor:
    """t [tokens, heads, width] as the kernels read it: contiguous heads, 16-byte aligned, no two on each other, rows less than 2^24 elements apart;
    copied where it is not"""
    (rows, heads, width), (row, head, one) = t.shape, t.stride()
    fits = one == 1 and t.data_ptr() % 16 == 0 and (rows <= 1 or (width <= row < 1 << 24 and row % 8 == 0)) and (heads <= 1 or (head >= width and head % 8 == 0))
    return t if fits else t.clone(memory_format=torch.contiguous_format)


class _PackedAttentionFn(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, table, ends_q, ends_k, bucket_of, causal: bool, scale: Optional[float]):
        _note_graph(ctx, q, k, v, table)
        q, k, v = _heads(q), _heads(k), _heads(v)
        train = any(ctx.needs_input_grad)                 # (narrow heads: the rounding of o would show in dq)
        o, lse, o32 = ops.packed_attention_forward(q, k, v, ends_q, ends_k, causal=causal, scale=scale, table=table, bucket_of=bucket_of,
                                                   want_lse=train, want_o32=train and (q.shape[2] <= 32 or (table is not None and ctx.needs_input_grad[3])))
        ctx.save_for_backward(q, k, v, table, ends_q, ends_k, bucket_of, o, lse, o32)
        ctx.how = (causal, scale)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, dout: Tensor):
        _refuse_stale(ctx, "packed_attention")
        q, k, v, table, ends_q, ends_k, bucket_of, o, lse, o32 = ctx.saved_tensors
        dq, dk, dv, dtable = ops.packed_attention_backward(q, k, v, o, lse, _heads(dout), ends_q, ends_k, causal=ctx.how[0], scale=ctx.how[1], table=table,
                                                           bucket_of=bucket_of, o32=o32, want_dtable=ctx.needs_input_grad[3])
        return dq, dk, dv, dtable, None, None, None, None, None


def packed_attention(q: Tensor, k: Tensor, v: Tensor, ends: Tensor, *, ends_k: Optional[Tensor] = None, causal: bool = False,
                     scale: Optional[float] = None, bias_table: Optional[Tensor] = None, bias_buckets: Optional[Tensor] = None) -> Tensor:
    """softmax(scale q k^T + bias) v within each of several sequences that lie one behind the other.

    q: [tokens, heads, width], k, v: [tokens, shared heads, width], bf16 or fp16; head h uses shared head h // (heads / shared heads).
    width: a multiple of 8 up to 128; scale: 1 / sqrt(width) unless given (positive).  Views of a packed projection's output are read in
    place; what the kernels cannot read in place (rows that are not contiguous or not 16-byte aligned) is copied first.
    ends: int32 [sequences + 1] on the device, ascending from 0: sequence b is the rows ends[b] .. ends[b + 1] - 1 of q (and of k, v, unless
    ends_k gives theirs).  Nothing is read back to the host, and no longest length is needed.  Rows outside of all sequences come out as zeros.
    causal: a query sees the keys up to its own place, counted from the sequences' ends where there are more or fewer keys than queries.
    A query that sees no key gets zeros.  A key or value that is not finite may make NaN of every query of its sequence, also of one that does not
    see it (zero times infinity); other sequences stay as they are.
    bias_table [buckets, heads] (fp32, learned) with bias_buckets [2 far + 1] (int32, relative_position_buckets): adds
    bias_table[bucket of (key's place - query's place), head] to the score.  A bias of -inf hides its distances; finite ones beyond +-5678
    (2^13 powers of two) count as that.  With a bias, a call that will have a gradient of the table keeps more of the probabilities' bits for the
    product with v than one that will not: the results may differ by a rounding.
    Differentiable once in q, k, v and bias_table (in reverse mode)."""
    for name, t in (("q", q), ("k", k), ("v", v)):
        if t.dim() != 3:
            raise ValueError(f"packed_attention: {name} of shape {tuple(t.shape)} is not [tokens, heads, width]")
    _no_tangents("packed_attention", q, k, v, bias_table)
    _need_gpu("packed_attention", q, k, v, ends, ends_k, bias_table, bias_buckets)
    if not _wants_grad(q, k, v, bias_table):
        return ops.packed_attention_forward(_heads(q), _heads(k), _heads(v), ends, ends_k, causal=bool(causal), scale=scale, table=bias_table,
                                            bucket_of=bias_buckets, want_lse=False)[0]
    return _PackedAttentionFn.apply(q, k, v, bias_table, ends, ends_k, bias_buckets, bool(causal), scale)


def relative_position_buckets(num_buckets: int = 32, max_distance: int = 128, bidirectional: bool = True) -> Tensor:
    """Bucket of every distance key - query from -far to far, int32 [2 far + 1] (what is further away shares the bucket at that end; far <=
    max_distance is the first distance of the last bucket).  Half of the buckets (bidirectional: of each direction's half) hold one
    distance each, e = 0, 1, ... of them; the other k have borders that grow geometrically, bucket e + t beginning at the first
    distance n with (n / e)^k >= (max_distance / e)^t.  The borders are found in whole numbers, so that none depends on how a logarithm
    is rounded.  Not bidirectional: keys behind the query share bucket 0."""
    num_buckets, max_distance = int(num_buckets), int(max_distance)
    side = num_buckets // 2 if bidirectional else num_buckets
    e = side // 2
    k = side - e
    if e < 1 or num_buckets % (2 if bidirectional else 1) or not e < max_distance <= 1024:
        raise ValueError(f"relative_position_buckets: {num_buckets} buckets for distances up to {max_distance} "
                         f"(at least {4 if bidirectional else 2} buckets, an even number if bidirectional, distances over {max(e, 1)} and up to 1024)")
    near = [n if n < e else e + min(k - 1, sum(n ** k * e ** t >= max_distance ** t * e ** k for t in range(1, k))) for n in range(max_distance + 1)]
    far = max(4, next(n for n, b in enumerate(near) if b == near[-1]))
    near = (near + [near[-1]] * far)[:far + 1]
    ahead = [(side + b if bidirectional else 0) for b in near[1:]]
    return torch.tensor(near[:0:-1] + near[:1] + ahead, dtype=torch.int32)


class RelativePositionBias(nn.Module):
    """A learned table of one bias per bucket and head, with the buckets of all distances: packed_attention(..., **bias()).  One of them
    may serve every layer of an encoder; its gradient is the sum over the layers."""

    def __init__(self, num_buckets: int, heads: int, max_distance: int = 128, bidirectional: bool = True, device=None):
        super().__init__()
        self.weight = nn.Parameter(torch.zeros(num_buckets, heads, device=device))
        self.register_buffer("buckets", relative_position_buckets(num_buckets, max_distance, bidirectional).to(device), persistent=False)

    def forward(self) -> dict:
        return {"bias_table": self.weight, "bias_buckets": self.buckets}
