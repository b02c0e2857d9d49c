"""``query_attention``: dense attention among the queries of a deformable decoder (or of queries over a memory), the layer
between two sampling ones, on matrix-core kernels forward and backward.

For every sequence and head, with ``scale`` the inverse root of the head width unless it is given,

    x_ij = scale * query_i . key_j
    s_ij = cap * tanh(x_ij / cap) - slopes[head] * |positions_i - key_positions_j|
    out_i = sum over the keys j that query i sees of softmax(s_i)_j * value_j

without the tanh where ``cap`` is 0 and without the distance where there are no positions.  Query i sees key j if i's segment
number is not negative and j's is the same or 0:

  * groups of denoising queries (1, 2, ...) that see themselves and the matching queries (0), which see each other alone;
  * sequences packed one behind the other (1, 2, ...), with or without a prefix (0) that all see;
  * padding (any negative number), which nothing sees and which sees nothing.

A row that sees nothing is zeros and sends no gradient.  What a row does not see has no influence on it whatever it holds,
infinities and NaN too.  One that it does see in a value takes its channel of the head's result with it, or the head's whole result of that
row: which of the two is a matter of how the keys fall into tiles.  Other heads, and rows that do not see it, are left as they are.

Gradients form the weights again from the logarithm of a row's sum, in fp32: they are off by 2^-23 of the size of the row's largest score, relatively.
A row whose largest score passes 7e5 in size, as where even the nearest key is that far away times the slope, has its result, and NaN as gradients.
"""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import ext

_native = ext._native


class QueryAttentionFunction(Function):
    """``apply(query, key, value, segments, key_segments, positions, key_positions, slopes, scale, cap)``, nothing left out."""

    @staticmethod
    def apply(*args):
        output = _native.query_attention(*args)      # None: declined, as under a tracer
        return super(QueryAttentionFunction, QueryAttentionFunction).apply(*args) if output is None else output

    @staticmethod
    def forward(ctx, query, key, value, segments, key_segments, positions, key_positions, slopes, scale, cap):
        args = (query, key, value, segments, key_segments, positions, key_positions, slopes)
        output, rest, lse = ext.query_attention_forward(*args, scale, cap)
        ctx.save_for_backward(*args, output, rest, lse)
        ctx.scalars = (scale, cap)
        return output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output):
        *args, output, rest, lse = ctx.saved_tensors
        grad_query, grad_key, grad_value, grad_slopes = ext.query_attention_backward(*args, *ctx.scalars, output, rest, lse,
                                                                                           grad_output)
        return grad_query, grad_key, grad_value, None, None, None, None, grad_slopes, None, None


def query_attention(query, key, value, *, scale=None, cap=0.0, segments=None, key_segments=None, positions=None,
                    key_positions=None, slopes=None):
    """``query`` (N, Lq, M, D), ``key`` and ``value`` (N, Lk, Mk, D) with M a multiple of Mk (heads that follow each other share a
    key head) and D up to 128, all float32, float16 or bfloat16; views of a fused projection are read as they lie.  ``segments``
    (N, Lq) and ``key_segments`` (N, Lk) int32: for self-attention one is enough; ``key_segments`` alone (0 and -1: padded keys)
    counts all queries as 0.  ``positions`` (N, Lq, 2), ``key_positions`` (N, Lk, 2; the queries' own if left out) and ``slopes``
    (M,) float32.  ``scale`` is at most 1e30 in size, ``cap`` 0 or 1e-30 to 1e30, the first at most 1e30 times the second.  Gradients
    reach query, key, value and slopes.  Under autocast the first three are cast to its type.  Returns (N, Lq, M, D)."""
    for points in (positions, key_positions):
        if points is not None and points.requires_grad and torch.is_grad_enabled():
            raise RuntimeError("query_attention has no gradient for positions: detach them")
    cap = float(cap or 0.0)
    if cap != 0.0 and not 1e-30 <= cap <= 1e30:      # (what is smaller is zero as a float)
        raise RuntimeError("cap must be zero (none) or between 1e-30 and 1e30")
    if torch.is_autocast_enabled() and query.is_cuda:
        dtype = torch.get_autocast_dtype("cuda")
        query, key, value = (t.to(dtype) if t.is_floating_point() and t.dtype != torch.float64 else t for t in (query, key, value))
    if key_segments is None:
        key_segments = segments
    if key_positions is None:
        key_positions = positions
    if scale is None:
        scale = query.shape[-1] ** -0.5 if query.dim() and query.shape[-1] else 1.0
    return QueryAttentionFunction.apply(query, key, value, segments, key_segments, positions, key_positions, slopes, float(scale), cap)
