"""``add_layer_norm``: ``norm(x + residual)``, the step between the layers of a transformer, as one kernel forward and two
backward; the sum is not rounded before it is normalised.

Runs on the library's kernels for rows of up to 8192 channels of any layout whose channels are dense, of any mix of float32 with
one 16-bit type; otherwise (other types, CPU tensors, a norm over several axes; a norm with hooks or a forward of its own, which run) the
expression is left to torch's own operators and autograd.
"""
import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from .. import ext

_native = ext._native
_MAX_CHANNELS = 8192
_TYPES = (torch.float32, torch.float16, torch.bfloat16)


class AddLayerNormFunction(Function):
    """``apply(input, residual, weight, bias, eps, wide, want_sum)``: the result, or (result, sum)."""

    @staticmethod
    def apply(*args):
        output = _native.add_layer_norm(*args)      # None: declined, as under a tracer
        return super(AddLayerNormFunction, AddLayerNormFunction).apply(*args) if output is None else output

    @staticmethod
    def forward(ctx, input, residual, weight, bias, eps, wide, want_sum):
        output, total, stats = ext.add_layer_norm_forward(input, residual, weight, bias, eps, wide)
        ctx.save_for_backward(input, residual, weight, bias, stats)
        ctx.scalars = (eps, wide)
        ctx.set_materialize_grads(False)
        return (output, total) if want_sum else output

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_output, grad_sum=None):
        input, residual, weight, bias, stats = ctx.saved_tensors
        if grad_output is None:
            around = [None if t is None or grad_sum is None else grad_sum.to(t.dtype) for t in (input, residual)]
            return (*around, None, None, None, None, None)
        return (*ext.add_layer_norm_backward(input, residual, weight, bias, *ctx.scalars, stats, grad_output, grad_sum), None, None, None)


def _fusable(x, residual, norm):
    if not x.is_cuda or not 1 <= x.shape[-1] <= _MAX_CHANNELS:
        return False
    tensors = [t for t in (x, residual, norm.weight, norm.bias) if t is not None]
    halves = {t.dtype for t in tensors if t.dtype != torch.float32}
    if any(t.dtype not in _TYPES or t.device != x.device for t in tensors) or len(halves) > 1:
        return False
    if norm.weight is not None and norm.bias is not None and norm.weight.dtype != norm.bias.dtype:
        return False
    return residual is None or residual.shape == x.shape


def add_layer_norm(x, residual, norm, return_sum=False):
    """``norm(x + residual)`` for an ``nn.LayerNorm`` over the last axis; ``residual`` of x's shape, or None.  The result has the
    wider type of the two, float32 under autocast as torch's own layer norm there.  With ``return_sum`` also the sum, in the wider type:
    ``(result, x + residual)``, the stream of a pre-norm network.  The backward reads x and residual again: neither is to be changed in
    place before it."""
    output = _native.add_layer_norm_of(norm, x, residual, return_sum)
    if output is not None:
        return output
    if x.dim() and _native.plain_layer_norm(norm, x.shape[-1]) and _fusable(x, residual, norm):
        return AddLayerNormFunction.apply(x, residual, norm.weight, norm.bias, norm.eps, torch.is_autocast_enabled(), bool(return_sum))
    total = x if residual is None else x + residual
    out = norm(total)
    return (out, total) if return_sum else out
