"""The dense operators around a block's attention.

``linear``         a matrix product with bias, activation, gate and residual in
                   its epilogue: y = residual + gate * activation(x W^T + b)
``residual_norm``  the end of one half of a block and the start of the next:
                   h = x + gate * post_norm(branch), y = norm(h)

With ``project_qkv`` and the attention they make up the reference's block
(saf3r/models/official_vggt/layers/block.py:81-107: LayerNorm, attention,
projection, LayerScale, residual, LayerNorm, MLP, LayerScale, residual);
``GlobalBlock`` (block.py) is that block.

Both are differentiable, once, in all their tensors.  Sums, statistics and
activations are formed in fp32 and rounded once, to the result's type; a
backward pass adds in a fixed order, so that equal calls give equal results.

Like the other operators these only enqueue work on the current stream of their
tensors' device, and may be captured in CUDA graphs.
"""
import os

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from .build import BLOCK_BINDING_PATH

_module = None


def _binding():
    """The compiled module of csrc/block_binding.cpp, which checks arguments
    and calls the C ABI; there is no fallback."""
    global _module
    if _module is None:
        if not os.path.exists(BLOCK_BINDING_PATH):
            raise _lib.ExtensionMissing("%s not found: build it with `python -m vggt_sparse.build`"
                                        % BLOCK_BINDING_PATH)
        _lib.load()
        from . import _block_binding
        _module = _block_binding
    return _module


def _any_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and getattr(t, "requires_grad", False):
                return True
    return False


def _bits(needs):
    return sum(1 << i for i, n in enumerate(needs) if n)


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, gate, residual, activation, head_major, status):
        keep = activation is not None
        y = _binding().linear(x, weight, bias, activation, gate, residual, head_major, None, keep,
                              status)
        y, z = y if keep else (y, None)
        ctx.save_for_backward(x, weight, bias, gate, z)
        ctx.how = activation, head_major, status
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias, gate, z = ctx.saved_tensors
        activation, head_major, status = ctx.how
        needs = ctx.needs_input_grad
        grads = (None,) * 4
        if any(needs[:4]):
            grads = _binding().linear_grad(x, weight, bias, activation, gate, None, head_major, dy,
                                           z, _bits(needs[:4]), status)
        return (*grads, dy if needs[4] else None, None, None, None)


def linear(x, weight, bias=None, *, activation=None, gate=None, residual=None, head_major=False,
           out=None, status=None):
    """residual + gate * activation(x @ weight.T + bias), in one kernel.

    x [..., inner] bf16 or fp16, weight [outer, inner], bias and gate [outer],
    all of x's dtype; residual [..., outer] of x's dtype or fp32, which is then
    the result's.  ``head_major``: x is [heads, rows, dim], as the attention
    operators return it, and is read in place as [rows, heads * dim] (the result
    is [rows, outer]).  ``activation`` is None, "gelu" (with the normal
    distribution), "gelu_tanh", "silu" or "relu"; ``gate`` scales per channel
    (LayerScale).

    x and weight are copied where their rows do not start on 16 bytes or have an
    inner size that is not a multiple of 8.  For a backward pass the activation's
    argument is kept, rounded to x's dtype; without an activation x, weight, bias
    and gate alone are.

    ``out`` (contiguous; may be residual) takes the result where no gradient is
    needed.  ``status``, an int32 tensor, gets VGGT_STATUS_TIMEOUT if a wait of
    the kernel ran out.
    """
    if _any_grad(x, weight, bias, gate, residual):
        if out is not None:
            raise ValueError("out is for calls without a gradient")
        return _Linear.apply(x, weight, bias, gate, residual, activation, head_major, status)
    return _binding().linear(x, weight, bias, activation, gate, residual, head_major, out, False,
                             status)


class _ResidualNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, branch, weight, bias, gate, post_weight, post_bias, norm, post_norm, eps,
                dtype):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(x, branch, weight, bias, gate, post_weight, post_bias)
        y, h = _binding().residual_norm(x, branch, weight, bias, gate, post_weight, post_bias, norm,
                                        post_norm, eps, dtype, None, None)
        ctx.how = norm, post_norm, eps, dtype
        return y if branch is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        needs = ctx.needs_input_grad[:7]
        if dy is None and dh is None:
            return (None,) * 11
        grads = _binding().residual_norm_grad(*ctx.saved_tensors, *ctx.how, dy, dh, _bits(needs))
        return (*grads, None, None, None, None)


def residual_norm(x, branch=None, weight=None, bias=None, *, norm="layer", gate=None,
                  post_norm=None, post_weight=None, post_bias=None, eps=1e-5, dtype=None, out=None,
                  stream_out=None):
    """(y, h): h = x + gate * post_norm(branch), y = norm(h) * weight + bias.

    x [..., width] is the residual stream (bf16, fp16 or fp32; width at most
    16384), branch [..., width] of x's dtype or, where that is fp32, of any.  h
    has x's dtype, y the branch's; without a branch h is x itself, and y has
    ``dtype`` (x's by default).

    ``norm`` and ``post_norm`` are "layer" or "rms" (``post_norm`` may be None:
    the branch is added as it is, with its gate).  Weights and biases are [width],
    ``gate`` is [width], or [groups, width] for as many runs of equally many
    rows each (a gate per sample of a batch, or per row), in any of the three
    dtypes.

    ``out`` and ``stream_out`` (contiguous; stream_out may be x) take y and h
    where no gradient is needed.
    """
    if _any_grad(x, branch, weight, bias, gate, post_weight, post_bias):
        if out is not None or stream_out is not None:
            raise ValueError("out and stream_out are for calls without a gradient")
        both = _ResidualNorm.apply(x, branch, weight, bias, gate, post_weight, post_bias, norm,
                                   post_norm, eps, dtype)
        return (both, x) if branch is None else both
    return _binding().residual_norm(x, branch, weight, bias, gate, post_weight, post_bias, norm,
                                    post_norm, eps, dtype, out, stream_out)
