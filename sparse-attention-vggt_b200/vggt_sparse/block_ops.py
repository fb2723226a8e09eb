"""The dense operators around a block's attention.

``linear``         a matrix product with bias, activation, gate and residual in
                   its epilogue: y = residual + gate * activation(x W^T + b)
``residual_norm``  the end of one half of a block and the start of the next:
                   h = x + gate * post_norm(branch), y = norm(h)

With ``project_qkv`` and the attention they make up the reference's block
(saf3r/models/official_vggt/layers/block.py:81-107: LayerNorm, attention,
projection, LayerScale, residual, LayerNorm, MLP, LayerScale, residual);
``GlobalBlock`` (block.py) is that block.

Both are differentiable, once, in all their tensors, by a backward pass (tensors
with a forward-mode tangent are refused).  Sums, statistics and
activations are formed in fp32 and rounded once, to the result's type; a
backward pass adds in a fixed order, so that equal calls give equal results, and
a gradient is the same alone and among others.

Like the other operators these only enqueue work on the current stream of their
tensors' device, and may be captured in CUDA graphs.
"""
import os

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


def linear(x, weight, bias=None, *, activation=None, gate=None, residual=None, head_major=False,
           out=None, status=None):
    """residual + gate * activation(x @ weight.T + bias), in one kernel.

    x [..., inner] bf16 or fp16, weight [outer, inner] and bias [outer] of x's
    dtype, gate [outer] of x's dtype or fp32; residual [..., outer] of x's dtype
    or fp32, which is then the result's.  ``head_major``: x is [heads, rows, dim],
    as the attention operators return it, and is read in place as
    [rows, heads * dim] (the result is [rows, outer]).  ``activation`` is None, "gelu" (with the normal
    distribution), "gelu_tanh", "silu" or "relu"; ``gate`` scales per channel
    (LayerScale).

    x and weight are copied where their rows do not start on 16 bytes.  For a
    backward pass the activation's argument is kept, rounded to x's dtype (with a
    gate in fp32); without an activation x, weight, bias and gate alone are.
    Gradients of the products are rounded to x's dtype: with fp16 scale the loss,
    as ever, where they may fall below its range.

    ``out`` (contiguous; residual itself, or apart from every input) takes the
    result where no gradient is needed.  ``status``, an int32 tensor, gets
    VGGT_STATUS_TIMEOUT if a wait of the kernel, or of its backward pass, ran out.
    """
    return _binding().linear(x, weight, bias, activation, gate, residual, head_major, out, status)


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

    ``out`` and ``stream_out`` (contiguous; each x or branch itself, or apart from
    every input and from the other) take y and h where no gradient is needed.
    """
    return _binding().residual_norm(x, branch, weight, bias, gate, post_weight, post_bias, norm,
                                    post_norm, eps, dtype, out, stream_out)
