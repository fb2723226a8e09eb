"""The block's operators where their numbers and layouts go to an edge, against 64-bit code.

Bounds as in test_gpu_block_ops.py (u: unit roundoff of an output's type, v: of the products').
"""
import math

import pytest
import torch

import vggt_sparse
from test_gpu_block_ops import BF, F32, FP, U, Linear, make, near

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e-3, 1e-4, 1e-5, 1e-6])
@pytest.mark.parametrize("rows,inner,outer", [(1100, 1024, 1024), (300, 256, 1000), (200, 512, 300)])
@pytest.mark.parametrize("misaligned", [False, True])
def test_fp16_gradient_with_small_gates(cuda, scale, rows, inner, outer, misaligned):
    """A scale per channel as it is initialised, and a loss scaled up until dy * gate is far from
    fp16's subnormal numbers: dx is off by its own rounding and one of a factor, no more.

    The factor dy * gate is off by v of itself, or by half a subnormal step (2^-25); the sum over
    `outer` products of fp32 as everywhere; the result by v, or half a subnormal step.
    """
    c = Linear(cuda, rows, inner, outer, FP, gate=True, bias=False)
    g = torch.Generator().manual_seed(rows)
    c.g = make(g, cuda, outer, dtype=FP, scale=scale)
    c.dy = make(g, cuda, rows, outer + 3, dtype=FP, scale=min(1e4, 0.04 / scale))
    c.dy = c.dy[:, 3:] if misaligned else c.dy[:, :outer].contiguous()
    c.x.requires_grad_()
    dx, = torch.autograd.grad(c.call(), c.x, c.dy)
    dz, w, v = c.dy.double() * c.g.double(), c.w.double(), U[FP]
    want = dz @ w
    room = (v * want.abs() + 1.01 * (v * dz.abs() + 2.0 ** -25) @ w.abs()
            + 2.0 ** -23 * (outer / 16 + 8) * (dz.abs() @ w.abs()) + 2.0 ** -25)
    near(dx, want, room, "dx")
