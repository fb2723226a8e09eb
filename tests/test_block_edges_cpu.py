"""Calls of the block's operators that are refused before anything is launched: a batch
of samples, derivatives that are not there, outputs that lie in inputs."""
import os

import pytest
import torch
import torch.autograd.forward_ad as fwAD

import vggt_sparse
from vggt_sparse import GlobalBlock

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
TPF = 41


@pytest.fixture(scope="module", autouse=True)
def lib():
    from vggt_sparse import _lib, build
    if not os.path.exists(_lib.LIB_PATH) or not os.path.exists(build.BLOCK_BINDING_PATH):
        build.build()
    return _lib.load()


def parts(dim=128):
    """The reference block's parts, by its names."""
    block = torch.nn.Module()
    block.norm1, block.norm2 = torch.nn.LayerNorm(dim), torch.nn.LayerNorm(dim)
    block.attn, block.mlp = torch.nn.Module(), torch.nn.Module()
    block.attn.num_heads = dim // 64
    block.attn.qkv, block.attn.proj = torch.nn.Linear(dim, 3 * dim), torch.nn.Linear(dim, dim)
    block.attn.q_norm = block.attn.k_norm = torch.nn.LayerNorm(64)
    block.mlp.fc1, block.mlp.fc2 = torch.nn.Linear(dim, 4 * dim), torch.nn.Linear(4 * dim, dim)
    block.ls1 = block.ls2 = torch.nn.Identity()
    return block


@pytest.mark.parametrize("shape,text", [((2, TPF, 128), "batch one only"),
                                        ((3, 2 * TPF, 128), "batch one only"),
                                        ((0, TPF, 128), "batch one only"),
                                        ((1, 1, TPF, 128), r"x must be \[N, C\]"),
                                        ((128,), r"x must be \[N, C\]")])
def test_block_takes_one_sample(shape, text):
    block = GlobalBlock.from_module(parts(), tokens_per_frame=TPF)
    x = torch.zeros(shape, dtype=BF)
    pos = torch.zeros(*shape[:-1], 2, dtype=torch.long)
    with pytest.raises(ValueError, match=text):
        block(x, pos, 7)


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("which", ["x", "weight", "bias", "gate", "residual"])
def test_linear_refuses_forward_mode(which, graph):
    """A dual tensor needs no backward graph: without a look at its tangent the result would have
    none, which reads as zero."""
    t = dict(x=torch.zeros(4, 64, dtype=BF), weight=torch.zeros(16, 64, dtype=BF),
             bias=torch.zeros(16, dtype=BF), gate=torch.zeros(16, dtype=BF),
             residual=torch.zeros(4, 16, dtype=F32))
    if graph:
        t["x"].requires_grad_()
    with fwAD.dual_level():
        t[which] = fwAD.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(ValueError, match="forward-mode"):
            vggt_sparse.linear(t.pop("x"), t.pop("weight"), **t)


@pytest.mark.parametrize("which", ["x", "branch", "weight", "bias", "gate", "post_weight", "post_bias"])
def test_residual_norm_refuses_forward_mode(which):
    t = {n: torch.zeros(64) for n in ("weight", "bias", "gate", "post_weight", "post_bias")}
    t.update(x=torch.zeros(4, 64), branch=torch.zeros(4, 64))
    with fwAD.dual_level():
        t[which] = fwAD.make_dual(t[which], torch.ones_like(t[which]))
        with pytest.raises(ValueError, match="forward-mode"), torch.no_grad():
            vggt_sparse.residual_norm(t.pop("x"), post_norm="layer", **t)
        with pytest.raises(ValueError, match="forward-mode"):
            vggt_sparse.residual_norm(torch.zeros(4, 64), out=fwAD.make_dual(
                torch.zeros(4, 64), torch.ones(4, 64)))
