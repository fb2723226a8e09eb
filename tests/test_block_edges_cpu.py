"""Calls of the block's operators that are refused before anything is launched: a batch
of samples, derivatives that are not there, outputs that lie in inputs."""
import os

import pytest
import torch

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
