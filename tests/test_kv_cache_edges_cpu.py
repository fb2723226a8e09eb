"""Refusals and page accounting of the streaming cache at the edges, without a
GPU: refusals come before any CUDA call."""
import pytest
import torch

import vggt_sparse


@pytest.fixture(scope="module", autouse=True)
def built():
    import os
    from vggt_sparse import _lib, build
    if not os.path.exists(_lib.LIB_PATH) or not os.path.exists(build.BINDING_PATH):
        build.build()


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("workspace", [torch.zeros(1, dtype=torch.uint8).expand(1 << 20),
                                       torch.zeros(1 << 20, dtype=torch.uint8)[::2]])
def test_workspace_must_be_contiguous(workspace):
    """An expanded tensor has as many elements as it says, but not as many bytes."""
    q = torch.zeros(4, 4, 64, dtype=torch.bfloat16)
    pool = torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="workspace must be contiguous"):
        vggt_sparse.paged_attention(q, pool, pool, ints(1, 3), ints(1), ints(2), max_new=1,
                                    workspace=workspace)
