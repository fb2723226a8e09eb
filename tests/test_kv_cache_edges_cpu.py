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


def test_workspace_size_of_any_expectation():
    """What is expected beyond what can be counts as the most that can be."""
    size = vggt_sparse.paged_attention_workspace_size
    for total, seqs, heads, group, dim in ((40, 2, 8, 4, 64), (1, 1, 16, 1, 128), (1374, 1, 16, 1, 64)):
        most = size(total, seqs, heads, group, dim, total, 2 ** 31 - 1)
        for max_new in (total, 2 ** 40, 2 ** 61, 2 ** 62, 2 ** 63 - 1):
            for max_len in (2 ** 31, 2 ** 50, 2 ** 62, 2 ** 63 - 1):
                assert size(total, seqs, heads, group, dim, max_new, max_len) == most


def test_binding_is_built_again_for_another_torch(monkeypatch, tmp_path):
    """The compiled module holds for the torch and the Python it was built for."""
    import subprocess
    from vggt_sparse import build
    made = []

    def run(cmd, **kw):
        made.append(cmd)
        (tmp_path / "binding.so").write_text("")
        return subprocess.CompletedProcess(cmd, 0, "", "")
    monkeypatch.setattr(build, "BINDING_PATH", str(tmp_path / "binding.so"))
    monkeypatch.setattr(build, "BUILD_DIR", str(tmp_path))
    monkeypatch.setattr(build.subprocess, "run", run)
    for version, builds in ((torch.__version__, 1), (torch.__version__, 1), ("0.1", 2), ("0.1", 2),
                            (torch.__version__, 3)):
        monkeypatch.setattr(torch, "__version__", version)
        build._build_binding(False)
        assert len(made) == builds
    build._build_binding(True)
    assert len(made) == 4


def test_runs_are_not_split_where_partial_results_cost_more():
    """The workspace shows the split: many row tiles stay whole (16 KB of
    counters alone), few ones over a long cache are cut."""
    size = vggt_sparse.paged_attention_workspace_size
    assert size(7300, 4, 8, 4, 128, 1999, 14288) == 16384
    assert size(3900, 8, 8, 4, 128, 500, 8500) == 16384
    frame = 11 * 16 * 128 * (64 + 2) * 4  # a run of each item
    assert size(1374, 1, 16, 1, 64, 1374, 43968) == 16384 + 5 * frame
