"""The block's dense operators without a GPU: the header, the library's symbols,
refused arguments (all found before anything is launched)."""
import ctypes
import os
import re
import shutil
import subprocess

import pytest
import torch

import vggt_sparse
from conftest import REPO
from vggt_sparse import block_ops

HEADER = os.path.join(REPO, "include", "vggt_block.h")
BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def lib():
    from vggt_sparse import _lib, build
    if not os.path.exists(_lib.LIB_PATH) or not os.path.exists(build.BLOCK_BINDING_PATH):
        build.build()
    return _lib.load()


def declared():
    return sorted(set(re.findall(r"^\w[\w\s\*]*?\b(vggt_\w+)\s*\(", open(HEADER).read(), re.M)))


def test_header_and_library_agree(lib):
    from vggt_sparse import _lib
    assert declared() == ["vggt_linear", "vggt_linear_grad", "vggt_linear_grad_workspace_size",
                          "vggt_linear_workspace_size", "vggt_residual_norm",
                          "vggt_residual_norm_grad", "vggt_residual_norm_grad_workspace_size"]
    for name in declared():
        assert hasattr(lib, name) and name in _lib.SIGNATURES


@pytest.mark.parametrize("lang,std", [("c", "-std=c99"), ("c++", "-std=c++17")])
def test_header_compiles_alone(lang, std):
    cc = shutil.which("gcc" if lang == "c" else "g++")
    if cc is None:
        pytest.skip("no host compiler")
    res = subprocess.run([cc, "-fsyntax-only", "-x", lang, std, "-Wall", "-Wextra", "-pedantic",
                          "-Werror", HEADER], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def test_null_arguments_are_refused(lib):
    null = ctypes.c_void_p(None)
    assert lib.vggt_linear(null, null, 0, null, 0, null, null, 0, null) < 0
    assert lib.vggt_linear_grad(null, null, null, null, 0, null) < 0
    assert lib.vggt_residual_norm(null, null, 0, null, 0, null) < 0
    assert lib.vggt_residual_norm_grad(null, null, null, 0, null) < 0
    assert lib.vggt_linear_workspace_size(null) == 0
    assert lib.vggt_linear_grad_workspace_size(null, null) == 0
    assert lib.vggt_residual_norm_grad_workspace_size(0, 64, 0) == 0


def z(*shape, dtype=BF):
    return torch.zeros(*shape, dtype=dtype)


@pytest.mark.parametrize("change,text", [
    (dict(x=z(4, 64, dtype=F32)), "BF16 or FP16"),
    (dict(x=z(4, 72)), "inner size"),
    (dict(weight=z(16, 64, dtype=FP)), "of x's dtype"),
    (dict(weight=z(64)), "weight must be"),
    (dict(weight=z(0, 64)), "weight must be"),
    (dict(bias=z(17)), "bias must be"),
    (dict(bias=z(16, dtype=F32)), "bias must be"),
    (dict(gate=z(1, 16)), "gate must be"),
    (dict(residual=z(5, 16)), "residual must have"),
    (dict(residual=z(4, 16, dtype=FP)), "residual must be"),
    (dict(activation="tanh"), "activation must be"),
    (dict(head_major=True), "head-major"),
    (dict(x=z(4, 3, 15), head_major=True), "head-major"),
    (dict(out=z(4, 17)), "out must be"),
    (dict(out=z(4, 16, dtype=F32)), "out must be"),
    (dict(out=z(16, 4).t()), "out must be"),
    (dict(status=z(1, dtype=F32)), "status"),
    (dict(x=3), "x must be a tensor"),
    (dict(), "CUDA tensors"),
])
def test_linear_refuses(change, text):
    args = dict(x=z(4, 64), weight=z(16, 64))
    args.update(change)
    with pytest.raises(ValueError, match=text):
        vggt_sparse.linear(args.pop("x"), args.pop("weight"), args.pop("bias", None), **args)


@pytest.mark.parametrize("change,text", [
    (dict(x=z(4, 64, dtype=torch.float64)), "BF16, FP16 or FP32"),
    (dict(x=z(4, 64, dtype=FP)), "branch's dtype"),
    (dict(branch=z(4, 65)), "x's shape"),
    (dict(branch=z(4, 64, dtype=F32)), "branch's dtype"),
    (dict(weight=z(63)), "weight must be"),
    (dict(bias=z(1, 64)), "bias must be"),
    (dict(gate=z(3, 64)), "multiple of gate's"),
    (dict(gate=z(2, 2, 64)), "gate must be"),
    (dict(gate=z(4)), "gate must be"),
    (dict(branch=None, gate=z(64)), "need a branch"),
    (dict(branch=None, post_norm="rms"), "need a branch"),
    (dict(post_weight=z(64)), "need a post_norm"),
    (dict(norm="batch"), "norm must be"),
    (dict(norm=None), "norm must be"),
    (dict(post_norm="batch"), "post_norm must be"),
    (dict(eps="small"), "eps must be"),
    (dict(dtype=F32), "dtype is the branch's"),
    (dict(dtype="bf16"), "torch.dtype"),
    (dict(branch=None, dtype=FP), "x must be of"),
    (dict(out=z(4, 63)), "out must be"),
    (dict(stream_out=z(4, 64, dtype=F32)), "stream_out must be"),
    (dict(branch=None, stream_out=z(4, 64)), "stream_out needs a branch"),
    (dict(), "CUDA tensors"),
])
def test_residual_norm_refuses(change, text):
    args = dict(x=z(4, 64), branch=z(4, 64))
    args.update(change)
    with pytest.raises(ValueError, match=text):
        vggt_sparse.residual_norm(args.pop("x"), args.pop("branch"), args.pop("weight", None),
                                  args.pop("bias", None), **args)


def test_outputs_are_not_given_where_a_gradient_is_needed():
    x, w = z(4, 64).requires_grad_(), z(16, 64)
    with pytest.raises(ValueError, match="without a gradient"):
        vggt_sparse.linear(x, w, out=z(4, 16))
    with pytest.raises(ValueError, match="without a gradient"):
        vggt_sparse.residual_norm(x, z(4, 64), out=z(4, 64))
    with pytest.raises(ValueError, match="without a gradient"):
        vggt_sparse.residual_norm(x, z(4, 64), stream_out=z(4, 64))


def test_missing_binding_fails_loudly(monkeypatch):
    from vggt_sparse import _lib
    monkeypatch.setattr(block_ops, "_module", None)
    monkeypatch.setattr(block_ops, "BLOCK_BINDING_PATH", "/nonexistent/_block_binding.so")
    with pytest.raises(_lib.ExtensionMissing):
        vggt_sparse.linear(z(4, 64), z(16, 64))
