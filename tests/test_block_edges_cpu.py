"""Calls of the block's operators that are refused before anything is launched: a batch
of samples, derivatives that are not there, outputs that lie in inputs."""
import ctypes
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


def linear_args(outer=64, stream=BF):
    t = dict(x=torch.zeros(4, 64, dtype=BF), weight=torch.zeros(outer, 64, dtype=BF),
             bias=torch.zeros(outer, dtype=BF), gate=torch.zeros(outer, dtype=BF),
             residual=torch.zeros(4, outer, dtype=stream))
    return t


def call_linear(t, **kw):
    t = dict(t)
    return vggt_sparse.linear(t.pop("x"), t.pop("weight"), **t, **kw)


@pytest.mark.parametrize("which", ["x", "weight", "bias", "gate", "residual", "status"])
def test_linear_out_does_not_lie_in_an_input(which):
    """Tiles that are done write their part of out while others still read: only the residual's own
    elements may be there."""
    t = linear_args()
    room = torch.zeros(16384, dtype=BF)
    t["status"] = torch.zeros(1, dtype=torch.int32)
    n = t[which].numel() * t[which].element_size() // 2
    place = lambda at: room[at:at + n].view(t[which].dtype).view(t[which].shape)  # noqa: E731
    out = room[4096:4352].view(4, 64)
    for at in (4096 - n + 2, 4096, 4350):  # its last elements in out, both from one place on, its first
        if which == "residual" and at == 4096:
            continue
        t[which] = place(at)
        with pytest.raises(ValueError, match="out must not"):
            call_linear(t, out=out)
    # beside it is fine: what is refused then is that there is no GPU
    for at in (4096 - n, 4352):
        t[which] = place(at)
        with pytest.raises(ValueError, match="CUDA tensors"):
            call_linear(t, out=out)


def test_linear_out_may_be_the_residual_or_lie_between_rows():
    t = linear_args()
    with pytest.raises(ValueError, match="CUDA tensors"):
        call_linear(t, out=t["residual"])
    # the same memory by other rows, or in another type
    room = torch.zeros(1024, dtype=BF)
    t["residual"] = room.as_strided((4, 64), (128, 1))
    with pytest.raises(ValueError, match="out must not"):
        call_linear(t, out=room[:256].view(4, 64))
    t["residual"] = room[:64].expand(4, 64)
    with pytest.raises(ValueError, match="out must not"):
        call_linear(t, out=room[:256].view(4, 64))
    # between the rows of x, and of head-major ones
    t = linear_args()
    t["x"] = room.as_strided((4, 64), (320, 1))
    with pytest.raises(ValueError, match="CUDA tensors"):
        call_linear(t, out=room[64:320].view(4, 64))
    with pytest.raises(ValueError, match="out must not"):
        call_linear(t, out=room[65:321].view(4, 64))
    t["x"] = room.as_strided((2, 4, 32), (512, 32, 1))
    with pytest.raises(ValueError, match="CUDA tensors"):
        call_linear(t, out=room[128:384].view(4, 64), head_major=True)
    with pytest.raises(ValueError, match="out must not"):
        call_linear(t, out=room[264:520].view(4, 64), head_major=True)


@pytest.mark.parametrize("which", ["weight", "bias", "gate", "post_weight", "post_bias"])
def test_residual_norm_outputs_do_not_lie_in_parameters(which):
    room = torch.zeros(1024)
    t = {n: torch.zeros(64) for n in ("weight", "bias", "gate", "post_weight", "post_bias")}
    t[which] = room[300:364]
    x, f = torch.zeros(4, 64), torch.zeros(4, 64)
    with pytest.raises(ValueError, match="stream_out must not"):
        vggt_sparse.residual_norm(x, f, post_norm="layer", stream_out=room[256:512].view(4, 64), **t)
    with pytest.raises(ValueError, match="^out must not"):
        vggt_sparse.residual_norm(x, f, post_norm="layer", out=room[256:512].view(4, 64), **t)


def test_residual_norm_outputs_are_rows_of_an_input_or_apart():
    room = torch.zeros(2048)
    x, f = room[:256].view(4, 64), room[1024:1280].view(4, 64)
    call = lambda **kw: vggt_sparse.residual_norm(x, f, **kw)  # noqa: E731
    # a row is read whole before it is written: either output may be either input
    for kw in (dict(out=x), dict(out=f), dict(stream_out=x), dict(stream_out=f),
               dict(out=f, stream_out=x), dict(out=room[256:512].view(4, 64))):
        with pytest.raises(ValueError, match="CUDA tensors"):
            call(**kw)
    for kw in (dict(out=x, stream_out=x), dict(out=room[64:320].view(4, 64)),
               dict(stream_out=room[1000:1256].view(4, 64)),
               dict(out=room[400:656].view(4, 64), stream_out=room[500:756].view(4, 64))):
        with pytest.raises(ValueError, match="out must not"):
            call(**kw)
    # other rows of the same memory, another type
    for x in (room.as_strided((4, 64), (128, 1)), room[:64].expand(4, 64)):
        with pytest.raises(ValueError, match="out must not"):
            call(out=room[:256].view(4, 64))
    with pytest.raises(ValueError, match="out must not"):
        vggt_sparse.residual_norm(room[:256].view(4, 64), dtype=BF,
                                  out=room.view(BF)[:256].view(4, 64))


def test_outputs_that_need_a_gradient_are_refused():
    """Written in place they would keep a gradient that knows nothing of it."""
    out = torch.zeros(4, 64, dtype=BF, requires_grad=True)
    t = linear_args()
    x = torch.zeros(4, 64, dtype=BF)
    for call in (lambda: call_linear(t, out=out), lambda: vggt_sparse.residual_norm(x, x, out=out),
                 lambda: vggt_sparse.residual_norm(x, x, stream_out=out)):
        with pytest.raises(ValueError, match="without a gradient"):
            call()
        with pytest.raises(ValueError, match="CUDA tensors"), torch.no_grad():
            call()


class Rope(torch.nn.Module):
    def __init__(self, base):
        super().__init__()
        self.base_frequency = base


def test_from_module_takes_the_module_s_activation():
    block = parts()
    build = lambda **kw: GlobalBlock.from_module(block, tokens_per_frame=TPF, **kw)  # noqa: E731
    assert build().activation == "gelu"
    for act, name in ((torch.nn.GELU(), "gelu"), (torch.nn.GELU(approximate="tanh"), "gelu_tanh"),
                      (torch.nn.SiLU(), "silu"), (torch.nn.ReLU(), "relu")):
        block.mlp.act = act
        assert build().activation == name
    for act in (torch.nn.Tanh(), torch.nn.LeakyReLU(), torch.nn.Identity()):
        block.mlp.act = act
        with pytest.raises(ValueError, match="activation"):
            build()
        assert build(activation="silu").activation == "silu"


def test_from_module_takes_the_module_s_rope():
    block = parts()
    build = lambda **kw: GlobalBlock.from_module(block, tokens_per_frame=TPF, **kw)  # noqa: E731
    assert build().rope_base == 100.0
    block.attn.rope = Rope(10000.0)
    assert build().rope_base == 10000.0
    assert build(rope_base=50.0).rope_base == 50.0
    block.attn.rope = torch.nn.Identity()
    with pytest.raises(ValueError, match="rope"):
        build()
    assert build(rope_base=50.0).rope_base == 50.0
    block.attn.rope = None  # positions are then not looked at
    assert build().rope_base is None


def test_from_module_without_rope_ignores_positions(monkeypatch):
    from vggt_sparse import block as module
    seen = []

    class Stop(Exception):
        pass

    def project(*args, **kw):
        seen.append(kw["pos"])
        raise Stop
    monkeypatch.setattr(module, "project_qkv", project)
    monkeypatch.setattr(module, "residual_norm", lambda x, *a, **kw: (x, x))
    block = parts()
    x, pos = torch.zeros(TPF, 128), torch.zeros(TPF, 2)
    for rope, given in ((Rope(100.0), True), (None, False)):
        block.attn.rope = rope
        with pytest.raises(Stop):
            GlobalBlock.from_module(block, tokens_per_frame=TPF)(x, pos, 7)
        assert (seen.pop() is not None) == given


def test_linear_takes_a_gate_of_its_type_or_fp32():
    t = linear_args()
    t["gate"] = torch.zeros(64)
    with pytest.raises(ValueError, match="CUDA tensors"):
        call_linear(t)
    for gate in (torch.zeros(64, dtype=FP), torch.zeros(64, dtype=torch.float64), torch.zeros(63)):
        t["gate"] = gate
        with pytest.raises(ValueError, match="gate must be"):
            call_linear(t)


def test_block_keeps_its_scales_in_fp32():
    block = parts()
    block.ls1, block.ls2 = torch.nn.Module(), torch.nn.Module()
    block.ls1.gamma = torch.nn.Parameter(torch.full((128,), 1e-8))
    block.ls2.gamma = torch.nn.Parameter(torch.full((128,), 1e-5))
    half = GlobalBlock.from_module(block, tokens_per_frame=TPF, dtype=FP)
    assert torch.equal(half.ls1, block.ls1.gamma) and torch.equal(half.ls2, block.ls2.gamma)


def test_a_flag_that_is_no_truth_value_is_refused():
    """Its exception must not stay behind a result."""
    t = linear_args()
    with pytest.raises(ValueError, match="head_major must be a truth value"):
        call_linear(t, head_major=torch.zeros(2))
    with pytest.raises(ValueError, match="CUDA tensors"):
        call_linear(t, head_major=0)


class LinearArgs(ctypes.Structure):
    """vggt_linear_args (include/vggt_block.h)."""
    _fields_ = ([(n, ctypes.c_int64) for n in ("rows", "inner", "outer")]
                + [("dtype", ctypes.c_int), ("stream_dtype", ctypes.c_int), ("x", ctypes.c_void_p)]
                + [(n, ctypes.c_int64) for n in ("x_stride", "x_head_stride", "heads")]
                + [("weight", ctypes.c_void_p), ("weight_stride", ctypes.c_int64)]
                + [(n, ctypes.c_void_p) for n in ("bias", "gate", "residual")]
                + [("residual_stride", ctypes.c_int64)]
                + [(n, ctypes.c_int) for n in ("activation", "z_dtype", "gate_fp32")])


@pytest.mark.parametrize("dtype", [0, 1])  # VGGT_DTYPE_BF16, VGGT_DTYPE_FP16
def test_a_gate_is_of_the_products_type_where_nothing_is_said(lib, dtype):
    """A caller that zeroes the arguments and sets what it has had to set so far."""
    a = LinearArgs(rows=0, inner=8, outer=8, dtype=dtype, stream_dtype=dtype, gate=256)
    assert lib.vggt_linear(ctypes.byref(a), None, 8, None, 0, None, None, 0, None) == 0
    a.dtype = 5
    assert lib.vggt_linear(ctypes.byref(a), None, 8, None, 0, None, None, 0, None) < 0
