"""The block's operators where their numbers and layouts go to an edge, against 64-bit code.

Bounds as in test_gpu_block_ops.py (u: unit roundoff of an output's type, v: of the products').
"""
import math

import pytest
import torch

import vggt_sparse
from test_gpu_block_ops import BF, F32, FP, U, Linear, make, near
from vggt_sparse import _lib

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


class Part(torch.nn.Module):
    """The reference block's parts, by its names."""

    def __init__(self, heads, scale=0.3):
        super().__init__()
        dim = heads * 64
        self.norm1, self.norm2 = torch.nn.LayerNorm(dim), torch.nn.LayerNorm(dim, eps=1e-6)
        self.attn, self.mlp = torch.nn.Module(), torch.nn.Module()
        self.attn.num_heads = heads
        self.attn.qkv, self.attn.proj = torch.nn.Linear(dim, 3 * dim), torch.nn.Linear(dim, dim)
        self.attn.q_norm, self.attn.k_norm = torch.nn.LayerNorm(64), torch.nn.LayerNorm(64)
        self.mlp.fc1, self.mlp.fc2 = torch.nn.Linear(dim, 4 * dim), torch.nn.Linear(4 * dim, dim)
        self.ls1, self.ls2 = torch.nn.Module(), torch.nn.Module()
        for ls in (self.ls1, self.ls2):
            ls.gamma = torch.nn.Parameter(scale * torch.randn(dim))


TPF, SPECIAL = 41, 5  # a frame: 5 special tokens and 6 x 6 patches


def positions(frames, dev):
    yy, xx = torch.meshgrid(torch.arange(6), torch.arange(6), indexing="ij")
    grid = torch.stack((yy.flatten() + 1, xx.flatten() + 1), -1)
    return torch.cat((torch.zeros(SPECIAL, 2, dtype=torch.long), grid)).repeat(frames, 1).to(dev)


@pytest.fixture
def short_waits():
    """Every product's first wait runs out, after two milliseconds (and its call returns)."""
    vggt_sparse.check_status()
    limit, test = _lib.set_wait_limit_ns(2_000_000), _lib.set_wait_selftest(True)

    def over():
        torch.cuda.synchronize()
        _lib.set_wait_selftest(test)
        _lib.set_wait_limit_ns(limit)
    yield over
    over()


def test_block_reports_a_wait_that_ran_out(cuda, short_waits):
    block = vggt_sparse.GlobalBlock.from_module(Part(2).to(cuda), tokens_per_frame=TPF, topk=2)
    x = torch.randn(3 * TPF, 128, device=cuda)
    block.mlp(x)
    short_waits()
    with pytest.raises(ValueError, match="earlier call.*timed out"):
        vggt_sparse.check_status()
    want = block.mlp(x)  # reported once, and the context lives
    vggt_sparse.check_status()
    assert torch.equal(block.mlp(x), want)


def test_block_reports_by_its_next_call(cuda, short_waits):
    block = vggt_sparse.GlobalBlock.from_module(Part(2).to(cuda), tokens_per_frame=TPF, topk=2)
    x = torch.randn(3 * TPF, 128, device=cuda)
    block.mlp(x)
    short_waits()
    with pytest.raises(ValueError, match="earlier call.*timed out"):
        block(x, positions(3, cuda), 7)
    assert bool(block(x, positions(3, cuda), 7).isfinite().all())
    vggt_sparse.check_status()


def test_check_status_sees_backward_passes_and_replays(cuda, short_waits):
    """Neither is followed by a copy of the status word."""
    short_waits()
    block = vggt_sparse.GlobalBlock.from_module(Part(2).to(cuda), tokens_per_frame=TPF, topk=2)
    x = torch.randn(3 * TPF, 128, device=cuda, requires_grad=True)
    y = block.mlp(x)
    _lib.set_wait_limit_ns(2_000_000), _lib.set_wait_selftest(True)
    torch.autograd.grad(y, x, torch.ones_like(y))
    short_waits()
    with pytest.raises(ValueError, match="timed out"):
        vggt_sparse.check_status()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    _lib.set_wait_limit_ns(2_000_000), _lib.set_wait_selftest(True)
    with torch.no_grad(), torch.cuda.graph(graph, stream=side):
        block.mlp(x)
    short_waits()
    vggt_sparse.check_status()
    graph.replay()
    with pytest.raises(ValueError, match="timed out"):
        vggt_sparse.check_status()
    vggt_sparse.check_status()


def test_every_call_of_a_block_reports(cuda, monkeypatch):
    """Each operator that a block calls gets the device's status word."""
    from vggt_sparse import block as module, ops
    seen = []

    def spy(place, name):
        real = getattr(place, name)

        def call(*args, **kw):
            seen.append((name, kw["status"].data_ptr()))
            return real(*args, **kw)
        monkeypatch.setattr(place, name, call)
    spy(module, "linear"), spy(module, "project_qkv"), spy(ops, "launch_block_attention")
    block = vggt_sparse.GlobalBlock.from_module(Part(2).to(cuda), tokens_per_frame=TPF, topk=2)
    block(torch.randn(3 * TPF, 128, device=cuda), positions(3, cuda), 7)
    assert sorted(n for n, _ in seen) == ["launch_block_attention"] + 3 * ["linear"] + ["project_qkv"]
    assert len({p for _, p in seen}) == 1


def test_block_does_not_wait_for_the_gpu(cuda):
    block = vggt_sparse.GlobalBlock.from_module(Part(2).to(cuda), tokens_per_frame=TPF, topk=2)
    x, pos = torch.randn(3 * TPF, 128, device=cuda), positions(3, cuda)
    block(x, pos, 7)
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        for _ in range(20):
            block(x, pos, 7)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    vggt_sparse.check_status()
