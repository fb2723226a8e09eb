"""The block's operators where their numbers and layouts go to an edge, against 64-bit code.

Bounds as in test_gpu_block_ops.py (u: unit roundoff of an output's type, v: of the products').
"""
import importlib
import math
import os
import subprocess
import sys
import threading

import pytest
import torch

import vggt_sparse
from test_gpu_block_ops import BF, F32, FP, SMALL, U, Linear, Norm, activation, make, near
from vggt_sparse import _lib

pytestmark = pytest.mark.gpu


class Call(Linear):
    """A call with the bounds of its gradients, in fp16 with those of its factors' subnormal numbers:
    dz is rounded before the products (and so is gate * dy or gate * W), to v of itself or to half a
    subnormal step, 2^-25, for each of the products that are added; a gate of 5e-6 is enough.
    """

    def check_grads(self, dx, dw, db, dg):
        self.define()
        v, step = U[self.dtype], 2.0 ** -25 if self.dtype == FP else 0.0
        dy = self.dy.detach().double().flatten(0, -2)
        one = torch.ones(1, device=dy.device, dtype=dy.dtype)
        g = one if self.g is None else self.g.detach().double()
        z, a, ez = self.z.detach(), self.a.detach(), self.ez.detach()
        zl = z.clone().requires_grad_()
        slope, = torch.autograd.grad(activation(zl, self.act).sum(), zl)
        dz, xd, wd = dy * g * slope, self.xd.detach(), self.wd.detach()
        if self.act is None:
            off = off_w = v * dz.abs()
            off_b = 2.0 ** -22 * dz.abs()
            off_g = v * dy.abs() * (xd.abs() @ wd.abs().t()) + 2.0 ** -20 * dy.abs() * a.abs()
        else:
            off_b = (dy * g).abs() * ((z.abs() <= ez).double() if self.act == "relu"
                                      else v * z.abs() + ez + 1e-5)
            off = off_w = off_b + v * dz.abs()
            off_g = dy.abs() * (1.13 * (v * z.abs() + ez) + 1e-5 * a.abs())
        add = lambda n: 2.0 ** -23 * (n / 16 + 8)  # noqa: E731
        n_rows = dy.shape[0]
        if dx is not None:
            want = dz @ wd
            dx = dx.transpose(0, 1).flatten(1) if self.heads else dx.flatten(0, -2)
            near(dx, want, v * want.abs() + 1.01 * ((off + step) @ wd.abs())
                 + add(self.outer) * (dz.abs() @ wd.abs()) + SMALL, "dx")
        if dw is not None:
            # without an activation the gate scales dW after the product of dy
            want = dz.t() @ xd
            near(dw, want, v * want.abs() + 1.01 * ((off_w + step).t() @ xd.abs())
                 + add(n_rows) * (dz.abs().t() @ xd.abs()) + SMALL, "dw")
        if db is not None:
            want = dz.sum(0)
            near(db, want, v * want.abs() + 1.01 * off_b.sum(0) + 2.0 ** -20 * dz.abs().sum(0) + SMALL,
                 "db")
        if dg is not None:
            want = (dy * a).sum(0)
            mag = (dy.abs() * (xd.abs() @ wd.abs().t())).sum(0)
            near(dg, want, v * want.abs() + 1.01 * off_g.sum(0) + (add(n_rows) + add(self.inner)) * mag
                 + SMALL, "dgate")


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


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("scale", [0.3, 1e-5, 1e-7])
def test_block_keeps_its_scales_per_channel(cuda, dtype, scale):
    """A scale per channel as small as it is initialised, fp16's subnormal numbers and below: on an
    fp32 stream what the block adds is off by the branches' own roundings, not by the scale's.

    The branch p = proj(attention) is rounded once (u) and scaled in fp32; the MLP half rounds y and
    the widened tokens once each and ends in fp32, with three roundings' room for each as in
    test_gpu_block.py: 2 u and 6 u of their norms.  The stream adds 2^-24 of itself, twice.
    """
    torch.manual_seed(3)
    part = Part(2, scale).to(cuda)
    block = vggt_sparse.GlobalBlock.from_module(part, tokens_per_frame=TPF, dtype=dtype, topk=2)
    # a stream of the size of what is added to it, so that it hides nothing
    x, pos = scale * torch.randn(3 * TPF, 128, device=cuda), positions(3, cuda)
    block.norm1 = block.norm1[:2] + (1e-20,)
    block.norm2 = block.norm2[:2] + (1e-20,)
    out = block(x, pos, 7)
    a = block.attention(x, pos, 7)
    d = lambda t: t.double()  # noqa: E731
    p = d(a).transpose(0, 1).flatten(1) @ d(block.proj[0]).t() + d(block.proj[1])
    p = p * d(part.ls1.gamma.detach())
    h = d(x) + p
    y = torch.nn.functional.layer_norm(h, (128,), d(block.norm2[0]), d(block.norm2[1]), 1e-20)
    z = y @ d(block.fc1[0]).t() + d(block.fc1[1])
    m = (z * torch.special.ndtr(z)) @ d(block.fc2[0]).t() + d(block.fc2[1])
    m = m * d(part.ls2.gamma.detach())
    u = U[dtype]
    room = 2 * u * p.norm() + 6 * u * m.norm() + 2 * U[F32] * (h + m).norm()
    assert float((d(out) - h - m).norm()) <= float(room)


SIZES = [(1, 64, 64), (20, 512, 4104), (43, 1001, 517), (129, 72, 257), (300, 136, 1024),
         (1374, 1024, 1024), (2000, 264, 136)]


@pytest.mark.parametrize("rows,inner,outer", SIZES)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("act,residual", [(None, None), ("gelu", F32)])
@pytest.mark.parametrize("misaligned", [False, True])
def test_linear_with_a_gate_in_fp32(cuda, rows, inner, outer, dtype, act, residual, misaligned):
    c = Call(cuda, rows, inner, outer, dtype, act=act, gate=True, residual=residual, seed=outer)
    g = torch.Generator().manual_seed(1)
    c.g = make(g, cuda, outer + 1, dtype=F32, scale=0.5)
    c.g = c.g[1:] if misaligned else c.g[:outer].contiguous()
    with torch.no_grad():
        c.check(c.call())
    leaves = [t.requires_grad_() for t in c.leaves()]
    y = c.call()
    grads = torch.autograd.grad(y, leaves, c.dy, retain_graph=True)
    assert [d.dtype for d in grads] == [t.dtype for t in leaves]
    c.check_grads(*grads[:4])
    one, = torch.autograd.grad(y, c.g, c.dy)
    assert torch.equal(one, grads[3])


def test_linear_without_rows_and_a_gate_in_fp32(cuda):
    x = torch.zeros(0, 64, dtype=BF, device=cuda)
    w = torch.ones(16, 64, dtype=BF, device=cuda)
    g = torch.ones(16, device=cuda, requires_grad=True)
    room = torch.ones(64, device=cuda)  # the allocator's next block, so that zeros are not by chance
    del room
    y = vggt_sparse.linear(x, w, gate=g)
    d, = torch.autograd.grad(y, g, torch.zeros_like(y))
    assert d.dtype == F32 and bool((d == 0).all())


@pytest.mark.parametrize("rows,inner,outer", [(300, 136, 200), (1374, 1024, 1024), (2049, 2056, 2040),
                                              (4000, 1024, 1024), (129, 4096, 128)])
def test_every_product_gives_up_its_waits(cuda, short_waits, rows, inner, outer):
    """One CTA to a tile and pairs, whole and split: each reports and leaves, and what comes after it
    on the SMs is right."""
    short_waits()
    c = Linear(cuda, rows, inner, outer, gate=True, residual=BF)
    want = c.call()
    leaves = [t.requires_grad_() for t in c.leaves()]
    y = c.call()
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    with torch.no_grad():
        _lib.set_wait_limit_ns(2_000_000), _lib.set_wait_selftest(True)
        c.call(status=status)
        short_waits()
        assert int(status) == _lib.STATUS_TIMEOUT
        status.zero_()
        assert torch.equal(c.call(status=status), want) and int(status) == 0
    grads = torch.autograd.grad(y, leaves, c.dy, retain_graph=True)
    _lib.set_wait_limit_ns(2_000_000), _lib.set_wait_selftest(True)
    torch.autograd.grad(y, leaves, c.dy, retain_graph=True)
    short_waits()
    for a, b in zip(grads, torch.autograd.grad(y, leaves, c.dy)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,stream", [(BF, BF), (FP, F32)])
@pytest.mark.parametrize("rows,width,norm,post,groups", [(200, 1024, "layer", "layer", 1),
                                                         (900, 264, "rms", "layer", 1),
                                                         (40, 4096, "layer", "rms", 4),
                                                         (300, 520, "layer", None, 3),
                                                         (33, 2100, "layer", "layer", 0)])
def test_norm_gradients_by_themselves(cuda, dtype, stream, rows, width, norm, post, groups):
    """Each gradient alone, and all but one, have the bits that they have among all."""
    c = Norm(cuda, rows, width, dtype, stream, norm, post, groups=groups)
    leaves = {n: t.requires_grad_() for n, t in c.leaves().items()}
    y, h = c.call()
    take = lambda names: torch.autograd.grad(  # noqa: E731
        (y, h), [leaves[n] for n in names], (c.dy, c.dh), retain_graph=True)
    all_of = dict(zip(leaves, take(list(leaves))))
    c.check(y.detach(), h.detach(), all_of, c.dy, c.dh)
    for n in leaves:
        others = [m for m in leaves if m != n]
        for names in ([n], others):
            for m, d in zip(names, take(names)):
                assert torch.equal(d, all_of[m]), (m, names)


def test_block_first_run_in_inference_mode(cuda, monkeypatch):
    """What the first call sets up must serve calls in every mode."""
    module = importlib.import_module("vggt_sparse.block_attention")
    monkeypatch.setattr(module, "_monitors", {})
    x, pos = torch.randn(3 * TPF, 128, device=cuda), positions(3, cuda)
    with torch.inference_mode():
        block = vggt_sparse.GlobalBlock.from_module(Part(2).to(cuda), tokens_per_frame=TPF, topk=2)
        want = block(x, pos, 7).clone()
    assert torch.equal(block(x, pos, 7), want)
    with torch.no_grad():
        assert torch.equal(block(x, pos, 7), want)
    with torch.inference_mode():
        assert torch.equal(block(x, pos, 7), want)
    vggt_sparse.check_status()


def test_check_status_within_a_capture(cuda):
    """It takes nothing into the graph, and the capture goes on."""
    block = vggt_sparse.GlobalBlock.from_module(Part(2).to(cuda), tokens_per_frame=TPF, topk=2)
    x = torch.randn(3 * TPF, 128, device=cuda)
    want = block.mlp(x)
    vggt_sparse.check_status()
    graph = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(graph):
        out = block.mlp(x)
        vggt_sparse.check_status()
    graph.replay()
    vggt_sparse.check_status()
    assert torch.equal(out, want)


FIRST = """
import sys
import torch
import vggt_sparse
x, w = (torch.ones(n, 64, dtype=torch.bfloat16, device="cuda", requires_grad=True) for n in (200, 64))
y = vggt_sparse.linear(x, w)
dy = torch.ones_like(y)
torch.cuda.synchronize()
dx, dw = torch.autograd.grad(y, (x, w), dy)
assert bool((dx == 64).all()) and bool((dw == 200).all())
"""


def test_first_gradient_of_a_process(cuda):
    """Autograd's thread has no CUDA context of its own before it has called the runtime."""
    path = os.pathsep.join(p for p in sys.path if p)
    subprocess.run([sys.executable, "-c", FIRST], check=True, env=dict(os.environ, PYTHONPATH=path))


def test_first_call_of_a_thread(cuda):
    """Nor has a thread of the caller's."""
    c, out = Linear(cuda, 200, 64, 64), torch.empty(200, 64, dtype=BF, device=cuda)
    want = c.call()
    a = torch.randn(3 * TPF, 128, device=cuda).to(BF)
    w = torch.randn(384, 128, device=cuda).to(BF)
    project = lambda: vggt_sparse.project_qkv(a, w, heads=2, tokens_per_frame=TPF)  # noqa: E731
    q = project().q
    torch.cuda.synchronize()
    got = []
    for run in (lambda: c.call(out=out), lambda: project().q):
        thread = threading.Thread(target=lambda: got.append(run()))
        thread.start()
        thread.join()
    assert len(got) == 2 and torch.equal(got[0], want) and torch.equal(got[1], q)
