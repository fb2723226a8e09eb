"""GlobalBlock: the dense operators and the sparse attention as one block.

The block's result against 64-bit code from its own attention on.  Bounds are norms
over the whole result; u is the unit roundoff of the block's type.  Every product and
norm rounds its result once (u) and reads an input that was rounded once: the attention
half adds p (u), scaled by ls1; the MLP half y, the widened tokens and the result, three
roundings, each carried on by maps whose gain the norms below contain.  So the branches
are off by 2 u and 6 u of their norms at most, and the result by u more (in its type).
"""
import pytest
import torch

import vggt_sparse
from vggt_sparse import GlobalBlock, SparseGlobalLayer

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0 ** -8, FP: 2.0 ** -11, F32: 2.0 ** -24}
TPF, SPECIAL = 41, 5  # a frame: 5 special tokens and 6 x 6 patches


class Scale(torch.nn.Module):
    def __init__(self, dim):
        super().__init__()
        self.gamma = torch.nn.Parameter(0.3 * torch.randn(dim))


class Module(torch.nn.Module):
    """The reference block's parts, by its names."""

    def __init__(self, heads, scales=True):
        super().__init__()
        dim = heads * 64
        self.norm1, self.norm2 = torch.nn.LayerNorm(dim), torch.nn.LayerNorm(dim, eps=1e-6)
        self.attn = torch.nn.Module()
        self.attn.num_heads = heads
        self.attn.qkv, self.attn.proj = torch.nn.Linear(dim, 3 * dim), torch.nn.Linear(dim, dim)
        self.attn.q_norm, self.attn.k_norm = torch.nn.LayerNorm(64), torch.nn.LayerNorm(64)
        self.mlp = torch.nn.Module()
        self.mlp.fc1, self.mlp.fc2 = torch.nn.Linear(dim, 4 * dim), torch.nn.Linear(4 * dim, dim)
        none = torch.nn.Identity()
        self.ls1, self.ls2 = (Scale(dim), Scale(dim)) if scales else (none, none)
        with torch.no_grad():
            for p in (self.norm1, self.norm2):
                p.weight.add_(0.2 * torch.randn(dim))
                p.bias.add_(0.2 * torch.randn(dim))


def positions(frames, dev):
    yy, xx = torch.meshgrid(torch.arange(6), torch.arange(6), indexing="ij")
    grid = torch.stack((yy.flatten() + 1, xx.flatten() + 1), -1)
    return torch.cat((torch.zeros(SPECIAL, 2, dtype=torch.long), grid)).repeat(frames, 1).to(dev)


def normed(x, norm):
    weight, bias, eps = norm
    return torch.nn.functional.layer_norm(x, x.shape[-1:], weight.double(), bias.double(), eps)


def mlp_64(block, h):
    y = normed(h, block.norm2)
    (w1, b1), (w2, b2) = ((w.double(), b.double()) for w, b in (block.fc1, block.fc2))
    z = y @ w1.t() + b1
    wide = z * torch.special.ndtr(z)
    out = wide @ w2.t() + b2
    return out if block.ls2 is None else out * block.ls2.double()


@pytest.mark.parametrize("dtype,stream", [(BF, BF), (BF, F32), (FP, FP), (FP, F32)])
@pytest.mark.parametrize("heads,frames,scales", [(2, 3, True), (4, 7, False)])
def test_block(cuda, dtype, stream, heads, frames, scales):
    torch.manual_seed(heads)
    block = GlobalBlock.from_module(Module(heads, scales).to(cuda), tokens_per_frame=TPF,
                                    dtype=dtype, mode="topk", topk=2, dense_heads=(0,))
    x = torch.randn(frames * TPF, heads * 64, device=cuda).to(stream)
    pos = positions(frames, cuda)
    out = block(x, pos, pos_count=7)
    assert out.shape == x.shape and out.dtype == stream
    assert torch.equal(block(x[None], pos)[0], out)
    # from the block's own attention on
    with torch.no_grad():
        a = block.attention(x, pos, 7)
    w, b = block.proj
    p = a.transpose(0, 1).flatten(1).double() @ w.double().t() + b.double()
    p = p if block.ls1 is None else p * block.ls1.double()
    h = x.double() + p
    m = mlp_64(block, h)
    want, u = h + m, U[dtype]
    room = 2 * u * p.norm() + 6 * u * m.norm() + 2 * U[stream] * want.norm()
    assert float((out.double() - want).norm()) <= float(room)
    # the attention half by hand
    y, _ = vggt_sparse.residual_norm(x, None, *block.norm1[:2], eps=block.norm1[2], dtype=dtype)
    layer = SparseGlobalLayer(heads, mode="topk", topk=2, dense_heads=(0,))
    qkv = vggt_sparse.project_qkv(y, *block.qkv, heads=heads, tokens_per_frame=TPF,
                                  q_norm=block.q_norm, k_norm=block.k_norm, pos=pos)
    assert torch.equal(layer.forward_projected(qkv), a)
    assert float((y.double() - normed(x.double(), block.norm1)).abs().max()) <= 8 * u


def test_mlp_half_trains(cuda):
    """The differentiable half of the block against the derivative of its 64-bit form."""
    torch.manual_seed(5)
    block = GlobalBlock.from_module(Module(2).to(cuda), tokens_per_frame=TPF, dtype=FP)
    x = torch.randn(3 * TPF, 128, device=cuda).requires_grad_()
    leaves = [x, *block.norm2[:2], *block.fc1, *block.fc2, block.ls2]
    for t in leaves:
        t.requires_grad_()
    dy = torch.randn_like(x)
    grads = torch.autograd.grad(block.mlp(x), leaves, dy)
    wide = [t.detach().double().requires_grad_() for t in leaves]
    block.norm2 = wide[1], wide[2], block.norm2[2]
    block.fc1, block.fc2, block.ls2 = (wide[3], wide[4]), (wide[5], wide[6]), wide[7]
    want = torch.autograd.grad(wide[0] + mlp_64(block, wide[0]), wide, dy.double())
    for t, got, ref in zip(leaves, grads, want):
        assert got.dtype == t.dtype and got.shape == t.shape
        # dy in the products' type, dz twice, y, z and the widened tokens: at most eight roundings
        # on any way from dy to a gradient
        assert float((got.double() - ref).norm()) <= 8 * U[FP] * float(ref.norm()) + 1e-4


def test_block_replays_from_a_graph(cuda):
    torch.manual_seed(6)
    block = GlobalBlock.from_module(Module(4).to(cuda), tokens_per_frame=TPF, mode="topk", topk=3)
    x, pos = torch.randn(5 * TPF, 256, device=cuda), positions(5, cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        block(x, pos, 7)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = block(x, pos, 7)
    x.copy_(torch.randn_like(x))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, block(x, pos, 7))


def test_block_refuses():
    parts = Module(2)
    with pytest.raises(ValueError, match="either layer or"):
        GlobalBlock.from_module(parts, tokens_per_frame=TPF, layer=SparseGlobalLayer(2), topk=2)
    with pytest.raises(ValueError, match="heads"):
        GlobalBlock.from_module(parts, tokens_per_frame=TPF, layer=SparseGlobalLayer(4))
