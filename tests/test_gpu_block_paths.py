"""Every kernel that the block's operators can choose, at sizes that end inside its tiles, and a
whole block against independent code.

Which kernels the sizes reach is read from the launches themselves.  Bounds as in
test_gpu_block_ops.py and test_gpu_block_edges.py.
"""
import itertools
import math
import re

import pytest
import torch

import vggt_sparse
from test_gpu_block_edges import SPECIAL, TPF, Call, Part, positions
from test_gpu_block_ops import BF, F32, FP, SMALL, U, Linear, Norm, make, near

pytestmark = pytest.mark.gpu

# rows, inner, outer: in each list the forward product and those of dx and dW, taken together, have
# every tile shape, whole and split
EVEN = [(66, 16, 16), (129, 136, 4944), (140, 4912, 200), (265, 5144, 984), (389, 4344, 784),
        (417, 632, 4992), (523, 680, 4632), (1039, 1136, 136), (1217, 16, 16), (1812, 1880, 1184),
        (4463, 776, 440), (4827, 616, 584)]
ODD = [(17, 17, 21), (129, 5005, 151), (131, 201, 4809), (391, 709, 4285), (439, 4471, 731),
       (527, 4719, 695), (601, 627, 4835), (1091, 133, 1193), (1275, 17, 17), (1645, 1707, 1409),
       (4413, 727, 475), (4999, 965, 311)]
# pairs of CTAs with 256 x 256 tiles, split: dW, dx, forward
LARGE = [(5231, 2776, 1744), (1781, 2776, 5288), (3087, 5616, 1464)]
LARGE_ODD = [(12963, 137, 2199), (1479, 3147, 5319), (1813, 8247, 1249)]


def check_call(c):
    status = torch.zeros(1, dtype=torch.int32, device=c.x.device)
    with torch.no_grad():
        c.check(c.call(status=status))
    leaves = [t.requires_grad_() for t in c.leaves()]
    y = c.call(status=status)
    c.check(y.detach())
    grads = torch.autograd.grad(y, leaves, c.dy, retain_graph=True)
    assert int(status) == 0
    named = dict(zip([n for n, t in zip("xwbgr", (c.x, c.w, c.b, c.g, c.r)) if t is not None], grads))
    c.check_grads(named["x"], named["w"], named.get("b"), named.get("g"))
    for t, d in zip(leaves, grads):
        one, = torch.autograd.grad(y, t, c.dy, retain_graph=True)
        assert torch.equal(one, d)


@pytest.mark.parametrize("rows,inner,outer", EVEN + ODD)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_linear_kernels(cuda, rows, inner, outer, dtype):
    check_call(Call(cuda, rows, inner, outer, dtype, gate=True, residual=dtype))
    check_call(Call(cuda, rows, inner, outer, dtype, act="gelu", gate=True, residual=F32, seed=1))
    check_call(Call(cuda, rows, inner, outer, dtype, act="silu", bias=False, seed=2))


@pytest.mark.parametrize("rows,inner,outer", LARGE + LARGE_ODD)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_linear_kernels_of_large_products(cuda, rows, inner, outer, dtype):
    check_call(Call(cuda, rows, inner, outer, dtype, gate=True, residual=dtype))
    check_call(Call(cuda, rows, inner, outer, dtype, act="gelu", residual=F32, seed=1))


@pytest.mark.parametrize("rows,heads,dim,outer", [(1820, 15, 128, 1184), (1039, 18, 64, 136),
                                                  (523, 10, 64, 4632), (140, 77, 64, 200),
                                                  (4830, 10, 64, 584), (1650, 24, 71, 1409)])
def test_linear_kernels_on_head_major_tensors(cuda, rows, heads, dim, outer):
    check_call(Call(cuda, rows, heads * dim, outer, BF, gate=True, residual=F32, heads=heads))


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("rows,inner,outer", [(1, 1032, 2056), (9, 4104, 1000), (20, 520, 4104),
                                              (31, 1032, 4097), (17, 264, 4000), (64, 2056, 2040)])
def test_linear_kernels_of_few_rows(cuda, rows, inner, outer, dtype):
    for act, residual in (("gelu", None), (None, F32), ("relu", dtype)):
        c = Linear(cuda, rows, inner, outer, dtype, act=act, gate=True, residual=residual)
        c.check(c.call())


def launched(run):
    """Template arguments of the kernels that `run` launches, by the kernels' names."""
    from torch.profiler import ProfilerActivity, profile
    torch.cuda.synchronize()
    with profile(activities=[ProfilerActivity.CPU, ProfilerActivity.CUDA]) as p:
        run()
        torch.cuda.synchronize()
    names = {e.name for e in p.events() if "CUDA" in str(e.device_type)}
    if not names:
        pytest.skip("launches cannot be recorded here (another profiler holds the device)")
    found = {}
    for name in names:
        m = re.search(r"(\w+)<([^<>]*)>\(", name)
        if m is None:
            continue
        values = [re.sub(r"^\(\w+\)", "", v.strip()) for v in m.group(2).split(",")]
        values = [{"true": 1, "false": 0}.get(v, int(v) if v.isdigit() else v) for v in values]
        found.setdefault(m.group(1), set()).add(tuple(values))
    return found


@pytest.mark.parametrize("sizes", [EVEN + LARGE, ODD + LARGE_ODD])
def test_linear_sizes_reach_every_product(cuda, sizes):
    def run():
        for rows, inner, outer in sizes:
            x = torch.zeros(rows, inner, dtype=BF, device=cuda, requires_grad=True)
            w = torch.zeros(outer, inner, dtype=BF, device=cuda, requires_grad=True)
            y = vggt_sparse.linear(x, w)
            torch.autograd.grad(y, (x, w), y.detach())
    got = launched(run)
    # CTAs, their columns, whether A's and B's rows lie along the reduced index, split
    majors = [(0, 0), (0, 1), (1, 1)]  # forward, dx, dW
    want = {("__nv_bfloat16", cta, cols) + major + (split,)
            for cta, cols, major, split in itertools.product((1, 2), (64, 128), majors, (0, 1))}
    assert got["product_kernel"] == want
    assert "finish_kernel" in got and "finish_weight_kernel" in got


def test_linear_sizes_reach_every_kernel_of_few_rows(cuda):
    def run():
        for rows, outer in ((1, 64), (9, 2048), (20, 64), (20, 4104), (40, 1024)):
            x = torch.zeros(rows, 64, dtype=BF, device=cuda)
            vggt_sparse.linear(x, torch.zeros(outer, 64, dtype=BF, device=cuda))
    want = {("__nv_bfloat16", blocks, cols) for blocks, cols in ((1, 8), (1, 16), (2, 8), (2, 32),
                                                               (4, 8))}
    assert launched(run)["rows_kernel"] == want


@pytest.mark.parametrize("rows,inner,outer", [(12, 128, 136), (200, 128, 136), (500, 4096, 512),
                                              (1812, 1880, 1184), (129, 5005, 151)])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_linear_keeps_what_is_not_finite_in_its_column(cuda, rows, inner, outer, act):
    """Rows of the weight that are not finite, and gates and biases, stay in their columns."""
    c = Linear(cuda, rows, inner, outer, act=act, gate=True, residual=BF)
    d = Linear(cuda, rows, inner, outer, act=act, gate=True, residual=BF)
    d.w[5, 3], d.w[9, inner - 1], d.b[64], d.g[70] = math.nan, math.inf, -math.inf, math.nan
    keep = torch.ones(outer, dtype=torch.bool)
    keep[[5, 9, 64, 70]] = False
    outs = []
    for t in (c, d):
        leaves = [u.requires_grad_() for u in (t.w, t.b, t.g)]
        y = t.call()
        outs.append((y.detach(), *torch.autograd.grad(y, leaves, t.dy)))
    (y, dw, db, dg), (y2, dw2, db2, dg2) = outs
    assert torch.equal(y[:, keep], y2[:, keep]) and bool(y2[:, 5].isnan().all())
    assert torch.equal(dw[keep], dw2[keep])
    assert torch.equal(db[keep], db2[keep]) and torch.equal(dg[keep], dg2[keep])


# ---- residual_norm: rows copied ahead -----------------------------------------------------------
# width, rows: a little more than two rows to each of the most slots there are, rows of every number
# of warps that end inside their last chunk
AHEAD = [(136, 4773), (264, 4773), (1000, 2405), (1032, 1813), (2056, 1813), (4104, 337), (8200, 333)]
TYPES = [(BF, BF), (FP, FP), (BF, F32), (FP, F32), (F32, F32)]
NORMS = [("layer", None, True), ("layer", None, False), ("layer", "layer", True), ("rms", "rms", True)]


@pytest.mark.parametrize("width,rows", AHEAD)
@pytest.mark.parametrize("dtype,stream", TYPES)
@pytest.mark.parametrize("norm,post,branch", NORMS)
def test_residual_norm_of_many_rows(cuda, width, rows, dtype, stream, norm, post, branch):
    Norm(cuda, rows, width, dtype, stream, norm, post, branch=branch, seed=width).check_all()


@pytest.mark.parametrize("width,rows,groups", [(264, 4773, 43), (2056, 1815, 3), (2056, 1815, 1815),
                                               (4104, 925, 37), (8200, 333, 9)])
@pytest.mark.parametrize("dtype,stream", [(BF, BF), (FP, F32), (F32, F32)])
@pytest.mark.parametrize("norm,post", [("layer", "layer"), ("rms", "rms"), ("layer", None)])
def test_residual_norm_gates_of_many_rows(cuda, width, rows, groups, dtype, stream, norm, post):
    Norm(cuda, rows, width, dtype, stream, norm, post, groups=groups).check_all()


@pytest.mark.parametrize("dtype,stream", TYPES)
def test_residual_norm_rows_reach_every_kernel(cuda, dtype, stream):
    """Of the kernels that copy rows ahead, each whose rows fit shared memory (224 KB)."""
    name = {BF: "__nv_bfloat16", FP: "__half", F32: "float"}
    units = stream.itemsize // 2 + dtype.itemsize // 2  # of 16 bytes, for 8 elements

    def run():
        for (width, rows), (norm, post, branch) in itertools.product(AHEAD, NORMS):
            c = Norm(cuda, rows, width, dtype, stream, norm, post, branch=branch)
            leaves = [t.requires_grad_() for t in c.leaves().values()]
            torch.autograd.grad(c.call()[0], leaves, c.dy)
    got = launched(run)
    pair = name[stream], name[dtype]
    shapes = [(1, 1), (1, 2), (2, 2), (4, 2), (8, 2), (16, 2), (16, 4)]  # warps of a row, chunks
    fits = lambda threads, n: threads * 2 * n * 16 <= 224 * 1024  # noqa: E731
    want = {pair + s + (0,) for s in shapes if fits(768 if s[0] in (4, 8) else 512, s[1] * units)}
    assert {k for k in got["forward_kernel"] if k[-1] == 0} == want
    halves = [(1, 1), (2, 1), (4, 1), (8, 1), (16, 1), (16, 2), (16, 4)]
    want = {pair + s + (post, 0) for post, list_ in ((0, shapes), (1, shapes), (2, halves))
            for s in list_ if fits(512, s[1] * 2 * units)}
    assert {k for k in got["backward_kernel"] if k[-1] == 0} == want


@pytest.mark.parametrize("dtype,stream", [(BF, F32), (FP, FP), (F32, F32)])
@pytest.mark.parametrize("rows,width", [(3001, 1024), (3001, 1000), (925, 4104)])
def test_residual_norm_in_place_of_many_rows(cuda, dtype, stream, rows, width):
    c = Norm(cuda, rows, width, dtype, stream, "layer", "rms")
    y, h = c.call()
    x, f = c.x.clone(), c.f.clone()
    for out, stream_out in ((f, x), (None, x), (f, None)) + (((x, f), (x, None)) if dtype == stream else ()):
        c.x.copy_(x), c.f.copy_(f)  # the arguments anew
        at = {id(x): c.x, id(f): c.f, id(None): None}
        y2, h2 = c.call(out=at[id(out)], stream_out=at[id(stream_out)])
        assert torch.equal(y, y2) and torch.equal(h, h2)


# ---- a whole block ------------------------------------------------------------------------------
def rotated(v, pos, base):
    """RoPE-2D of [heads, tokens, 64], from the formula."""
    freq = base ** (-torch.arange(16, device=v.device, dtype=torch.float64) / 16)
    halves = []
    for half, p in ((v[..., :32], pos[:, 0]), (v[..., 32:], pos[:, 1])):
        angle = p.double()[:, None] * freq
        a, b = half[..., :16], half[..., 16:]
        halves += [a * angle.cos() - b * angle.sin(), b * angle.cos() + a * angle.sin()]
    return torch.cat(halves, -1)


@pytest.mark.parametrize("dtype,stream", [(FP, F32), (BF, F32), (BF, BF)])
@pytest.mark.parametrize("heads,frames,rope", [(2, 3, 100.0), (3, 12, 100.0), (2, 7, None)])
def test_whole_block_with_dense_heads(cuda, dtype, stream, heads, frames, rope):
    """All heads dense, against the block's formula in 64 bits from x on.

    Bounds in norms, u the roundoff of the block's type.  q and k carry three roundings each (the
    normed tokens, the projection, their norm's result), independent of one another and, as the tokens
    are random, from token to token.  A logit, the sum of 64 products over 8, is off by their root of
    squares, below 6 u (sum (q k)^2)^(1/2) / 8 <= 6 u |q| |k| / 64 = 6 u (|q| = |k| = 8, both being
    normed); its softmax's result by that for each key, p_j |v_j - a| of it, as a root of squares
    again.  v (twice: from the tokens, and its own), the probabilities and the result are rounded too.
    All of it is doubled for the norm's chance to be above its expectation.  The projection
    and the MLP half carry it on with gains that the norms of their matrices bound (1.13: gelu's slope;
    the norm: its weight over the least deviation of a row).  From there on as in test_gpu_block.py.
    """
    torch.manual_seed(heads + frames)
    dim, u = heads * 64, U[dtype]
    part = Part(heads).to(cuda)
    block = vggt_sparse.GlobalBlock.from_module(part, tokens_per_frame=TPF, dtype=dtype,
                                                dense_heads=tuple(range(heads)), rope_base=rope)
    x, pos = torch.randn(frames * TPF, dim, device=cuda).to(stream), positions(frames, cuda)
    out = block(x, pos, 7).double()
    d = lambda t: t.detach().double()  # noqa: E731
    ln = lambda t, m: torch.nn.functional.layer_norm(t, t.shape[-1:], d(m.weight), d(m.bias), m.eps)  # noqa: E731,E501
    weights = {n: (d(w), d(b)) for n, (w, b) in (("qkv", block.qkv), ("proj", block.proj),
                                                ("fc1", block.fc1), ("fc2", block.fc2))}
    apply = lambda t, n: t @ weights[n][0].t() + weights[n][1]  # noqa: E731
    q, k, v = apply(ln(d(x), part.norm1), "qkv").view(-1, 3, heads, 64).permute(1, 2, 0, 3)
    q, k = ln(q, part.attn.q_norm), ln(k, part.attn.k_norm)
    if rope is not None:
        q, k = rotated(q, pos, rope), rotated(k, pos, rope)
    prob = torch.softmax(q @ k.transpose(1, 2) / 8, -1)
    a = prob @ v
    ls1, ls2 = d(part.ls1.gamma), d(part.ls2.gamma)
    p = ls1 * apply(a.transpose(0, 1).flatten(1), "proj")
    h = d(x) + p
    z = apply(ln(h, part.norm2), "fc1")
    m = ls2 * apply(z * torch.special.ndtr(z), "fc2")
    far = (v * v).sum(-1)[:, None] - 2 * a @ v.transpose(1, 2) + (a * a).sum(-1)[:, :, None]
    da = 2 * u * (6 * float((prob * prob * far).sum().sqrt())
                  + 3 * float((prob * prob @ (v * v)).sum().sqrt()) + float(a.norm()))
    gain = lambda t: float(torch.linalg.matrix_norm(t, 2))  # noqa: E731
    dh = da * gain(ls1[:, None] * weights["proj"][0])
    on = (float(d(part.norm2.weight).abs().max()) / float(h.std(-1, unbiased=False).min())
          * gain(weights["fc1"][0]) * 1.13 * gain(ls2[:, None] * weights["fc2"][0]))
    room = (dh * (1 + on) + 2 * u * float(p.norm()) + 6 * u * float(m.norm())
            + 2 * U[stream] * float((h + m).norm()))
    assert float((out - h - m).norm()) <= room
    # the attention by itself, which the rest hides in part
    got = block.attention(x, pos, 7).double()
    assert float((got - a).norm()) <= da
