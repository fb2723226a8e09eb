"""The block's dense operators on the GPU against plain 64-bit code.

Bounds (u: unit roundoff of an output's type, 2^-8 bf16, 2^-11 fp16, 2^-24 fp32;
v: that of the products' type), elementwise, from the magnitudes of what is added:

linear.  z is summed in fp32 over `inner` products, 16 of them an instruction, with
a truncation of at most 2^-23 of the running magnitude each: ez = 2^-23 (inner / 16 +
8) (|x| |W| + |b|).  An activation is good to 1e-5 |a| and has a slope of at most
1.13 (gelu; the others 1.1), so y: u |y| + |g| (1.13 ez + 1e-5 |a|) + 2^-22 (|r| +
|g a|) + 2^-25 (half a step of fp16's subnormal numbers).
Gradients.  z is kept in v (with a gate better, in fp32): dz is off by d = |dy g| (v |z| + ez + 1e-5) (the second
derivatives stay below 1), for relu by |dy g| where |z| <= ez; then rounded: v |dz|.
A product of dz adds 2^-23 (n / 16 + 8) of its magnitudes.  Without an activation the
gate goes to dy or to W: one rounding v of a factor, and dy in fp32 is rounded too.
dgate sums dy a: |dy| (1.13 (v |z| + ez) + 1e-5 |a|), or without an activation
<W, dy^T x>: v |dy| |x| |W|.

residual_norm.  Everything is fp32: a mean, a variance and what is formed from them
are off by 2^-17 of the magnitudes that are added at an element (a few 2^-24 for each
of the sums, times the condition of a row, |mean| / deviation, at most 8 here).
"""
import math

import pytest
import torch

import vggt_sparse
from vggt_sparse import _lib

pytestmark = pytest.mark.gpu

BF, FP, F32 = torch.bfloat16, torch.float16, torch.float32
U = {BF: 2.0 ** -8, FP: 2.0 ** -11, F32: 2.0 ** -24}
SMALL = 2.0 ** -25


def make(gen, dev, *shape, dtype=BF, scale=1.0, mean=0.0):
    return (torch.randn(*shape, generator=gen) * scale + mean).to(dtype).to(dev)


def near(got, want, bound, name=""):
    assert got.shape == want.shape, (name, got.shape, want.shape)
    err = (got.double() - want).abs()
    worst = (err - bound).max()
    assert bool((err <= bound).all()), (name, float(worst), float(err.max()))


def activation(z, name):
    if name == "gelu":
        return z * torch.special.ndtr(z)
    if name == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if name == "silu":
        return z * torch.sigmoid(z)
    if name == "relu":
        return z.clamp(min=0)
    return z


class Linear:
    """A call's tensors, its definition in 64 bits, and the bounds above."""

    def __init__(self, dev, rows, inner, outer, dtype=BF, act=None, bias=True, gate=False,
                 residual=None, heads=0, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.dtype, self.act, self.heads = dtype, act, heads
        self.rows, self.inner, self.outer = rows, inner, outer
        self.x = (make(g, dev, heads, rows, inner // heads, dtype=dtype) if heads
                  else make(g, dev, rows, inner, dtype=dtype))
        self.w = make(g, dev, outer, inner, dtype=dtype, scale=inner ** -0.5)
        self.b = make(g, dev, outer, dtype=dtype, scale=0.3) if bias else None
        self.g = make(g, dev, outer, dtype=dtype, scale=0.5) if gate else None
        self.r = make(g, dev, rows, outer, dtype=residual, scale=2.0) if residual else None
        self.dy = make(g, dev, rows, outer, dtype=residual or dtype)

    def call(self, **kw):
        return vggt_sparse.linear(self.x, self.w, self.b, activation=self.act, gate=self.g,
                                  residual=self.r, head_major=self.heads > 0, **kw)

    def leaves(self):
        return [t for t in (self.x, self.w, self.b, self.g, self.r) if t is not None]

    def define(self):
        wide = [None if t is None else t.detach().double() for t in (self.x, self.w, self.b, self.g,
                                                                    self.r)]
        x = wide[0].transpose(0, 1).flatten(1) if self.heads else wide[0].flatten(0, -2)
        w, b, g, r = wide[1:]
        r = None if r is None else r.flatten(0, -2)
        b = torch.zeros(1, device=x.device, dtype=x.dtype) if b is None else b
        gg = torch.ones(1, device=x.device, dtype=x.dtype) if g is None else g
        self.xd, self.wd = x, w
        z = x @ w.t() + b
        self.z, self.ez = z, 2.0 ** -23 * (self.inner / 16 + 8) * (x.abs() @ w.abs().t() + b.abs())
        a = activation(z, self.act)
        self.a = a
        y = gg * a + (0 if r is None else r)
        u = U[self.r.dtype if self.r is not None else self.dtype]
        bound = (u * y.abs() + gg.abs() * (1.13 * self.ez + 1e-5 * a.abs())
                 + 2.0 ** -22 * ((0 if r is None else r.abs()) + (gg * a).abs()) + SMALL)
        return y, bound

    def check(self, got):
        y, bound = self.define()
        near(got.flatten(0, -2), y, bound, "y")

    def check_grads(self, dx, dw, db, dg):
        self.define()
        v = U[self.dtype]
        dy = self.dy.double().flatten(0, -2)
        n_rows, one = dy.shape[0], torch.ones(1, device=dy.device, dtype=dy.dtype)
        g = one if self.g is None else self.g.double()
        zl = self.z.detach().clone().requires_grad_()
        slope, = torch.autograd.grad(activation(zl, self.act).sum(), zl)
        dz = dy * g * slope
        if self.act is None:
            off = v * dz.abs()      # the gate's product, rounded
            off_w = v * dz.abs()    # dy in fp32, rounded
            off_b = 2.0 ** -22 * dz.abs()
            off_g = (v * dy.abs() * (self.xd.abs() @ self.wd.abs().t())
                     + 2.0 ** -20 * dy.abs() * self.a.abs())
        else:
            off_b = (dy * g).abs() * ((self.z.abs() <= self.ez).double() if self.act == "relu"
                                      else v * self.z.abs() + self.ez + 1e-5)
            off = off_w = off_b + v * dz.abs()
            off_g = dy.abs() * (1.13 * (v * self.z.abs() + self.ez) + 1e-5 * self.a.abs())
        add = lambda n: 2.0 ** -23 * (n / 16 + 8)  # noqa: E731
        if dx is not None:
            want = dz @ self.wd
            if self.heads:
                dx = dx.transpose(0, 1).flatten(1)
            mag = dz.abs() @ self.wd.abs()
            near(dx.flatten(0, -2), want,
                 v * want.abs() + 1.01 * (off @ self.wd.abs()) + add(self.outer) * mag + SMALL, "dx")
        if dw is not None:
            want = dz.t() @ self.xd
            mag = dz.abs().t() @ self.xd.abs()
            near(dw, want,
                 v * want.abs() + 1.01 * (off_w.t() @ self.xd.abs()) + add(n_rows) * mag + SMALL,
                 "dw")
        if db is not None:
            want = dz.sum(0)
            near(db, want, v * want.abs() + 1.01 * off_b.sum(0)
                 + 2.0 ** -20 * dz.abs().sum(0) + SMALL, "db")
        if dg is not None:
            want = (dy * self.a).sum(0)
            near(dg, want, v * want.abs() + 1.01 * off_g.sum(0)
                 + (add(n_rows) + add(self.inner)) * (dy.abs().t() @ (self.xd.abs() @ self.wd.abs().t())
                                                      ).diagonal() + SMALL, "dgate")


SHAPES = [(1, 8, 1), (1, 64, 64), (1, 1024, 4096), (2, 1000, 72), (7, 65, 63), (16, 4096, 136),
          (17, 72, 517), (33, 200, 264), (64, 1024, 1024), (65, 512, 2048), (127, 1, 130),
          (128, 128, 128), (129, 264, 257), (300, 1001, 200), (500, 4096, 512), (1374, 1024, 1024),
          (2500, 320, 1300)]


@pytest.mark.parametrize("rows,inner,outer", SHAPES)
@pytest.mark.parametrize("dtype", [BF, FP])
def test_linear_shapes(cuda, rows, inner, outer, dtype):
    c = Linear(cuda, rows, inner, outer, dtype)
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    c.check(c.call(status=status))
    assert int(status) == 0
    c = Linear(cuda, rows, inner, outer, dtype, act="gelu", gate=True, residual=dtype, seed=1)
    c.check(c.call())
    c = Linear(cuda, rows, inner, outer, dtype, bias=False, gate=True, residual=F32, seed=2)
    got = c.call()
    assert got.dtype == F32
    c.check(got)


@pytest.mark.parametrize("act", ["gelu", "gelu_tanh", "silu", "relu", None])
@pytest.mark.parametrize("rows", [3, 40, 200])
@pytest.mark.parametrize("gate,residual", [(False, None), (True, FP), (True, F32)])
def test_linear_activations(cuda, act, rows, gate, residual):
    c = Linear(cuda, rows, 256, 192, FP, act=act, gate=gate, residual=residual, seed=3)
    c.x *= 4  # arguments well into both tails
    c.check(c.call())


@pytest.mark.parametrize("heads,dim", [(16, 64), (4, 128), (1, 64), (3, 40), (2, 65)])
@pytest.mark.parametrize("rows", [1, 20, 333])
def test_linear_reads_head_major_tensors(cuda, heads, dim, rows):
    c = Linear(cuda, rows, heads * dim, 200, heads=heads, gate=True, residual=BF)
    c.check(c.call())
    # heads between the rows, as the paged attention leaves them
    c.x = c.x.transpose(0, 1).contiguous().transpose(0, 1)
    c.check(c.call())


@pytest.mark.parametrize("rows", [5, 150])
def test_linear_layouts(cuda, rows):
    """Strided, misaligned, expanded and batched tensors."""
    g = torch.Generator().manual_seed(5)
    wide = make(g, cuda, rows, 400)
    c = Linear(cuda, rows, 128, 96, residual=BF)
    for x in (wide[:, 8:136], wide[:, 3:131], wide[:1, :128].expand(rows, 128),
              wide[:, :256:2], make(g, cuda, 128, rows).t()):
        c.x = x
        c.check(c.call())
    c.w = make(g, cuda, 128, 96, scale=0.1).t()
    c.check(c.call())
    c.w = make(g, cuda, 96, 300, scale=0.1)[:, 8:136]
    c.check(c.call())
    c.r = wide[:, 7:103]
    c.check(c.call())
    c.r = wide[:1, :96].expand(rows, 96)
    c.check(c.call())
    c.r = make(g, cuda, 96, rows).t()
    c.check(c.call())
    c.b = make(g, cuda, 192)[::2]
    c.check(c.call())
    c = Linear(cuda, 24, 64, 40, residual=F32)
    c.x, c.r = c.x.view(2, 3, 4, 64), c.r.view(2, 3, 4, 40)
    got = c.call()
    assert got.shape == (2, 3, 4, 40)
    c.check(got)


def test_linear_out_may_be_the_residual(cuda):
    for rows in (9, 400):
        c = Linear(cuda, rows, 128, 256, gate=True, residual=F32)
        want = c.call()
        r = c.r.clone()
        assert vggt_sparse.linear(c.x, c.w, c.b, gate=c.g, residual=r, out=r) is r
        assert torch.equal(r, want)


def test_linear_without_rows(cuda):
    x = torch.zeros(0, 64, dtype=BF, device=cuda, requires_grad=True)
    w = torch.ones(16, 64, dtype=BF, device=cuda, requires_grad=True)
    b = torch.ones(16, dtype=BF, device=cuda, requires_grad=True)
    g = torch.ones(16, dtype=BF, device=cuda, requires_grad=True)
    y = vggt_sparse.linear(x, w, b, activation="gelu", gate=g)
    assert y.shape == (0, 16)
    for t in torch.autograd.grad(y, (x, w, b, g), torch.zeros_like(y)):
        assert bool((t == 0).all())


def test_linear_keeps_what_is_not_finite_in_its_row(cuda):
    for rows in (12, 200):
        c = Linear(cuda, rows, 128, 136, FP, act="gelu")
        want = c.call()
        c.x[3, 5], c.x[7] = math.nan, 6e4
        c.x[7, ::2] = -6e4
        got = c.call()
        assert bool(got[3].isnan().all())
        keep = torch.ones(rows, dtype=torch.bool)
        keep[3] = keep[7] = False
        assert torch.equal(got[keep], want[keep])
        # z is infinite in fp16; the activation is formed before any rounding
        b = torch.full((136,), 6e4, dtype=FP, device=cuda)
        for act in ("gelu", "gelu_tanh", "silu", "relu"):
            x = c.x.clone().fill_(0).requires_grad_()
            y = vggt_sparse.linear(x, c.w, b, activation=act,
                                   gate=torch.full_like(b, 2.0 ** -4))
            assert bool((y == 3750).all())
            y = vggt_sparse.linear(x, c.w, -b, activation=act)
            assert bool((y == 0).all())
            d, = torch.autograd.grad(y, x, torch.ones_like(y))
            assert bool((d == 0).all())


GRADS = [(1, 64, 64, 0), (5, 8, 1, 0), (43, 1001, 517, 0), (64, 256, 136, 0), (129, 72, 257, 0),
         (200, 1024, 300, 16), (300, 136, 1024, 0), (700, 512, 640, 4), (2000, 264, 136, 0)]


@pytest.mark.parametrize("rows,inner,outer,heads", GRADS)
@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("act,gate,residual", [(None, False, None), (None, True, F32),
                                               (None, True, "same"), ("gelu", False, None),
                                               ("silu", True, "same"), ("gelu_tanh", True, F32),
                                               ("relu", True, None)])
def test_linear_gradients(cuda, rows, inner, outer, heads, dtype, act, gate, residual):
    residual = dtype if residual == "same" else residual
    c = Linear(cuda, rows, inner, outer, dtype, act=act, gate=gate, residual=residual, heads=heads,
               seed=rows)
    leaves = [t.requires_grad_() for t in c.leaves()]
    y = c.call()
    c.check(y.detach())
    grads = torch.autograd.grad(y, leaves, c.dy, retain_graph=True)
    named = dict(zip([n for n, t in zip("xwbgr", (c.x, c.w, c.b, c.g, c.r)) if t is not None],
                     grads))
    c.check_grads(named["x"], named["w"], named["b"], named.get("g"))
    for t, d in zip(leaves, grads):
        assert d.shape == t.shape and d.dtype == t.dtype
    if residual:
        assert torch.equal(named["r"], c.dy)
    # the same again, and each gradient by itself
    again = torch.autograd.grad(y, leaves, c.dy, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(grads, again))
    for t, d in zip(leaves, grads):
        one, = torch.autograd.grad(y, t, c.dy, retain_graph=True)
        assert torch.equal(one, d)


def test_linear_gradient_layouts(cuda):
    """A gradient that is expanded, strided or misaligned; a tensor used twice."""
    c = Linear(cuda, 150, 128, 96, FP, gate=True)
    leaves = [t.requires_grad_() for t in c.leaves()]
    y = c.call()
    g = torch.Generator().manual_seed(6)
    for dy in (torch.ones(1, 1, dtype=FP, device=cuda).expand(150, 96),
               make(g, cuda, 96, 150, dtype=FP).t(), make(g, cuda, 150, 200, dtype=FP)[:, 3:99],
               make(g, cuda, 1, 96, dtype=FP).expand(150, 96)):
        c.dy = dy
        c.check_grads(*torch.autograd.grad(y, leaves, dy, retain_graph=True))
    x = make(g, cuda, 40, 64, dtype=FP).requires_grad_()
    w = make(g, cuda, 64, 64, dtype=FP, scale=0.1).requires_grad_()
    twice = vggt_sparse.linear(vggt_sparse.linear(x, w), w, residual=x)
    dx, dw = torch.autograd.grad(twice.float().sum(), (x, w))
    xd, wd = (t.detach().double().requires_grad_() for t in (x, w))
    ref = torch.autograd.grad((xd + xd @ wd.t() @ wd.t()).sum(), (xd, wd))
    for got, want in zip((dx, dw), ref):
        assert float((got.double() - want).norm() / want.norm()) < 4 * U[FP]


def test_linear_gradient_against_differences(cuda):
    """The kernel's gradient along a direction, against differences of the 64-bit definition."""
    for act in ("gelu", "gelu_tanh", "silu", None):
        c = Linear(cuda, 70, 96, 80, FP, act=act, gate=True, residual=F32)
        leaves = [t.requires_grad_() for t in c.leaves()]
        grads = torch.autograd.grad(c.call(), leaves, c.dy)
        g = torch.Generator().manual_seed(8)
        for i, (t, d) in enumerate(zip(leaves, grads)):
            way = torch.randn(t.shape, generator=g, dtype=torch.float64).to(cuda)

            def at(step):
                wide = [q.detach().double() for q in leaves]
                wide[i] = wide[i] + step * way
                x, w, b, gg, r = wide
                return ((r + gg * activation(x @ w.t() + b, act)) * c.dy.double()).sum()
            want = float((at(1e-4) - at(-1e-4)) / 2e-4)
            # every gradient element is off by few roundings, of independent signs or not
            room = 4 * U[FP] * float((d.double() * way).abs().sum()) + 1e-6
            assert abs(float((d.double() * way).sum()) - want) <= room


def test_linear_is_differentiable_once(cuda):
    c = Linear(cuda, 10, 64, 32)
    c.x.requires_grad_()
    d, = torch.autograd.grad(c.call(), c.x, c.dy, create_graph=True)
    assert not d.requires_grad or d.grad_fn is not None
    with pytest.raises(RuntimeError):
        torch.autograd.grad(d.sum(), c.x)


# ---- residual_norm ----------------------------------------------------------------------------
class Norm:
    def __init__(self, dev, rows, width, dtype=BF, stream=None, norm="layer", post=None, branch=True,
                 affine=True, groups=1, params=F32, seed=0):
        g = torch.Generator().manual_seed(seed)
        stream = stream or dtype
        self.norm, self.post, self.dtype, self.stream, self.groups = norm, post, dtype, stream, groups
        self.x = make(g, dev, rows, width, dtype=stream, scale=2.0, mean=1.0)
        self.f = make(g, dev, rows, width, dtype=dtype, mean=0.5) if branch else None
        self.g = None
        if branch and groups:
            shape = (width,) if groups == 1 else (groups, width)
            self.g = make(g, dev, *shape, dtype=params, scale=0.5)
        p = lambda mean: make(g, dev, width, dtype=params, scale=0.3, mean=mean)  # noqa: E731
        self.w, self.b = (p(1.0), p(0.0) if norm == "layer" else None) if affine else (None, None)
        self.pw, self.pb = (p(1.0), p(0.0) if post == "layer" else None) if affine and post else (
            None, None)
        self.dy = make(g, dev, rows, width, dtype=dtype)
        self.dh = make(g, dev, rows, width, dtype=stream)

    def call(self, **kw):
        return vggt_sparse.residual_norm(self.x, self.f, self.w, self.b, norm=self.norm, gate=self.g,
                                         post_norm=self.post, post_weight=self.pw, post_bias=self.pb,
                                         dtype=self.dtype, **kw)

    NAMES = ("x", "f", "g", "w", "b", "pw", "pb")

    def leaves(self):
        return {n: getattr(self, n) for n in self.NAMES if getattr(self, n) is not None}

    @staticmethod
    def normed(v, kind):
        if kind == "layer":
            v = v - v.mean(-1, keepdim=True)
        r = 1 / torch.sqrt((v * v).mean(-1, keepdim=True) + 1e-5)
        return v * r, r

    def check(self, y, h, grads=None, dy=None, dh=None):
        e = 2.0 ** -17
        d = {n: t.detach().double() for n, t in self.leaves().items()}
        x = d["x"]
        one, zero = torch.ones(1, device=x.device, dtype=x.dtype), torch.zeros(1, device=x.device)
        gate = d.get("g", one)
        if gate.dim() == 2:
            gate = gate.repeat_interleave(x.shape[0] // gate.shape[0], 0)
        hw, hmag = x, x.abs()
        if "f" in d:
            p, pmag = d["f"], d["f"].abs()
            if self.post:
                fhat, fr = self.normed(p, self.post)
                pw, pb = d.get("pw", one), d.get("pb", zero)
                pmag = (fhat.abs() + fr * (p.abs() + p.abs().mean(-1, keepdim=True))) * pw.abs() + pb.abs()
                p = fhat * pw + pb
            hw = x + gate * p
            hmag = x.abs() + gate.abs() * pmag
            near(h, hw, U[self.stream] * hw.abs() + e * hmag + SMALL, "h")
        hat, r = self.normed(hw, self.norm)
        w, b = d.get("w", one), d.get("b", zero)
        hatmag = hat.abs() + r * (hmag + hmag.mean(-1, keepdim=True)) * (1 + hat.abs())
        yw = hat * w + b
        near(y, yw, U[self.dtype] * yw.abs() + e * (hatmag * w.abs() + b.abs()) + SMALL, "y")
        if grads is None:
            return
        mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731

        def back(g, gmag, hat, hatmag, r, kind):
            out = g - hat * mean(g * hat)
            mag = gmag + hatmag * mean(gmag * hatmag)
            if kind == "layer":
                out, mag = out - mean(g), mag + mean(gmag)
            return out * r, mag * r
        dy = torch.zeros_like(x) if dy is None else dy.double()
        dh = torch.zeros_like(x) if dh is None else dh.double()
        t, tmag = back(dy * w, (dy * w).abs(), hat, hatmag, r, self.norm)
        total, mag = dh + t, dh.abs() + tmag
        want = {"x": (total, mag), "w": ((dy * hat).sum(0), (dy.abs() * hatmag).sum(0)),
                "b": (dy.sum(0), dy.abs().sum(0))}
        if "f" in d:
            runs = d["g"].shape[0] if "g" in d and d["g"].dim() == 2 else 1
            fold = lambda t: t.unflatten(0, (runs, -1)).sum(1)  # noqa: E731
            if "g" in d:
                shape = d["g"].shape
                want["g"] = (fold(total * p).view(shape), fold(mag * pmag).view(shape))
            dp, dpmag = total * gate, mag * gate.abs()
            if self.post:
                fm = fhat.abs() + fr * (d["f"].abs() + mean(d["f"].abs())) * (1 + fhat.abs())
                want["pw"] = ((dp * fhat).sum(0), (dpmag * fm).sum(0))
                want["pb"] = (dp.sum(0), dpmag.sum(0))
                want["f"] = back(dp * pw, dpmag * pw.abs(), fhat, fm, fr, self.post)
            else:
                want["f"] = (dp, dpmag)
        for n, got in grads.items():
            leaf = self.leaves()[n]
            assert got.shape == leaf.shape and got.dtype == leaf.dtype, n
            value, m = want[n]
            near(got, value, U[got.dtype] * value.abs() + e * m + SMALL, n)

    def check_all(self):
        with torch.no_grad():
            self.check(*self.call())
        leaves = {n: t.requires_grad_() for n, t in self.leaves().items()}
        y, h = self.call()
        self.check(y.detach(), h.detach())
        for dy, dh in ((self.dy, self.dh), (self.dy, None), (None, self.dh)):
            if self.f is None and dh is not None:
                continue  # h is x itself
            if dy is None:
                use = {n: t for n, t in leaves.items() if n not in ("w", "b")}
            else:
                use = leaves
            outs = [o for o, g in ((y, dy), (h, dh)) if g is not None]
            given = [g for g in (dy, dh) if g is not None]
            grads = torch.autograd.grad(outs, list(use.values()), given, retain_graph=True)
            self.check(y.detach(), h.detach(), dict(zip(use, grads)), dy, dh)
            again = torch.autograd.grad(outs, list(use.values()), given, retain_graph=True)
            assert all(torch.equal(a, b) for a, b in zip(grads, again))


WIDTHS = [1, 5, 8, 64, 65, 256, 264, 512, 1000, 1024, 1032, 2048, 4096, 4104, 8192, 8200, 16384]


@pytest.mark.parametrize("width", WIDTHS)
@pytest.mark.parametrize("rows", [1, 37])
@pytest.mark.parametrize("post", [None, "layer", "rms"])
def test_residual_norm_widths(cuda, width, rows, post):
    if width == 1 and post == "layer":
        pytest.skip("a layer norm of one element is zero over zero")
    norm = "rms" if width == 1 or post == "rms" else "layer"
    Norm(cuda, rows, width, norm=norm, post=post, seed=width).check_all()


@pytest.mark.parametrize("dtype,stream,params", [(BF, BF, BF), (FP, FP, FP), (FP, FP, F32),
                                                 (BF, F32, F32), (FP, F32, FP), (F32, F32, F32),
                                                 (F32, F32, BF)])
@pytest.mark.parametrize("norm,post,affine", [("layer", None, True), ("rms", "rms", True),
                                              ("layer", "layer", False), ("rms", "layer", True)])
def test_residual_norm_types(cuda, dtype, stream, params, norm, post, affine):
    Norm(cuda, 67, 200, dtype, stream, norm, post, affine=affine, params=params).check_all()
    Norm(cuda, 29, 203, dtype, stream, norm, post, affine=affine, params=params).check_all()


@pytest.mark.parametrize("rows,groups", [(12, 0), (12, 12), (12, 3), (3000, 2), (3000, 3000),
                                         (3003, 429), (700, 100), (9, 3)])
@pytest.mark.parametrize("width,post", [(64, None), (1024, "rms"), (2100, None)])
def test_residual_norm_gates(cuda, rows, groups, width, post):
    Norm(cuda, rows, width, BF, F32, groups=groups, post=post, norm="rms").check_all()


@pytest.mark.parametrize("norm", ["layer", "rms"])
def test_residual_norm_without_a_branch(cuda, norm):
    c = Norm(cuda, 50, 264, BF, F32, norm, branch=False)
    c.check_all()
    y, h = c.call()
    assert h is c.x
    c = Norm(cuda, 50, 264, norm=norm, branch=False, affine=False)
    c.check_all()
    # the gradient of the stream beside the norm is added by the graph
    x = c.x.detach().requires_grad_()
    y, h = vggt_sparse.residual_norm(x, norm=norm)
    both, = torch.autograd.grad((y, h * 1), x, (c.dy, c.dh))
    one, = torch.autograd.grad(vggt_sparse.residual_norm(x, norm=norm)[0], x, c.dy)
    assert torch.equal(both, one + c.dh)


def test_residual_norm_layouts(cuda):
    g = torch.Generator().manual_seed(3)
    wide = make(g, cuda, 40, 700)
    c = Norm(cuda, 40, 136)
    for t in (wide[:, 8:144], wide[:, 3:139], wide[:1, :136].expand(40, 136), wide[:, :272:2],
              make(g, cuda, 136, 40).t()):
        c.x = c.x.detach()
        c.f, c.dy, c.dh = t, t, t
        c.check(*c.call())
        c.check_all()
        c.f, c.x = c.x.detach(), t.detach()
        c.check_all()
    big = Norm(cuda, 24, 72, groups=6)
    y, h = big.call()
    big3 = vggt_sparse.residual_norm(big.x.view(2, 3, 4, 72), big.f.view(2, 3, 4, 72), big.w, big.b,
                                     gate=big.g)
    assert torch.equal(big3[0].flatten(0, 2), y) and torch.equal(big3[1].flatten(0, 2), h)
    big.w = make(g, cuda, 144, dtype=F32)[::2]
    big.g = make(g, cuda, 72, 6, dtype=F32).t()
    big.check_all()


def test_residual_norm_in_place(cuda):
    c = Norm(cuda, 300, 1024, BF, F32)
    y, h = c.call()
    stream, out = c.x.clone(), torch.empty_like(y)
    y2, h2 = vggt_sparse.residual_norm(stream, c.f, c.w, c.b, gate=c.g, out=out, stream_out=stream)
    assert h2 is stream and y2 is out
    assert torch.equal(y, y2) and torch.equal(h, h2)


def test_residual_norm_rows_far_from_zero_and_not_finite(cuda):
    """Means a thousand deviations from zero lose nothing but what the input has lost; a row
    that is not finite stays by itself."""
    g = torch.Generator().manual_seed(4)
    x = (torch.randn(20, 512, generator=g, dtype=torch.float64) + 1000).float().to(cuda)
    y, _ = vggt_sparse.residual_norm(x)
    want, _ = Norm.normed(x.double(), "layer")
    assert float((y.double() - want).abs().max()) <= 1000 * 2.0 ** -20 + 5 * 2.0 ** -22
    x = make(g, cuda, 20, 512)
    want, _ = vggt_sparse.residual_norm(x)
    x[3, 7], x[11, 0] = math.inf, math.nan
    got, _ = vggt_sparse.residual_norm(x)
    keep = torch.ones(20, dtype=torch.bool)
    keep[3] = keep[11] = False
    assert torch.equal(got[keep], want[keep]) and not bool(got[11].isfinite().any())
    z = torch.zeros(4, 64, dtype=BF, device=cuda, requires_grad=True)
    for norm in ("layer", "rms"):
        y, _ = vggt_sparse.residual_norm(z, norm=norm)
        assert bool((y == 0).all())
        d, = torch.autograd.grad(y, z, torch.ones_like(y))
        assert bool(d.isfinite().all())


def test_residual_norm_without_rows(cuda):
    for groups in (0, 1, 3):
        check_no_rows(Norm(cuda, 0, 64, groups=groups, post="layer"))


def check_no_rows(c):
    leaves = [t.requires_grad_() for t in c.leaves().values()]
    y, h = c.call()
    assert y.shape == h.shape == (0, 64)
    for d in torch.autograd.grad((y, h), leaves, (c.dy, c.dh)):
        assert bool((d == 0).all())


def test_residual_norm_gradient_against_differences(cuda):
    """Differences of the kernel itself, in fp32."""
    c = Norm(cuda, 30, 120, F32, F32, "layer", "rms", groups=3)
    leaves = {n: t.requires_grad_() for n, t in c.leaves().items()}
    grads = torch.autograd.grad(c.call(), list(leaves.values()), (c.dy, c.dh))
    g = torch.Generator().manual_seed(9)

    def value():
        with torch.no_grad():
            y, h = c.call()
        return float((y.double() * c.dy.double()).sum() + (h.double() * c.dh.double()).sum())
    for (n, t), d in zip(leaves.items(), grads):
        way = torch.randn(t.shape, generator=g).to(cuda)
        step = 2.0 ** -7
        with torch.no_grad():
            t += step * way
            up = value()
            t -= 2 * step * way
            down = value()
            t += step * way
        got, want = float((d.double() * way.double()).sum()), (up - down) / (2 * step)
        # the third derivative's share, step^2 / 6 of sums of this size, and the values' roundings
        size = float((d.double() * way.double()).abs().sum())
        assert abs(got - want) <= 4 * step ** 2 * size + 1e-2, n


# ---- together, and with the rest of a program ---------------------------------------------------
def test_operators_on_another_stream(cuda):
    c, n = Linear(cuda, 1374, 1024, 512, act="gelu", gate=True, residual=F32), Norm(cuda, 999, 512)
    leaves = [t.requires_grad_() for t in c.leaves()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        y = c.call()
        grads = torch.autograd.grad(y, leaves, c.dy)
        both = n.call()
    torch.cuda.current_stream().wait_stream(side)
    c.check(y.detach())
    c.check_grads(*grads[:4])
    n.check(*both)


def test_operators_captured_in_a_graph(cuda):
    """Forward and backward in one graph, replayed on new values, while another graph of the same
    sizes replays on a second stream (workspaces belong to a graph)."""
    def build(seed):
        c = Linear(cuda, 300, 512, 384, act="gelu", gate=True, seed=seed)
        n = Norm(cuda, 300, 384, seed=seed)
        leaves = [t.requires_grad_() for t in (c.x, c.w, c.b, c.g, n.x, n.g, n.w)]

        def step():
            y = c.call()
            out, h = vggt_sparse.residual_norm(n.x, y, n.w, n.b, gate=n.g)
            return [out, h, *torch.autograd.grad((out, h), leaves, (n.dy, n.dh))]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
        return c, step, graph, outs
    sets = [build(1), build(2)]
    streams = [torch.cuda.Stream() for _ in sets]
    for c, *_ in sets:
        with torch.no_grad():
            c.x += 0.5
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (_, _, graph, _) in zip(streams, sets):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for _, step, _, outs in sets:
        for a, b in zip(outs, step()):
            assert torch.equal(a, b)


def test_wait_timeout_is_reported_and_the_context_lives(cuda):
    c = Linear(cuda, 1374, 1024, 1024)
    want = c.call()
    status = torch.zeros(1, dtype=torch.int32, device=cuda)
    limit, test = _lib.set_wait_limit_ns(2_000_000), _lib.set_wait_selftest(True)
    try:
        c.call(status=status)
        torch.cuda.synchronize()
    finally:
        _lib.set_wait_selftest(test)
        _lib.set_wait_limit_ns(limit)
    assert int(status) == _lib.STATUS_TIMEOUT
    status.zero_()
    assert torch.equal(c.call(status=status), want) and int(status) == 0


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="two GPUs")
def test_operators_on_a_device_that_is_not_current(cuda):
    c = Linear(torch.device("cuda:1"), 200, 128, 64, gate=True)
    c.check(c.call())
    n = Norm(torch.device("cuda:1"), 50, 264)
    n.check_all()
    with pytest.raises(ValueError, match="one device"):
        vggt_sparse.linear(c.x, c.w.to(cuda))


@pytest.mark.parametrize("rows,inner,outer", [(1, 64, 64), (90, 520, 1040), (700, 1001, 130),
                                              (5000, 1032, 2000)])
@pytest.mark.parametrize("bias", [False, True])
def test_gate_gradients_by_themselves(cuda, rows, inner, outer, bias):
    """Every subset of weight, bias and gate: dgate with dW from the tiles, and without it from
    partial sums, is the same to its bounds."""
    c = Linear(cuda, rows, inner, outer, FP, gate=True, bias=bias, seed=rows)
    x = c.x
    for mask in range(1, 8):
        leaves = [t for i, t in enumerate((c.w, c.b, c.g)) if mask >> i & 1 and t is not None]
        for t in (c.w, c.b, c.g):
            if t is not None:
                t.requires_grad_(any(t is u for u in leaves))
        if not leaves:
            continue
        grads = dict(zip(map(id, leaves), torch.autograd.grad(c.call(), leaves, c.dy)))
        c.check_grads(None, *(grads.get(id(t)) for t in (c.w, c.b, c.g)))
    assert not x.requires_grad
