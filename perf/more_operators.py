"""The dense operators around the attention of a block: their cases, their plain forms and their 64-bit definitions.

A transformer block is more than its attention: its output is projected, scaled per channel and added to the residual
stream, normed, widened, activated, narrowed, scaled and added again.  One case is one pass through one of these:

linear       y = residual + gate * activation(x W^T + b): a matrix product whose epilogue does the rest of its half of
             the block; x may be head-major, as the attention leaves it
linear_grad  the same with the gradients of x, W, b, gate and residual
norm         h = x + gate * post_norm(branch), y = norm(h): the end of one half of a block and the start of the next
             (a layer norm or a root-mean-square one; gates per channel or per channel and group of rows)
norm_grad    the same with the gradients of x, branch, gate and the norms' weights and biases
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _linear(op, rows, inner, outer, activation, bias, gate, residual, heads, dtype, stream):
    """stream: the type of the residual and of y; heads: 0, or those of a head-major x."""
    return dict(op=op, rows=rows, inner=inner, outer=outer, activation=activation, bias=bias, gate=gate,
                residual=residual, heads=heads, dtype=dtype, stream=stream)


def _norm(op, rows, width, norm, post, branch, affine, groups, dtype, stream, params):
    """post: the norm of the branch or ""; affine: whether the norms have weights and (layer norms) biases; groups: 0
    without a gate, 1 with one for all rows, else one for each of so many runs of rows."""
    return dict(op=op, rows=rows, width=width, norm=norm, post=post, branch=branch, affine=affine, groups=groups,
                dtype=dtype, stream=stream, params=params)


def listed():
    return [
        # one token of a decoder's first MLP product
        dict(_linear("linear", 1, 1024, 4096, "gelu", True, False, False, 0, "bf16", "bf16"), name="linear, a token"),
        # a decode batch's second one: scaled per channel, added to the residual
        dict(_linear("linear", 32, 4096, 1024, "", True, True, True, 0, "fp16", "fp16"), name="linear, 32 tokens"),
        # a frame's attention output, head-major, back into the residual stream
        dict(_linear("linear", 1374, 1024, 1024, "", True, True, True, 16, "bf16", "bf16"), name="linear, a frame"),
        # 32 frames widened
        dict(_linear("linear", 43968, 1024, 4096, "gelu", True, False, False, 0, "bf16", "bf16"),
             name="linear, 32 frames up"),
        # 32 frames narrowed again, onto a residual stream held in 32 bits
        dict(_linear("linear", 43968, 4096, 1024, "", True, True, True, 0, "bf16", "fp32"),
             name="linear, 32 frames down"),
        # a few dozen rows of odd widths: a head on pooled tokens, trained
        dict(_linear("linear_grad", 43, 1001, 517, "silu", True, True, True, 0, "fp16", "fp16"),
             name="linear gradient, odd"),
        # a frame's first MLP product, trained
        dict(_linear("linear_grad", 1374, 1024, 4096, "gelu", True, False, False, 0, "bf16", "bf16"),
             name="linear gradient, a frame up"),
        # 16 frames' second one, trained
        dict(_linear("linear_grad", 21984, 4096, 1024, "", True, True, True, 0, "bf16", "bf16"),
             name="linear gradient, 16 frames down"),
        # one token between two halves of a block
        dict(_norm("norm", 1, 1024, "layer", "", True, True, 1, "bf16", "bf16", "bf16"), name="norm, a token"),
        # 32 frames between two halves of a block, the stream held in 32 bits
        dict(_norm("norm", 43968, 1024, "layer", "", True, True, 1, "bf16", "fp32", "fp32"), name="norm, 32 frames"),
        # four prompts of a wide model with norms before and after, trained
        dict(_norm("norm_grad", 7996, 4096, "rms", "rms", True, True, 1, "fp16", "fp16", "fp16"),
             name="norm gradient, 4 prompts"),
        # 32 frames, a gate for each frame, trained
        dict(_norm("norm_grad", 43968, 1024, "layer", "", True, True, 32, "bf16", "bf16", "fp32"),
             name="norm gradient, 32 frames"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear_grad", "norm", "norm_grad"])
    dtype = rng.choice(["bf16", "fp16"])
    stream = rng.choice([dtype, dtype, "fp32"])
    if op.startswith("linear"):
        heads = rng.choice([0, 0, 0, 8, 16])
        step = rng.choice([64, 64, 8, 1])
        inner = heads * 64 if heads else max(1, _log(rng, 64, 8192) // step) * step
        outer = max(1, _log(rng, 64, 8192) // step) * step
        most = max(1, (43968 * 1024 * 4096 if op == "linear" else 21984 * 4096 * 1024) // (inner * outer))
        rows = min(most, rng.choice([_log(rng, 1, 43968), _log(rng, 1, 96)]))
        activation = rng.choice(["", "", "gelu", "gelu_tanh", "silu", "relu"])
        residual = rng.random() < 0.5
        return _linear(op, rows, inner, outer, activation, rng.random() < 0.7, rng.random() < 0.4, residual, heads,
                       dtype, stream if residual else dtype)
    width = max(1, _log(rng, 32, 8192) // 8) * 8 - rng.choice([0, 0, 0, 3])
    rows = min(_log(rng, 1, 43968), 43968 * 1024 // width)
    norm, branch = rng.choice(["layer", "rms"]), rng.random() < 0.85
    post = rng.choice(["", "", norm]) if branch else ""
    groups = rng.choice([0, 1, 1, rows, max(1, rows // 7)]) if branch else 0
    rows = max(1, rows // groups) * groups if groups else rows
    if rng.random() < 0.1:
        dtype = stream = "fp32"
        rows = max(1, rows // 2 // max(1, groups)) * max(1, groups)
    return _norm(op, rows, width, norm, post, branch, rng.random() < 0.8, groups, dtype, stream,
                 rng.choice([dtype, "fp32"]))


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype, stream = DTYPES[case["dtype"]], DTYPES[case["stream"]]

    def normal(*shape, scale=1.0, mean=0.0, type=dtype):
        return (torch.empty(shape, device=dev).normal_(generator=gen) * scale + mean).to(type)

    st = dict(case=case, op=case["op"])
    rows = case["rows"]
    if case["op"].startswith("linear"):
        inner, outer, heads = case["inner"], case["outer"], case["heads"]
        st["x"] = normal(heads, rows, inner // heads) if heads else normal(rows, inner)
        st["weight"] = normal(outer, inner, scale=inner ** -0.5)
        st["bias"] = normal(outer, scale=0.2) if case["bias"] else None
        st["gate"] = normal(outer, scale=0.3) if case["gate"] else None  # a layer's scale per channel, trained
        st["residual"] = normal(rows, outer, scale=2.0, type=stream) if case["residual"] else None
        leaves = ("x", "weight", "bias", "gate", "residual")
        if case["op"] == "linear_grad":
            st["dy"] = normal(rows, outer, scale=0.1, type=stream)
    else:
        width, params = case["width"], DTYPES[case["params"]]
        # a stream whose channels differ in size, and a mean that is not zero
        st["x"] = (normal(rows, width, scale=2.0, mean=0.3, type=torch.float32)
                   * (1.0 + 4.0 * normal(width, type=torch.float32).abs() ** 2 / 4.0)).to(stream)
        st["branch"] = normal(rows, width) if case["branch"] else None
        shape = (width,) if case["groups"] == 1 else (case["groups"], width)
        st["gate"] = normal(*shape, scale=0.3, type=params) if case["groups"] else None
        affine = lambda: normal(width, scale=0.2, mean=1.0, type=params)  # noqa: E731
        shift = lambda: normal(width, scale=0.2, type=params)  # noqa: E731
        st["weight"] = affine() if case["affine"] else None
        st["bias"] = shift() if case["affine"] and case["norm"] == "layer" else None
        st["post_weight"] = affine() if case["affine"] and case["post"] else None
        st["post_bias"] = shift() if case["affine"] and case["post"] == "layer" else None
        leaves = ("x", "branch", "gate", "weight", "bias", "post_weight", "post_bias")
        if case["op"] == "norm_grad":
            st["dy"] = normal(rows, width, scale=0.1)
            st["dh"] = normal(rows, width, scale=0.1, type=stream)
    st["leaves"] = [n for n in leaves if st[n] is not None]
    if case["op"].endswith("grad"):
        for n in st["leaves"]:
            st[n].requires_grad_()
    return st


# ---------------------------------------------------------------------------------------------
# plain forms, in 32 bits
# ---------------------------------------------------------------------------------------------
SQRT_HALF = math.sqrt(0.5)
TANH_IN = math.sqrt(2.0 / math.pi)


def _f(t):
    return None if t is None else t.float()


def _activate(z, name):
    """The activation of z and its derivative there."""
    if name == "gelu":
        phi = 0.5 * torch.erfc(-z * SQRT_HALF)
        return z * phi, phi + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
    if name == "gelu_tanh":
        s = torch.sigmoid(2.0 * TANH_IN * (z + 0.044715 * z * z * z))
        return z * s, s + z * s * (1.0 - s) * (2.0 * TANH_IN) * (1.0 + 3.0 * 0.044715 * z * z)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1.0 - s)
    if name == "relu":
        return z.clamp(min=0.0), (z > 0).float()
    return z, torch.ones_like(z)


def _plain_linear(st):
    c = st["case"]
    x, w, b, gate, res = (_f(st[n]) for n in ("x", "weight", "bias", "gate", "residual"))
    if c["heads"]:
        x = x.transpose(0, 1).flatten(1)
    z = torch.matmul(x, w.t())
    if b is not None:
        z += b
    a, slope = _activate(z, c["activation"])
    y = a if gate is None else a * gate
    if res is not None:
        y = y + res
    y = y.to(DTYPES[c["stream"]])
    if st["op"] == "linear":
        return y
    dy = st["dy"].float()
    da = dy if gate is None else dy * gate
    dz = da * slope
    dx = torch.matmul(dz, w)
    if c["heads"]:
        dx = dx.unflatten(1, (c["heads"], -1)).transpose(0, 1)
    grads = dict(x=dx, weight=torch.matmul(dz.t(), x), bias=dz.sum(0), gate=(dy * a).sum(0), residual=dy)
    return [y] + [grads[n].to(st[n].dtype).contiguous() for n in st["leaves"]]


def _normed(x, kind, eps):
    """x normed over its last dimension, and one over its deviation (or root mean square)."""
    if kind == "layer":
        x = x - x.mean(-1, keepdim=True)
    r = torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    return x * r, r


def _norm_slope(g, hat, r, kind):
    """The gradient of what was normed to `hat`, from that of the normed values."""
    d = g - hat * (g * hat).mean(-1, keepdim=True)
    if kind == "layer":
        d = d - g.mean(-1, keepdim=True)
    return d * r


def _plain_norm(st):
    c = st["case"]
    x, f, gate, w, b, pw, pb = (_f(st[n]) for n in ("x", "branch", "gate", "weight", "bias", "post_weight", "post_bias"))
    if gate is not None and gate.dim() == 2:
        gate = gate.repeat_interleave(c["rows"] // c["groups"], 0)
    h, p = x, f
    if f is not None:
        if c["post"]:
            fhat, fr = _normed(f, c["post"], 1e-5)
            p = fhat if pw is None else fhat * pw
            p = p if pb is None else p + pb
        h = x + (p if gate is None else p * gate)
    hat, r = _normed(h, c["norm"], 1e-5)
    y = hat if w is None else hat * w
    y = y if b is None else y + b
    out = [y.to(DTYPES[c["dtype"]]), h.to(DTYPES[c["stream"]])]
    if st["op"] == "norm":
        return out
    dy = st["dy"].float()
    dh = st["dh"].float() + _norm_slope(dy if w is None else dy * w, hat, r, c["norm"])
    grads = dict(x=dh, weight=(dy * hat).sum(0), bias=dy.sum(0))
    if f is not None:
        dp = dh if gate is None else dh * gate
        if gate is not None:
            grads["gate"] = (dh * p).unflatten(0, (c["groups"], -1)).sum(1).view(st["gate"].shape)
        grads["branch"] = dp
        if c["post"]:
            grads |= dict(post_weight=(dp * fhat).sum(0), post_bias=dp.sum(0))
            grads["branch"] = _norm_slope(dp if pw is None else dp * pw, fhat, fr, c["post"])
    return out + [grads[n].to(st[n].dtype) for n in st["leaves"]]


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if not own:
        with torch.no_grad():
            return _plain_linear(st) if st["op"].startswith("linear") else _plain_norm(st)
    vs = _framework()
    if st["op"].startswith("linear"):
        y = vs.linear(st["x"], st["weight"], st["bias"], activation=c["activation"] or None, gate=st["gate"],
                      residual=st["residual"], head_major=c["heads"] > 0)
        if st["op"] == "linear":
            return y
        return [y.detach(), *torch.autograd.grad(y, [st[n] for n in st["leaves"]], st["dy"])]
    y, h = vs.residual_norm(st["x"], st["branch"], st["weight"], st["bias"], norm=c["norm"], gate=st["gate"],
                            post_norm=c["post"] or None, post_weight=st["post_weight"], post_bias=st["post_bias"],
                            eps=1e-5, dtype=DTYPES[c["dtype"]])
    if st["op"] == "norm":
        return [y, h]
    grads = torch.autograd.grad([y, h], [st[n] for n in st["leaves"]], [st["dy"], st["dh"]])
    return [y.detach(), h.detach(), *grads]


_vs = None


def _framework():
    global _vs
    if _vs is None:
        import os
        import sys
        root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "sparse-attention-vggt_b200")
        if root not in sys.path:
            sys.path.insert(0, root)
        import vggt_sparse
        _vs = vggt_sparse
    return _vs


# ---------------------------------------------------------------------------------------------
# what a pass cannot do without
# ---------------------------------------------------------------------------------------------
def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    e, s, rows = size[case["dtype"]], size[case["stream"]], case["rows"]
    grad = case["op"].endswith("grad")
    if case["op"].startswith("linear"):
        k, n = case["inner"], case["outer"]
        small = n * (case["bias"] + case["gate"]) * e
        fwd = (rows * k + n * k) * e + small + rows * n * s * (2 if case["residual"] else 1)
        # the gradients read dy too and write dx, dW, db and dgate; the residual's is dy itself
        bwd = rows * n * s + (rows * k + n * k) * e + small if grad else 0
        return {"bytes": fwd + bwd, "flops": (6 if grad else 2) * rows * n * k}
    n, p = rows * case["width"], size[case["params"]]
    both = 1 if case["branch"] else 0
    few = case["width"] * p * (case["groups"] + case["affine"] * ((1 if case["norm"] == "rms" else 2)
                                                                 + {"": 0, "rms": 1, "layer": 2}[case["post"]]))
    fwd = n * (2 * s + (both + 1) * e) + few
    bwd = n * (2 * s + (both + 1) * e) + few if grad else 0
    return {"bytes": fwd + bwd, "flops": n * (30 if grad else 10)}


# ---------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def exact(case, seed):
    """The operator written down in 64 bits; its gradients by differentiating that."""
    st = prepare(case, seed)
    grad = case["op"].endswith("grad")
    with torch.set_grad_enabled(grad):
        v = {n: st[n].detach().double().requires_grad_(grad) for n in st["leaves"]}
        outs, given = _define_linear(case, v, st) if case["op"].startswith("linear") else _define_norm(case, v, st)
        if not grad:
            return outs[0] if case["op"] == "linear" else outs
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, [v[n] for n in st["leaves"]], given))


def _define_linear(case, v, st):
    x = v["x"]
    if case["heads"]:
        x = torch.einsum("hnd->nhd", x).reshape(case["rows"], case["inner"])
    z = torch.einsum("mk,nk->mn", x, v["weight"])
    z = z + v["bias"] if "bias" in v else z
    if case["activation"] == "gelu":
        z = z * torch.special.ndtr(z)
    elif case["activation"] == "gelu_tanh":
        z = 0.5 * z * (1 + torch.tanh((2 / math.pi) ** 0.5 * (z + 0.044715 * z ** 3)))
    elif case["activation"] == "silu":
        z = z / (1 + torch.exp(-z))
    elif case["activation"] == "relu":
        z = torch.maximum(z, torch.zeros_like(z))
    y = z * v["gate"] if "gate" in v else z
    y = v["residual"] + y if "residual" in v else y
    return [y], [st["dy"].double()] if "dy" in st else None


def _define_norm(case, v, st):
    def norm(t, kind, weight, bias):
        if kind == "layer":
            var, mean = torch.var_mean(t, -1, correction=0, keepdim=True)
            t = (t - mean) / torch.sqrt(var + 1e-5)
        else:
            t = t / torch.sqrt(torch.linalg.vector_norm(t, dim=-1, keepdim=True) ** 2 / t.shape[-1] + 1e-5)
        t = t * weight if weight is not None else t
        return t + bias if bias is not None else t

    h = v["x"]
    if case["branch"]:
        p = v["branch"]
        if case["post"]:
            p = norm(p, case["post"], v.get("post_weight"), v.get("post_bias"))
        if "gate" in v:
            runs = case["groups"]
            p = (p.reshape(runs, -1, case["width"]) * v["gate"].reshape(runs, 1, case["width"])).reshape(p.shape)
        h = h + p
    y = norm(h, case["norm"], v.get("weight"), v.get("bias"))
    return [y, h], [st["dy"].double(), st["dh"].double()] if "dy" in st else None
