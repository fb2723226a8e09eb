"""A whole global-attention block.

``GlobalBlock`` is the reference's block around the sparse global attention
(saf3r/models/official_vggt/layers/block.py:27-107):

    x = x + ls1 * proj(attention(norm1(x)))
    x = x + ls2 * fc2(gelu(fc1(norm2(x))))

in seven calls: the first norm, ``project_qkv``, block selection, attention, the
output projection (which reads the attention's head-major output in place), the
gated residual with the second norm, and the MLP's two products, of which the
last scales by ls2 and adds the residual.  Nothing between them goes through
another layout or an elementwise pass.
"""
import torch

from .block_attention import deferred_status
from .block_ops import linear, residual_norm
from .layer import SparseGlobalLayer
from .qkv import project_qkv


def _fp32(t):
    return None if t is None else t.detach().float().contiguous()


def _norm(norm):
    """(weight, bias, eps) of a LayerNorm module or triple, in fp32."""
    if isinstance(norm, torch.nn.LayerNorm):
        norm = norm.weight, norm.bias, norm.eps
    weight, bias, eps = norm
    return _fp32(weight), _fp32(bias), float(eps)


def _activation(act):
    """The name, as ``linear`` takes it, of an activation's module."""
    if act is None:  # the MLP's default
        return "gelu"
    name = {torch.nn.GELU: "gelu_tanh" if getattr(act, "approximate", "none") == "tanh" else "gelu",
            torch.nn.SiLU: "silu", torch.nn.ReLU: "relu"}.get(type(act))
    if name is None:
        raise ValueError("the module's activation %s is not one of linear's: give activation"
                         % type(act).__name__)
    return name


def _rope_base(attn):
    """The rotary embedding's base of an attention module; None where it has none."""
    if not hasattr(attn, "rope"):
        return 100.0
    if attn.rope is None:
        return None
    for name in ("base_frequency", "frequency"):
        if hasattr(attn.rope, name):
            return float(getattr(attn.rope, name))
    raise ValueError("the module's rope has no base_frequency: give rope_base")


class GlobalBlock:
    """``block(x, pos)`` for the tokens of a fixed set of frames.

    norm1, norm2     LayerNorm modules or (weight, bias, eps)
    qkv, proj, fc1, fc2
                     Linear modules or (weight, bias)
    ls1, ls2         the scales per channel, or None
    q_norm, k_norm   as ``project_qkv`` takes them
    rope_base        likewise; None: positions are not looked at
    activation       the MLP's, as ``linear`` takes it
    layer            the ``SparseGlobalLayer`` (by default one with
                     ``layer_options``)

    Weights are converted to ``dtype`` (bf16 or fp16) once, here; the norms'
    and the scales per channel, which may be far below fp16's range, stay in fp32.
    x [N, C] may be of ``dtype`` or fp32 (a residual stream held in 32 bits), and so
    is the result.  A wait that runs out on the device is raised as a ValueError by
    a later call or by ``check_status``, without the host's waiting for it; what the
    call at fault returned is not valid.  Calls
    share the layer's buffers: they belong on one stream, or behind one another.
    There is no gradient through the attention: a call runs without one.  ``mlp``
    alone is differentiable in x.
    """

    def __init__(self, heads, *, tokens_per_frame, norm1, qkv, proj, norm2, fc1, fc2, ls1=None,
                 ls2=None, q_norm=None, k_norm=None, special_per_frame=5, rope_base=100.0,
                 activation="gelu", layer=None, dtype=torch.bfloat16, **layer_options):
        if layer is not None and layer_options:
            raise ValueError("give either layer or its options")
        self.layer = layer or SparseGlobalLayer(heads, **layer_options)
        if self.layer.heads != heads:
            raise ValueError("the layer has %d heads, the block %d" % (self.layer.heads, heads))
        self.heads, self.dtype = heads, dtype
        self.tokens_per_frame, self.special_per_frame = tokens_per_frame, special_per_frame
        self.rope_base, self.q_norm, self.k_norm = rope_base, q_norm, k_norm
        self.activation = activation
        cast = lambda t: None if t is None else t.detach().to(dtype).contiguous()  # noqa: E731
        pair = lambda m: (m.weight, m.bias) if isinstance(m, torch.nn.Linear) else m  # noqa: E731
        self.norm1, self.norm2 = _norm(norm1), _norm(norm2)
        self.qkv, self.proj, self.fc1, self.fc2 = (tuple(cast(t) for t in pair(m))
                                                  for m in (qkv, proj, fc1, fc2))
        self.ls1, self.ls2 = _fp32(ls1), _fp32(ls2)
        with deferred_status(self.qkv[0].device):
            pass  # a graph's capture finds the status word in place

    @classmethod
    def from_module(cls, block, *, tokens_per_frame, **options):
        """From the reference's Block (its attention's qkv, q_norm, k_norm, proj
        and rope, its MLP's layers and activation, the LayerScales' gamma where there
        are any); an activation or a rope that is not known is refused, unless the
        option is given."""
        gamma = lambda m: getattr(m, "gamma", None)  # noqa: E731
        attn = block.attn
        if "activation" not in options:
            options["activation"] = _activation(getattr(block.mlp, "act", None))
        if "rope_base" not in options:
            options["rope_base"] = _rope_base(attn)
        return cls(attn.num_heads, tokens_per_frame=tokens_per_frame, norm1=block.norm1,
                   qkv=attn.qkv, proj=attn.proj, norm2=block.norm2, fc1=block.mlp.fc1,
                   fc2=block.mlp.fc2, ls1=gamma(block.ls1), ls2=gamma(block.ls2),
                   q_norm=attn.q_norm, k_norm=attn.k_norm, **options)

    def attention(self, x, pos=None, pos_count=None):
        """The attention of the normed tokens, head-major [heads, N, 64]."""
        with deferred_status(x.device) as status:
            return self._attention(x, pos, pos_count, status)

    def _attention(self, x, pos, pos_count, status):
        weight, bias, eps = self.norm1
        y, _ = residual_norm(x, None, weight, bias, eps=eps, dtype=self.dtype)
        if self.rope_base is None:
            pos = None
        qkv = project_qkv(y, *self.qkv, heads=self.heads, tokens_per_frame=self.tokens_per_frame,
                          special_per_frame=self.special_per_frame, q_norm=self.q_norm,
                          k_norm=self.k_norm, pos=pos, rope_base=self.rope_base,
                          pos_count=pos_count, status=status)
        return self.layer.forward_projected(qkv, status=status)

    def mlp(self, x, branch=None):
        """h + ls2 * fc2(gelu(fc1(norm2(h)))) with h = x, or x + ls1 * branch."""
        with deferred_status(x.device) as status:
            return self._mlp(x, branch, status)

    def _mlp(self, x, branch, status):
        weight, bias, eps = self.norm2
        y, h = residual_norm(x, branch, weight, bias, eps=eps, dtype=self.dtype,
                             gate=self.ls1 if branch is not None else None)
        wide = linear(y, *self.fc1, activation=self.activation, status=status)
        return linear(wide, *self.fc2, gate=self.ls2, residual=h, status=status)

    @torch.no_grad()
    def __call__(self, x, pos=None, pos_count=None):
        """x [N, C] (or [1, N, C]); pos as in ``project_qkv``."""
        # the tokens of one sample attend to one another: flattened, a batch would be one
        if x.dim() == 3 and x.shape[0] != 1:
            raise ValueError("batch one only")
        if x.dim() not in (2, 3):
            raise ValueError("x must be [N, C]")
        flat = x.reshape(-1, x.shape[-1])
        with deferred_status(x.device) as status:
            a = self._attention(flat, pos, pos_count, status)
            p = linear(a, *self.proj, head_major=True, status=status)
            return self._mlp(flat, p, status).view(x.shape)
