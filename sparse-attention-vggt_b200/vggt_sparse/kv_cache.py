"""Streaming: a paged key/value cache and the operators that work on it.

The reference's streaming model keeps the keys and values of the frames seen
so far and attends to them from each new frame
(saf3r/models/official_streamvggt); its cache grows with the stream.  Here the
cache is paged, bounded by eviction, and served by five operators:

``rotary``           queries or keys turned by their positions
``paged_append``     new keys (turned) and values written into the cache
``paged_attention``  attention of the new tokens over the cache, with the
                     log-sum-exp of every row
``paged_weights``    the probability that each cached key received, added up
``paged_evict``      the keys of least weight evicted down to a budget

``PagedKVCache`` holds pools, page tables, lengths, ids and weights, gives out
pages and calls the operators in turn.

Layouts.  Pools are [pages, kv_heads, page, dim] bf16 or fp16 (any strides
whose last dimension is contiguous, K and V alike; dim 64 or 128, page a power
of two from 16 to 1024).  ``table`` [seqs, width] int32 names the pages of
each sequence; slot s lies in page table[b, s // page].  New tokens of all
sequences are packed: rows starts[b] .. starts[b + 1] of q, k and v
[tokens, heads, dim] belong to sequence b.  ids and weights are
[seqs, kv_heads, width * page].

Like the other operators these only enqueue work on the current stream.
Page numbers, lengths and starts are checked on the device; ``status`` (an
int32 tensor) collects VGGT_STATUS_* bits, see ``check_cache_status``.
"""
import math

import torch

from . import _lib
from .ops import _ptr, _require_cuda, _stream, dtype_code

_LAYOUTS = {"half": _lib.ROTARY_HALF, "interleaved": _lib.ROTARY_INTERLEAVED}
_ROTARY_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16,
                  torch.float32: _lib.DTYPE_FP32}


def rotary_frequencies(rotary_dim, *, base=10000.0, axes=1, scaling=None, factor=1.0,
                       original_length=None, slow_turns=1.0, fast_turns=32.0, device="cuda"):
    """(frequencies, lengthen) for ``rotary`` and ``paged_append``.

    ``rotary_dim`` elements of a head turn, split evenly over ``axes`` position
    axes; pair i of n turns by base ** (-i / n) radians per position.
    ``scaling`` stretches a model trained on short contexts by ``factor``:
      "linear"    every frequency divided by factor (positions interpolated)
      "base"      base * factor ** (n / (n - 1)): the slowest pair is slowed by
                  factor, the fastest one kept
      "by_parts"  pairs that make fewer than ``slow_turns`` turns over
                  ``original_length`` positions are divided by factor, those
                  with more than ``fast_turns`` kept, with a linear ramp
                  between; results are lengthened by 0.1 ln(factor) + 1
    Frequencies are float64 [n] on ``device``.
    """
    if rotary_dim < 2 or axes < 1 or rotary_dim % (2 * axes):
        raise ValueError("rotary_dim must be a positive multiple of 2 * axes")
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be positive")
    n = rotary_dim // (2 * axes)
    lengthen = 1.0
    if scaling == "base":
        base = base * factor ** (n / (n - 1)) if n > 1 else base
    f = [base ** (-i / n) for i in range(n)]
    if scaling == "linear":
        f = [v / factor for v in f]
    elif scaling == "by_parts":
        if not original_length or not fast_turns > slow_turns:
            raise ValueError("by_parts needs original_length, and fast_turns above slow_turns")
        keep = [(original_length * v / (2 * math.pi) - slow_turns) / (fast_turns - slow_turns)
                for v in f]
        keep = [min(1.0, max(0.0, k)) for k in keep]
        f = [v * (k + (1.0 - k) / factor) for v, k in zip(f, keep)]
        lengthen = 0.1 * math.log(factor) + 1.0 if factor > 1 else 1.0
    elif scaling not in (None, "base"):
        raise ValueError("scaling must be None, 'linear', 'base' or 'by_parts'")
    return torch.tensor(f, dtype=torch.float64, device=device), lengthen


def _ints(name, t, shape):
    if t.dtype != torch.int32 or t.shape != shape or not t.is_contiguous():
        raise ValueError("%s must be a contiguous int32 tensor of shape %s" % (name, tuple(shape)))
    return t.data_ptr()


def _status(status):
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() < 1:
        raise ValueError("status must be an int32 tensor with at least one element")
    return status.data_ptr()


def _positions(positions, tokens, frequencies, layout):
    """(pointer, axes) of positions [tokens] or [tokens, axes]."""
    axes = 1 if positions.dim() == 1 else positions.shape[-1]
    if positions.dim() > 2 or positions.shape[0] != tokens or positions.dtype != torch.int32 \
            or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32 [tokens] or [tokens, axes]")
    if frequencies is None or frequencies.dtype != torch.float64 or frequencies.dim() != 1 \
            or not frequencies.is_contiguous():
        raise ValueError("frequencies must be a contiguous float64 vector (rotary_frequencies)")
    if layout not in _LAYOUTS:
        raise ValueError("layout must be 'half' or 'interleaved'")
    return positions.data_ptr(), axes


def rotary(x, positions, frequencies, *, layout="half", lengthen=1.0, inverse=False, out=None):
    """x [tokens, heads, dim] (bf16, fp16 or fp32; last dimension contiguous)
    with the first 2 * axes * len(frequencies) elements of each head turned by
    ``positions`` ([tokens] or [tokens, axes] int32) and the rest copied.

    layout "half" pairs element i with i + n of an axis's 2n elements,
    "interleaved" 2i with 2i + 1.  ``inverse`` turns the other way, which is
    the gradient of ``rotary`` with respect to x.  ``out`` may be x itself.
    """
    if x.dim() != 3 or x.dtype not in _ROTARY_DTYPES or x.stride(2) != 1:
        raise ValueError("x must be [tokens, heads, dim], BF16, FP16 or FP32, last dimension "
                         "contiguous")
    t, h, d = x.shape
    pos, axes = _positions(positions, t, frequencies, layout)
    if out is None:
        out = torch.empty((t, h, d), dtype=x.dtype, device=x.device)
    elif out.shape != x.shape or out.dtype != x.dtype or out.stride(2) != 1:
        raise ValueError("out must have x's shape and dtype, last dimension contiguous")
    _require_cuda(x, positions, frequencies, out)
    _lib.check(_lib.load().vggt_rotary(
        x.data_ptr(), _ROTARY_DTYPES[x.dtype], t, h, d, x.stride(0), x.stride(1), pos, axes,
        frequencies.data_ptr(), frequencies.shape[0], _LAYOUTS[layout], lengthen, int(inverse),
        out.data_ptr(), out.stride(0), out.stride(1), _stream(x.device)))
    return out


def _pool_args(k_pages, v_pages, table, seqs):
    """The pool arguments of the C ABI (sizes, strides, table)."""
    if k_pages.dim() != 4 or k_pages.stride(3) != 1:
        raise ValueError("pools must be [pages, kv_heads, page, dim], last dimension contiguous")
    if v_pages is not None and (v_pages.shape != k_pages.shape or v_pages.dtype != k_pages.dtype
                                or v_pages.stride() != k_pages.stride()):
        raise ValueError("k_pages and v_pages must have the same shape, strides and dtype")
    if table.dim() != 2 or table.dtype != torch.int32 or not table.is_contiguous() \
            or (seqs is not None and table.shape[0] != seqs):
        raise ValueError("table must be contiguous int32 [seqs, width]")
    n, h, p, d = k_pages.shape
    s = k_pages.stride()
    return (n, h, p, d, s[0], s[1], s[2], table.data_ptr(), table.shape[1], table.shape[0])


def _rows_of(name, t, heads, k_pages):
    """t [tokens, heads, dim] with strides that the kernels take (else a copy)."""
    if t.dim() != 3 or t.shape[2] != k_pages.shape[3] or t.dtype != k_pages.dtype \
            or (heads is not None and t.shape[1] != heads):
        raise ValueError("%s must be [tokens, %s, %d] %s" % (
            name, "heads" if heads is None else heads, k_pages.shape[3], k_pages.dtype))
    if t.stride(2) != 1 or t.stride(0) % 8 or t.stride(1) % 8 or t.data_ptr() % 16:
        t = t.contiguous()
    return t


def paged_append(k, v, k_pages, v_pages, table, before, starts, *, positions=None,
                 frequencies=None, layout="half", lengthen=1.0, ids=None, new_ids=None,
                 weights=None, new_weights=None, after=None, status=None):
    """Write the packed new tokens' keys and values behind each sequence's
    ``before[b]`` cached tokens and return the new lengths.

    k, v [tokens, kv_heads, dim].  With ``positions`` the keys are turned as by
    ``rotary`` on their way.  ``ids`` and ``weights``, where given, get
    ``new_ids`` [tokens] and ``new_weights`` [tokens] (0 when None) in every
    head; a weight of +inf keeps a token from eviction.  Tokens past a
    sequence's last slot are dropped (STATUS_BAD_LENGTH).
    """
    code = dtype_code(k_pages.dtype)
    pool = _pool_args(k_pages, v_pages, table, None)
    seqs, slots = pool[9], pool[8] * pool[2]
    k, v = _rows_of("k", k, pool[1], k_pages), _rows_of("v", v, pool[1], k_pages)
    total = k.shape[0]
    if v.shape != k.shape:
        raise ValueError("k and v must have the same shape")
    pos, axes, freq, pairs = None, 0, None, 0
    if positions is not None:
        pos, axes = _positions(positions, total, frequencies, layout)
        freq, pairs = frequencies.data_ptr(), frequencies.shape[0]
    if ids is not None:
        _ints("ids", ids, (seqs, pool[1], slots))
        if new_ids is None:
            raise ValueError("ids needs new_ids")
        _ints("new_ids", new_ids, (total,))
    if weights is not None:
        _weights("weights", weights, (seqs, pool[1], slots))
        if new_weights is not None:
            _weights("new_weights", new_weights, (total,))
    if after is None:
        after = torch.empty_like(before)
    elif after.data_ptr() == before.data_ptr():
        raise ValueError("after must not be before")
    _require_cuda(k, v, k_pages, v_pages, table, before, starts, positions, frequencies, ids,
                  new_ids, weights, new_weights, after, status)
    _lib.check(_lib.load().vggt_paged_append(
        k.data_ptr(), v.data_ptr(), code, total, k.stride(0), k.stride(1), v.stride(0),
        v.stride(1), k_pages.data_ptr(), v_pages.data_ptr(), *pool,
        _ints("before", before, (seqs,)), _ints("starts", starts, (seqs + 1,)), pos, axes, freq,
        pairs, _LAYOUTS.get(layout, 0), lengthen, _ptr(ids), _ptr(new_ids), _ptr(weights),
        _ptr(new_weights), _ints("after", after, (seqs,)), _status(status), _stream(k.device)))
    return after


def _weights(name, t, shape):
    if t.dtype != torch.float32 or t.shape != shape or not t.is_contiguous():
        raise ValueError("%s must be a contiguous float32 tensor of shape %s"
                         % (name, tuple(shape)))


# One zeroed workspace per stream: its calls run one after another, and every
# call leaves the part that has to be zero at zero.
_WORKSPACES = {}


def _workspace(need, device, stream):
    if torch.cuda.is_current_stream_capturing():
        # a graph may be replayed on any stream: it gets a workspace of its own
        return torch.zeros(need, dtype=torch.uint8, device=device)
    key = (device.index, stream)
    ws = _WORKSPACES.get(key)
    if ws is None or ws.numel() < need:
        ws = _WORKSPACES[key] = torch.zeros(max(need, 1 << 20), dtype=torch.uint8, device=device)
    return ws


def paged_attention_workspace_size(total, seqs, kv_heads, group, dim, max_new, max_len):
    """Bytes of the workspace of ``paged_attention`` (zero-filled before its
    first use; one stream at a time)."""
    return int(_lib.load().vggt_paged_attention_workspace_size(total, seqs, kv_heads, group, dim,
                                                               max_new, max_len))


def paged_attention(q, k_pages, v_pages, table, lengths, starts, *, max_new, max_len=None,
                    causal=True, scale=None, out=None, lse=None, workspace=None, status=None):
    """Attention of the packed new tokens, which are already in the cache, over
    the cache; returns (out, lse).

    q [tokens, q_heads, dim], q_heads a multiple of the pools' heads (grouped
    heads); ``lengths`` count the new tokens.  With ``causal`` new token i of n
    sees the slots up to lengths[b] - n + i, otherwise every slot of its
    sequence.  lse [tokens, q_heads] fp32 is the row's log-sum-exp; a row
    without keys gives zeros and -inf.

    ``max_new`` and ``max_len`` (default: all the table can hold) are the most
    new tokens of a sequence and the greatest length expected: they choose the
    kernel and the split, the result holds for any.  Without ``workspace`` the
    current stream's own is used.
    """
    code = dtype_code(k_pages.dtype)
    pool = _pool_args(k_pages, v_pages, table, None)
    kv_heads, dim, seqs = pool[1], pool[3], pool[9]
    q = _rows_of("q", q, None, k_pages)
    total, heads = q.shape[0], q.shape[1]
    if heads < 1 or heads % kv_heads:
        raise ValueError("q's heads (%d) must be a multiple of the pools' (%d)" % (heads, kv_heads))
    if out is None:
        out = torch.empty((total, heads, dim), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(2) != 1 \
            or out.stride(0) % 8 or out.stride(1) % 8 or out.data_ptr() % 16:
        raise ValueError("out must have q's shape and dtype and 16-byte aligned rows")
    if lse is None:
        lse = torch.empty((total, heads), dtype=torch.float32, device=q.device)
    else:
        _weights("lse", lse, (total, heads))
    _require_cuda(q, k_pages, v_pages, table, lengths, starts, out, lse, workspace, status)
    max_len = pool[8] * pool[2] if max_len is None else max_len
    lib = _lib.load()
    need = lib.vggt_paged_attention_workspace_size(total, seqs, kv_heads, heads // kv_heads, dim,
                                                   max_new, max_len)
    stream = _stream(q.device)
    if workspace is None:
        workspace = _workspace(max(need, 1), q.device, stream)
    _lib.check(lib.vggt_paged_attention(
        q.data_ptr(), code, total, q.stride(0), q.stride(1), k_pages.data_ptr(),
        v_pages.data_ptr(), *pool, _ints("lengths", lengths, (seqs,)),
        _ints("starts", starts, (seqs + 1,)), heads // kv_heads, int(causal),
        dim ** -0.5 if scale is None else scale, max_new, max_len, out.data_ptr(), out.stride(0),
        out.stride(1), lse.data_ptr(), _status(status), workspace.data_ptr(),
        workspace.numel() * workspace.element_size(), stream))
    return out, lse


def paged_weights(q, lse, k_pages, table, lengths, starts, weights, *, max_new, max_len=None,
                  causal=True, scale=None, decay=1.0, status=None):
    """Add to ``weights`` (in place, returned) the probabilities that the new
    tokens' rows gave each cached key: decay * weights + sum exp(s - lse) over
    the rows and the query heads of the key's head.  q, lse, lengths, starts,
    causal and scale as in ``paged_attention``, whose lse it takes."""
    code = dtype_code(k_pages.dtype)
    pool = _pool_args(k_pages, None, table, None)
    kv_heads, dim, seqs, slots = pool[1], pool[3], pool[9], pool[8] * pool[2]
    q = _rows_of("q", q, None, k_pages)
    total, heads = q.shape[0], q.shape[1]
    if heads < 1 or heads % kv_heads:
        raise ValueError("q's heads (%d) must be a multiple of the pools' (%d)" % (heads, kv_heads))
    _weights("lse", lse, (total, heads))
    _weights("weights", weights, (seqs, kv_heads, slots))
    _require_cuda(q, lse, k_pages, table, lengths, starts, weights, status)
    _lib.check(_lib.load().vggt_paged_weights(
        q.data_ptr(), code, total, q.stride(0), q.stride(1), lse.data_ptr(), k_pages.data_ptr(),
        *pool, _ints("lengths", lengths, (seqs,)), _ints("starts", starts, (seqs + 1,)),
        heads // kv_heads, int(causal), dim ** -0.5 if scale is None else scale, decay, max_new,
        slots if max_len is None else max_len, weights.data_ptr(), _status(status),
        _stream(q.device)))
    return weights


def paged_evict(weights, ids, k_pages, v_pages, table, lengths, budget, *, max_len=None,
                recent_from=None, out=None, status=None):
    """Cut every sequence to at most ``budget`` tokens; returns (weights, ids,
    lengths), new tensors (or the three of ``out``), and moves keys and values
    within the pools.

    Each key head keeps its own slots of largest weight, ties to the lower
    slot, NaN last; tokens whose id is recent_from[b] or more are kept before
    all others.  Kept slots below the new length stay where they are, the
    others fill the holes there in order.  The sequences' pages must not be
    shared with other sequences.
    """
    code = dtype_code(k_pages.dtype)
    pool = _pool_args(k_pages, v_pages, table, None)
    seqs, slots = pool[9], pool[8] * pool[2]
    shape = (seqs, pool[1], slots)
    _weights("weights", weights, shape)
    _ints("ids", ids, shape)
    if out is None:
        out = torch.empty_like(weights), torch.empty_like(ids), torch.empty_like(lengths)
    new_weights, new_ids, new_lengths = out
    _weights("out[0]", new_weights, shape)
    _ints("out[1]", new_ids, shape)
    if recent_from is not None:
        _ints("recent_from", recent_from, (seqs,))
    _require_cuda(weights, ids, k_pages, v_pages, table, lengths, recent_from, *out, status)
    lib = _lib.load()
    ws = torch.empty(max(1, lib.vggt_paged_evict_workspace_size(seqs, pool[1], slots, budget)),
                     dtype=torch.uint8, device=weights.device)
    _lib.check(lib.vggt_paged_evict(
        weights.data_ptr(), ids.data_ptr(), code, k_pages.data_ptr(), v_pages.data_ptr(), *pool,
        _ints("lengths", lengths, (seqs,)), budget, _ptr(recent_from),
        slots if max_len is None else max_len, new_weights.data_ptr(), new_ids.data_ptr(),
        _ints("out[2]", new_lengths, (seqs,)), _status(status), ws.data_ptr(), ws.numel(),
        _stream(weights.device)))
    return new_weights, new_ids, new_lengths


_MESSAGES = ((_lib.STATUS_TIMEOUT, "a device pipeline wait timed out"),
             (_lib.STATUS_BAD_PAGE, "a page number is outside the pool"),
             (_lib.STATUS_BAD_LENGTH, "a length or a start is out of range, or a sequence is full"))


def check_cache_status(status):
    """Wait for ``status`` and raise ValueError if an operator set a bit."""
    bits = int(status[0].item())
    if bits:
        raise ValueError("paged cache: " + "; ".join(m for b, m in _MESSAGES if bits & b))
