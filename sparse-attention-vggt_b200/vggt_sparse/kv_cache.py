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

Layouts.  Pools are [pages, kv_heads, page, dim] bf16 or fp16 (strides that are
multiples of 8 elements, the last dimension contiguous, 16-byte aligned, K and V
alike; dim 64 or 128, page a power of two from 16 to 1024).  ``table`` [seqs, width] int32 names the pages of
each sequence; slot s lies in page table[b, s // page].  New tokens of all
sequences are packed: rows starts[b] .. starts[b + 1] of q, k and v
[tokens, heads, dim] belong to sequence b; where their strides or address do not
suit the kernels they are copied.  ids and weights are
[seqs, kv_heads, width * page].

Gradients.  ``rotary`` is differentiable in x.  The cache holds values: what is
appended to it takes no part in a graph, nor do weights.  ``paged_attention`` has
no gradient; called with grad mode on and a q (or pools) that requires one, its
results are part of the graph, and a backward pass through them raises.

Like the other operators these only enqueue work on the current stream.
Page numbers, lengths and starts are checked on the device; ``status`` (an
int32 tensor) collects VGGT_STATUS_* bits, see ``check_cache_status``.
"""
import math
import os

import torch

from . import _lib
from .build import BINDING_PATH

_module = None


def _binding():
    """The compiled module of csrc/cache_binding.cpp, which checks arguments
    and calls the C ABI; there is no fallback."""
    global _module
    if _module is None:
        if not os.path.exists(BINDING_PATH):
            raise _lib.ExtensionMissing(
                "%s not found: build it with `python -m vggt_sparse.build`" % BINDING_PATH)
        _lib.load()
        from . import _cache_binding
        _module = _cache_binding
    return _module


class _Rotary(torch.autograd.Function):
    """The map is linear, its transpose the turn the other way."""

    @staticmethod
    def forward(ctx, x, positions, frequencies, layout, lengthen, inverse, out):
        ctx.save_for_backward(positions, frequencies)
        ctx.turn = layout, lengthen, not inverse
        if out is not None:
            ctx.mark_dirty(out)
        return _binding().rotary(x, positions, frequencies, layout, lengthen, inverse, out)

    @staticmethod
    def backward(ctx, grad):
        positions, frequencies = ctx.saved_tensors
        layout, lengthen, inverse = ctx.turn
        if grad.stride(2) != 1:
            grad = grad.contiguous()
        return (rotary(grad, positions, frequencies, layout=layout, lengthen=lengthen,
                       inverse=inverse), None, None, None, None, None, None)


class _NoGradient(torch.autograd.Function):
    """Makes ``t``, computed from ``inputs``, part of their graph."""

    @staticmethod
    def forward(ctx, t, *inputs):
        ctx.mark_dirty(t)
        return t

    @staticmethod
    def backward(ctx, grad):
        raise RuntimeError("paged_attention has no gradient: call it under torch.no_grad(), or "
                           "train with an attention that has one")


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


def rotary(x, positions, frequencies, *, layout="half", lengthen=1.0, inverse=False, out=None):
    """x [tokens, heads, dim] (bf16, fp16 or fp32; last dimension contiguous)
    with the first 2 * axes * len(frequencies) elements of each head turned by
    ``positions`` ([tokens] or [tokens, axes] int32) and the rest copied.

    layout "half" pairs element i with i + n of an axis's 2n elements,
    "interleaved" 2i with 2i + 1.  ``inverse`` turns the other way, which is
    the gradient of ``rotary`` with respect to x (autograd uses it).  ``out``
    may be x itself.
    """
    if getattr(x, "requires_grad", False) and torch.is_grad_enabled():
        return _Rotary.apply(x, positions, frequencies, layout, lengthen, inverse, out)
    return _binding().rotary(x, positions, frequencies, layout, lengthen, inverse, out)


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
    return _binding().append(k, v, k_pages, v_pages, table, before, starts, positions, frequencies,
                             layout, lengthen, ids, new_ids, weights, new_weights, after, status)


def paged_attention_workspace_size(total, seqs, kv_heads, group, dim, max_new, max_len):
    """Bytes of the workspace of ``paged_attention``: a contiguous uint8 tensor
    zeroed before its first use, used by one stream at a time."""
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
    without keys gives zeros and -inf, and so does one that belongs to no
    sequence (STATUS_BAD_LENGTH).

    ``max_new`` and ``max_len`` (default: all the table can hold) are the most
    new tokens of a sequence and the greatest length expected: they choose the
    kernel and the split, the result holds for any.  Without ``workspace`` the
    current stream's own is used.
    """
    both = _binding().attention(q, k_pages, v_pages, table, lengths, starts, max_new, max_len,
                                causal, scale, out, lse, workspace, status)
    if ((q.requires_grad or k_pages.requires_grad or v_pages.requires_grad)
            and torch.is_grad_enabled()):
        both = tuple(_NoGradient.apply(t, q, k_pages, v_pages) for t in both)
    return both


def paged_weights(q, lse, k_pages, table, lengths, starts, weights, *, max_new, max_len=None,
                  causal=True, scale=None, decay=1.0, status=None):
    """Add to ``weights`` (in place, returned) the probabilities that the new
    tokens' rows gave each cached key: decay * weights + sum exp(s - lse) over
    the rows and the query heads of the key's head; weights of +inf stay.  q,
    lse, lengths, starts, causal and scale as in ``paged_attention``, whose lse
    it takes."""
    return _binding().weigh(q, lse, k_pages, table, lengths, starts, weights, max_new, max_len,
                            causal, scale, decay, status)


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
    new = (None, None, None) if out is None else out
    return _binding().evict(weights, ids, k_pages, v_pages, table, lengths, budget, max_len,
                            recent_from, *new, status)


_MESSAGES = ((_lib.STATUS_TIMEOUT, "a device pipeline wait timed out"),
             (_lib.STATUS_BAD_PAGE, "a page number is outside the pool"),
             (_lib.STATUS_BAD_LENGTH, "a length or a start is out of range, or a sequence is full"))


def check_cache_status(status):
    """Wait for ``status`` and raise ValueError if an operator set a bit."""
    bits = int(status[0].item())
    if bits:
        raise ValueError("paged cache: " + "; ".join(m for b, m in _MESSAGES if bits & b))


class PagedKVCache:
    """Pools, page tables and books of a streaming cache.

    seqs sequences share ``pages`` pages of ``page`` slots; each may hold up to
    ``max_length`` tokens.  A step appends new tokens, attends from them and,
    where the cache is bounded, evicts:

        starts = cache.append(k, v, counts, positions=..., frequencies=...)
        out, lse = cache.attend(q, causal=False)     # also adds to the weights
        cache.evict(budget, recent=...)

    Lengths are known on the host (eviction leaves min(length, budget)), so
    pages are given out and taken back without waiting for the device.  All
    calls belong on one stream; ``check()`` waits and raises what the device
    found wrong.
    """

    def __init__(self, seqs, kv_heads, dim, *, pages, max_length, page=64,
                 dtype=torch.bfloat16, device="cuda"):
        if seqs < 1 or pages < 1 or max_length < 1:
            raise ValueError("seqs, pages and max_length must be positive")
        self.seqs, self.page, self.max_length = seqs, page, max_length
        self.width = -(-max_length // page)
        shape = (pages, kv_heads, page, dim)
        self.k_pages = torch.empty(shape, dtype=dtype, device=device)
        self.v_pages = torch.empty(shape, dtype=dtype, device=device)
        self.table = torch.zeros(seqs, self.width, dtype=torch.int32, device=device)
        slots = (seqs, kv_heads, self.width * page)
        self.ids = torch.full(slots, -1, dtype=torch.int32, device=device)
        self.weights = torch.zeros(slots, device=device)
        self._spare = torch.empty_like(self.weights), torch.empty_like(self.ids)
        self.length = torch.zeros(seqs, dtype=torch.int32, device=device)
        self.status = torch.zeros(1, dtype=torch.int32, device=device)
        self.lengths = [0] * seqs        # the same on the host
        self.seen = [0] * seqs           # tokens ever appended: the next token's id
        self._pages = [[] for _ in range(seqs)]
        self._free = list(range(pages - 1, -1, -1))
        self._step = None                # (starts, counts) of the last append

    def _ints(self, values):
        return torch.tensor(values, dtype=torch.int32).to(self.table.device, non_blocking=True)

    def append(self, k, v, counts, *, positions=None, frequencies=None, layout="half",
               lengthen=1.0, new_weights=None):
        """Append counts[b] tokens to sequence b (k, v packed in that order).
        Tokens are numbered as they come (``ids``); ``positions`` default to
        those numbers where ``frequencies`` are given.  ``new_weights`` of +inf
        keep tokens from eviction.  Returns starts."""
        if len(counts) != self.seqs or min(counts) < 0:
            raise ValueError("counts needs one number, not negative, per sequence")
        if sum(counts) != k.shape[0]:
            raise ValueError("counts add up to %d, k has %d tokens" % (sum(counts), k.shape[0]))
        need = []
        for b, n in enumerate(counts):
            if self.lengths[b] + n > self.max_length:
                raise ValueError("sequence %d would pass max_length %d" % (b, self.max_length))
            need.append(-(-(self.lengths[b] + n) // self.page) - len(self._pages[b]))
        if sum(max(0, n) for n in need) > len(self._free):
            raise ValueError("the pool is out of pages (%d free)" % len(self._free))
        for b, n in enumerate(need):
            if n > 0:
                first = len(self._pages[b])
                self._pages[b] += [self._free.pop() for _ in range(n)]
                self.table[b, first:first + n] = self._ints(self._pages[b][first:])
        starts, ids = [0], []
        for b, n in enumerate(counts):
            starts.append(starts[-1] + n)
            ids += range(self.seen[b], self.seen[b] + n)
        starts, ids = self._ints(starts), self._ints(ids)
        if frequencies is not None and positions is None:
            positions = ids
        self.length = paged_append(k, v, self.k_pages, self.v_pages, self.table, self.length,
                                   starts, positions=positions, frequencies=frequencies,
                                   layout=layout, lengthen=lengthen, ids=self.ids, new_ids=ids,
                                   weights=self.weights, new_weights=new_weights,
                                   status=self.status)
        for b, n in enumerate(counts):
            self.lengths[b] += n
            self.seen[b] += n
        self._step = (starts, max(1, max(counts)))
        return starts

    def attend(self, q, *, causal=True, scale=None, weigh=True, decay=1.0, out=None):
        """Attention of the last appended tokens over the cache: (out, lse).
        With ``weigh`` their probabilities are added to the keys' weights."""
        if self._step is None:
            raise ValueError("append comes before attend")
        starts, most = self._step
        longest = max(self.lengths)
        out, lse = paged_attention(q, self.k_pages, self.v_pages, self.table, self.length, starts,
                                   max_new=most, max_len=longest, causal=causal, scale=scale,
                                   out=out, status=self.status)
        if weigh:
            paged_weights(q, lse, self.k_pages, self.table, self.length, starts, self.weights,
                          max_new=most, max_len=longest, causal=causal, scale=scale, decay=decay,
                          status=self.status)
        return out, lse

    def evict(self, budget, *, recent=0):
        """Keep at most ``budget`` tokens of every sequence and key head; the
        ``recent`` last appended ones of a sequence go last.  A sequence that
        is evicted from can not be attended from again before an append."""
        if budget < 0:
            raise ValueError("budget must not be negative")
        longest = max(self.lengths)
        if longest <= budget:
            return
        newest = self._ints([n - recent for n in self.seen]) if recent > 0 else None
        new = (*self._spare, torch.empty_like(self.length))
        paged_evict(self.weights, self.ids, self.k_pages, self.v_pages, self.table, self.length,
                    budget, max_len=longest, recent_from=newest, out=new, status=self.status)
        self._spare = self.weights, self.ids
        self.weights, self.ids, self.length = new
        self._step = None
        for b in range(self.seqs):
            self.lengths[b] = min(self.lengths[b], budget)
            keep = -(-self.lengths[b] // self.page)
            self._free += reversed(self._pages[b][keep:])
            del self._pages[b][keep:]

    def release(self, seq):
        """Empty a sequence and take its pages back."""
        self._free += reversed(self._pages[seq])
        self._pages[seq] = []
        self.lengths[seq] = self.seen[seq] = 0
        self.length = self.length.clone()
        self.length[seq] = 0
        self.ids[seq] = -1
        self.weights[seq] = 0
        self._step = None

    def check(self):
        """Wait for the device and raise ValueError if an operator found bad
        pages, lengths or starts, or timed out."""
        check_cache_status(self.status)
