"""A global-attention layer over a stream of frames.

Where ``SparseGlobalLayer`` attends within a fixed set of frames,
``StreamingGlobalLayer`` takes one frame at a time, as the reference's
streaming model does (saf3r/models/official_streamvggt): the frame's tokens
attend to themselves and to the cached tokens of the frames before.  The cache
holds ``budget`` tokens per head; beyond that the tokens that received the
least attention are evicted: never the newest frame's, nor the special tokens of
the first frames, as many as fit beside it.
"""
import math

import torch

from .kv_cache import PagedKVCache, rotary, rotary_frequencies


class StreamingGlobalLayer:
    """``layer(q, k, v, positions)`` for the frames of one stream in turn.

    q, k, v [tokens, heads, dim] of the new frame before rotation, positions
    [tokens, 2] int32 (y, x): each half of a head turns by one of them, with
    the base of the framework's RoPE-2D.

    After a call the cache holds all of that frame.  The first ``special``
    tokens of a frame (camera and registers) are kept for good in the first
    ``pinned_frames`` = (budget - tokens_per_frame) // special frames of the
    stream; in later frames they are weighed like any other token, since the
    cache has no room to keep them and a whole new frame.
    """

    def __init__(self, heads, dim, tokens_per_frame, budget, *, special=5, base=100.0, page=64,
                 dtype=torch.bfloat16, device="cuda"):
        if budget < tokens_per_frame:
            raise ValueError("budget must hold a frame at least")
        special = min(special, tokens_per_frame)
        longest = budget + tokens_per_frame
        self.budget, self.special, self.tokens = budget, special, tokens_per_frame
        self.cache = PagedKVCache(1, heads, dim, pages=-(-longest // page), max_length=longest,
                                  page=page, dtype=dtype, device=device)
        self.frequencies, _ = rotary_frequencies(dim, base=base, axes=2, device=device)
        self.pinned_frames = (budget - tokens_per_frame) // special if special > 0 else 0
        self._init = torch.zeros(tokens_per_frame, device=device)
        self._init[:special] = math.inf

    def __call__(self, q, k, v, positions):
        if k.shape[0] != self.tokens:
            raise ValueError("frames of %d tokens expected, got %d" % (self.tokens, k.shape[0]))
        q = rotary(q, positions, self.frequencies)
        pinned = self.cache.seen[0] // self.tokens < self.pinned_frames
        self.cache.append(k, v, [self.tokens], positions=positions, frequencies=self.frequencies,
                          new_weights=self._init if pinned else None)
        out, _ = self.cache.attend(q, causal=False)
        self.cache.evict(self.budget, recent=self.tokens)
        return out
