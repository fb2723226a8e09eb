"""The streaming key/value cache's operators: their cases, their plain forms and their 64-bit definitions.

A streaming program keeps a paged cache of keys and values, ``[pages, kv_heads, page, dim]`` with a
page table per sequence.  Each step it rotates the new tokens' queries and keys, writes keys and
values into the cache, attends from the new tokens to the whole cache, adds the probabilities that
each cached key received to that key's weight, and, when the cache is over its budget, evicts the
keys of least weight.  One case is one pass through one of these operators:

rotary     queries rotated by their positions (half or interleaved pairs, part of the head, one or
           two position axes, frequencies scaled for long contexts)
append     keys rotated and written with their values behind each sequence's cached tokens
attend     attention of a chunk of new tokens over the paged cache, with the log-sum-exp per row
weigh      the probabilities of a chunk, recomputed from the log-sum-exp, summed per cached key
evict      per head, the keys of largest weight kept (ties to the lower slot); kept keys beyond the
           budget move into the slots that evicted ones leave
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---------------------------------------------------------------------------------------------
# cases
# ---------------------------------------------------------------------------------------------
def _rotary(tokens, heads, dim, rot, layout, axes, scaling, top, dtype):
    return dict(op="rotary", tokens=tokens, heads=heads, dim=dim, rot=rot, layout=layout, axes=axes,
                scaling=scaling, top=top, dtype=dtype)


def _append(seqs, new, cached, ragged, heads, dim, page, rot, layout, scaling, dtype):
    return dict(op="append", seqs=seqs, new=new, cached=cached, ragged=ragged, heads=heads, dim=dim, page=page,
                rot=rot, layout=layout, scaling=scaling, dtype=dtype)


def _attend(op, seqs, new, cached, ragged, q_heads, heads, dim, page, causal, dtype):
    return dict(op=op, seqs=seqs, new=new, cached=cached, ragged=ragged, q_heads=q_heads, heads=heads, dim=dim,
                page=page, causal=causal, dtype=dtype)


def _evict(seqs, cached, ragged, budget, recent, heads, dim, page, dtype):
    return dict(op="evict", seqs=seqs, cached=cached, ragged=ragged, budget=budget, recent=recent, heads=heads,
                dim=dim, page=page, dtype=dtype)


def listed():
    return [
        # 32 frames' queries on arrival, positions on the patch grid (two axes, as this framework's projection)
        dict(_rotary(43968, 16, 64, 64, "half", 2, "none", 39, "bf16"), name="rotary, 32 frames"),
        # one token of each of 16 sequences far into a long context: a quarter of the head, interleaved pairs
        dict(_rotary(16, 32, 128, 32, "interleaved", 1, "linear", 120000, "fp16"), name="rotary, 16 tokens"),
        # a new frame behind 31 cached ones
        dict(_append(1, 1374, 42594, 0.0, 16, 64, 64, 64, "half", "none", "bf16"), name="append, a frame"),
        # a prompt chunk of several sequences behind ragged caches, grouped heads, by-parts scaling
        dict(_append(4, 2048, 14000, 0.5, 8, 128, 32, 128, "half", "by_parts", "fp16"), name="append, 4 prompts"),
        # the smallest decode step: one token over one frame's keys
        dict(_attend("attend", 1, 1, 1374, 0.0, 16, 16, 64, 64, True, "bf16"), name="attend, a token"),
        # a decode batch over long ragged caches, four query heads to a key head
        dict(_attend("attend", 32, 1, 32768, 0.6, 32, 8, 128, 64, True, "bf16"), name="attend, 32 tokens"),
        # a new frame, all of whose tokens see one another and the 31 cached frames
        dict(_attend("attend", 1, 1374, 42594, 0.0, 16, 16, 64, 64, False, "bf16"), name="attend, a frame"),
        # prompt chunks of several sequences, causal, odd sizes, small pages
        dict(_attend("attend", 4, 1999, 12289, 0.5, 32, 8, 128, 16, True, "fp16"), name="attend, 4 prompts"),
        # the frame's weights over the whole cache
        dict(_attend("weigh", 1, 1374, 42594, 0.0, 16, 16, 64, 64, False, "bf16"), name="weigh, a frame"),
        # a decode batch's weights
        dict(_attend("weigh", 32, 1, 32768, 0.6, 32, 8, 128, 64, True, "fp16"), name="weigh, 32 tokens"),
        # the cache goes back from 32 frames to 31
        dict(_evict(1, 43968, 0.0, 42594, 1374, 16, 64, 64, "bf16"), name="evict, a frame"),
        # prompts cut down to a decode budget
        dict(_evict(16, 16383, 0.4, 4096, 256, 8, 128, 16, "bf16"), name="evict, 16 prompts"),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["rotary", "append", "attend", "attend", "weigh", "evict"])
    dtype = rng.choice(["bf16", "fp16"])
    dim = rng.choice([64, 128])
    page = rng.choice([16, 32, 64, 128])
    ragged = round(rng.uniform(0.0, 0.8), 2)
    scaling = rng.choice(["none", "linear", "by_parts"])
    layout = rng.choice(["half", "interleaved"])
    if op == "rotary":
        heads = rng.choice([1, 8, 12, 16, 32])
        axes = rng.choice([1, 2])
        rot = rng.choice([dim, dim // 2, dim // 4])
        tokens = _log(rng, 1, 43968 * 16 * 64 // (heads * dim))
        dtype = rng.choice(["bf16", "fp16", "fp32"])
        tokens = max(1, tokens // 2) if dtype == "fp32" else tokens
        return _rotary(tokens, heads, dim, rot, layout, axes, scaling, rng.choice([40, 4096, 130000]), dtype)
    if op == "append":
        heads = rng.choice([1, 2, 4, 8, 16])
        seqs = _log(rng, 1, 32)
        new = _log(rng, 1, max(1, 8192 * 8 * 128 // (seqs * heads * dim)))
        cached = _log(rng, 1, max(2, 65536 * 8 // (seqs * heads)))
        return _append(seqs, new, cached, ragged, heads, dim, page, rng.choice([dim, dim // 2]), layout, scaling, dtype)
    if op == "evict":
        heads = rng.choice([1, 2, 4, 8, 16])
        seqs = _log(rng, 1, 16)
        cached = _log(rng, 2, max(64, 43968 * 16 // (seqs * heads)) if seqs * heads > 16 else 43968)
        budget = max(1, int(cached * rng.uniform(0.1, 1.0)))
        return _evict(seqs, cached, ragged, budget, int(budget * rng.uniform(0.0, 0.5)), heads, dim, page, dtype)
    group = rng.choice([1, 2, 4, 7, 8])
    heads = rng.choice([1, 2, 4, 8, 16]) if group < 4 else rng.choice([1, 2, 4, 8])
    if rng.random() < 0.5:  # single tokens, or a few
        seqs = _log(rng, 1, 32)
        new = rng.choice([1, 1, 2, 5])
        cached = _log(rng, 1, max(64, 32768 * 32 * 8 * 128 // (seqs * heads * dim) // 8))
        cached = min(cached, 65536)
    else:
        seqs = _log(rng, 1, 4)
        new = _log(rng, 8, 2048)
        most = 1374 * 43968 * 16 * 64 // (seqs * new * heads * group * dim)
        cached = max(1, min(_log(rng, 16, 43968), most))
    return _attend(op, seqs, new, cached, ragged, heads * group, heads, dim, page, rng.random() < 0.7, dtype)


def _lengths(case):
    """Cached tokens of each sequence before the pass: the case's, less by up to `ragged` of it."""
    n = case["seqs"]
    return [max(1 if case["op"] == "evict" else 0,
                case["cached"] - int(case["cached"] * case["ragged"] * ((7 * b) % n) / n)) for b in range(n)]


def _new(case):
    """New tokens of each sequence: the case's, less by up to half of `ragged` of it, one at least."""
    n = case["seqs"]
    return [max(1, case["new"] - int(case["new"] * case["ragged"] * 0.5 * ((5 * b) % n) / n)) for b in range(n)]


# ---------------------------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------------------------
def _frequencies(rot, axes, scaling):
    """Angular steps per position of the pairs of one axis (64 bits) and the factor on cos and sin.  linear: positions
    divided by 4; by_parts: pairs that turn fewer than once in 8,192 positions are slowed 16-fold, those that turn more
    than 32 times are left, a linear ramp between, and both rotated vectors lengthened by 0.1 ln 16 + 1."""
    n = rot // axes // 2
    f = [10000.0 ** (-i / n) for i in range(n)]
    if scaling == "linear":
        return [v / 4.0 for v in f], 1.0
    if scaling == "by_parts":
        keep = [min(1.0, max(0.0, (8192 * v / (2 * math.pi) - 1.0) / 31.0)) for v in f]
        return [v * (k + (1.0 - k) / 16.0) for v, k in zip(f, keep)], 0.1 * math.log(16.0) + 1.0
    return f, 1.0


def _cache(case, lengths, gen, dev):
    """Two pools of pages, filled, and a page table whose pages lie in random order (-1 past a sequence's last page)."""
    dtype, page = DTYPES[case["dtype"]], case["page"]
    need = [-(-n // page) for n in lengths]
    order = torch.randperm(sum(need) + 3, generator=gen, device=dev).to(torch.int32)
    table = torch.full((len(need), max(1, max(need))), -1, device=dev, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    shape = (order.numel(), case["heads"], page, case["dim"])
    pools = [torch.empty(shape, device=dev, dtype=dtype).normal_(generator=gen) for _ in range(2)]
    return pools[0], pools[1], table


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    st = dict(case=case, op=case["op"])
    ints = lambda v: torch.tensor(v, device=dev, dtype=torch.int32)  # noqa: E731
    if case["op"] in ("rotary", "append"):
        f, st["lengthen"] = _frequencies(case["rot"], case.get("axes", 1), case["scaling"])
        st["freq"] = torch.tensor(f, device=dev, dtype=torch.float64)
    if case["op"] == "rotary":
        shape = (case["tokens"], case["heads"], case["dim"])
        st["x"] = torch.empty(shape, device=dev, dtype=dtype).normal_(generator=gen)
        st["pos"] = torch.randint(0, case["top"], (case["tokens"], case["axes"]), generator=gen, device=dev, dtype=torch.int32)
        return st
    before = _lengths(case)
    new = _new(case) if case["op"] != "evict" else [0] * case["seqs"]
    after = [a + b for a, b in zip(before, new)]
    st["k_pages"], st["v_pages"], st["table"] = _cache(case, after, gen, dev)
    st["max_len"] = max(after)
    width = st["table"].shape[1] * case["page"]
    slots = (case["seqs"], case["heads"], width)
    if case["op"] == "evict":
        st["before"] = ints(before)
        inside = torch.arange(width, device=dev) < st["before"][:, None, None]
        # heavy-tailed, with exact zeros and ties, as accumulated probabilities of keys that few queries look at
        w = torch.rand(slots, generator=gen, device=dev) ** 8 * 4.0
        w = torch.where(w < 1e-6, torch.zeros_like(w), w)
        w[:, :, :5] = math.inf  # the first tokens are never evicted
        st["weights"] = torch.where(inside, w, torch.zeros_like(w))
        # an earlier eviction has already put some newer tokens into older slots
        ids = torch.arange(width, device=dev, dtype=torch.int32).expand(slots).clone()
        jump = torch.rand(slots, generator=gen, device=dev) < 0.1
        ids += jump.to(torch.int32) * (case["cached"] // 16)
        st["ids"] = torch.where(inside, ids, torch.full_like(ids, -1))
        st["recent"] = ints([n - case["recent"] for n in before])
        return st
    total = sum(new)
    st["before"], st["after"] = ints(before), ints(after)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    st["starts"], st["max_new"] = ints(starts), max(new)
    if case["op"] == "append":
        shape = (total, 2, case["heads"], case["dim"])  # keys and values as slices of one projection
        kv = torch.empty(shape, device=dev, dtype=dtype).normal_(generator=gen)
        st["k"], st["v"] = kv[:, 0], kv[:, 1]
        st["pos"] = torch.cat([torch.arange(a, a + n, device=dev, dtype=torch.int32) for a, n in zip(before, new)])
        st["ids"] = torch.full(slots, -1, device=dev, dtype=torch.int32)
        st["weights"] = torch.zeros(slots, device=dev)
        first = torch.rand(total, generator=gen, device=dev) < 5 / 1374  # tokens never to be evicted
        st["init"] = torch.where(first, math.inf, 0.0)
        return st
    st["q"] = torch.empty((total, case["q_heads"], case["dim"]), device=dev, dtype=dtype).normal_(generator=gen) * 2
    if case["op"] == "weigh":
        st["lse"] = _plain_scores(st)[1]
        st["weights"] = torch.rand(slots, generator=gen, device=dev)
    return st


# ---------------------------------------------------------------------------------------------
# plain forms, in 32 bits
# ---------------------------------------------------------------------------------------------
def _turn(x, pos, freq, lengthen, layout):
    """x [T, H, D] turned by positions [T, axes].  The angle is formed in 64 bits: in 32, positions in the ten
    thousands leave too few bits of the fast pairs' angles."""
    angle = (pos.double()[:, :, None] * freq).flatten(1)  # axis by axis: [T, pairs]
    cos, sin = angle.cos().float()[:, None] * lengthen, angle.sin().float()[:, None] * lengthen
    axes, n = pos.shape[1], freq.numel()
    rot, rest = x[..., :2 * axes * n].float(), x[..., 2 * axes * n:].float()
    if layout == "half":  # per axis: first members of the pairs, then the second ones
        parts = rot.unflatten(-1, (axes, 2, n))
        a, b = parts[..., 0, :].flatten(-2), parts[..., 1, :].flatten(-2)
    else:
        a, b = rot[..., 0::2], rot[..., 1::2]
    c, d = a * cos - b * sin, a * sin + b * cos
    if layout == "half":
        out = torch.stack((c.unflatten(-1, (axes, n)), d.unflatten(-1, (axes, n))), -2).flatten(-3)
    else:
        out = torch.stack((c, d), -1).flatten(-2)
    return torch.cat((out, rest), -1).to(x.dtype)


def _rows(starts, most):
    """[B, most] row numbers of the packed new tokens and which of them are there."""
    at = torch.arange(most, device=starts.device)
    there = at < (starts[1:] - starts[:-1])[:, None]
    return torch.where(there, starts[:-1, None] + at, torch.zeros_like(at)).long(), there


def _gather(pages, table):
    """[B, heads, slots, D] in 32 bits."""
    return pages[table.clamp(min=0).long()].permute(0, 2, 1, 3, 4).flatten(2, 3).float()


def _plain_scores(st):
    """Masked scores [B, heads, group * most, slots], their log-sum-exp [T, q_heads], and the rows' numbers."""
    c = st["case"]
    rows, there = _rows(st["starts"], st["max_new"])
    group = c["q_heads"] // c["heads"]
    q = st["q"].float()[rows].unflatten(2, (c["heads"], group)).permute(0, 2, 3, 1, 4).flatten(2, 3)
    s = torch.matmul(q, _gather(st["k_pages"], st["table"]).transpose(2, 3))
    s *= c["dim"] ** -0.5
    slot = torch.arange(s.shape[-1], device=s.device)
    last = st["after"][:, None].expand(-1, st["max_new"])
    if c["causal"]:
        last = st["before"][:, None] + torch.arange(st["max_new"], device=s.device) + 1
    last = torch.where(there, last, torch.zeros_like(last))
    seen = (slot < last[:, :, None])[:, None].repeat(1, 1, group, 1)
    s.masked_fill_(~seen, -math.inf)
    del seen
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    lse = top[..., 0] + torch.log(torch.exp(s - top).sum(-1))
    lse = lse.unflatten(2, (group, st["max_new"])).permute(0, 3, 1, 2).flatten(2)
    return s, lse[there], rows, there


def _plain_attend(st):
    c = st["case"]
    s, lse, rows, there = _plain_scores(st)
    group = c["q_heads"] // c["heads"]
    wide = torch.zeros(there.shape + (c["q_heads"],), device=s.device)
    wide[there] = lse
    wide = wide.unflatten(2, (c["heads"], group)).permute(0, 2, 3, 1).flatten(2)
    s -= wide[..., None]
    s.exp_()
    o = torch.matmul(s, _gather(st["v_pages"], st["table"]))
    o = o.unflatten(2, (group, st["max_new"])).permute(0, 3, 1, 2, 4).flatten(2, 3)
    return o[there].to(st["q"].dtype), lse


def _plain_weigh(st):
    c = st["case"]
    s, _, rows, there = _plain_scores(st)
    group = c["q_heads"] // c["heads"]
    lse = st["lse"][rows].unflatten(2, (c["heads"], group)).permute(0, 2, 3, 1).flatten(2)
    s -= lse[..., None]
    s.exp_()
    st["weights"] += s.sum(2)
    return st["weights"]


def _put(pages, table, seq, slot, rows):
    page = pages.shape[2]
    at = table[seq, slot // page].long()
    pages[at, :, slot % page] = rows


def _plain_append(st):
    c = st["case"]
    rows, there = _rows(st["starts"], st["max_new"])
    seq = torch.arange(c["seqs"], device=rows.device)[:, None].expand_as(rows)[there]
    slot = (st["before"][:, None] + torch.arange(st["max_new"], device=rows.device))[there]
    _put(st["k_pages"], st["table"], seq, slot,
         _turn(st["k"], st["pos"][:, None], st["freq"], st["lengthen"], c["layout"]))
    _put(st["v_pages"], st["table"], seq, slot, st["v"])
    st["ids"][seq, :, slot] = st["pos"][:, None]
    st["weights"][seq, :, slot] = st["init"][:, None]
    after = st["before"] + (st["starts"][1:] - st["starts"][:-1])
    return st["k_pages"], st["v_pages"], st["ids"], st["weights"], after


def _plain_evict(st):
    c = st["case"]
    w, ids, budget, page = st["weights"], st["ids"], c["budget"], c["page"]
    slots = torch.arange(w.shape[2], device=w.device)
    inside = slots < st["before"][:, None, None]
    rank = torch.where(ids >= st["recent"][:, None, None], torch.full_like(w, math.inf), w)
    rank = torch.where(inside, rank, torch.full_like(w, -math.inf))
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(inside.expand_as(w))
    kept.scatter_(2, order[..., :budget], True)
    kept &= inside
    after = st["before"].clamp(max=budget)
    low = slots < after[:, None, None]
    hole, mover = ~kept & low, kept & ~low
    # the n-th hole takes the n-th mover, both in the order of their slots
    b, h, dst = hole.nonzero(as_tuple=True)
    _, _, src = mover.nonzero(as_tuple=True)
    for pages in (st["k_pages"], st["v_pages"]):
        pages[st["table"][b, dst // page].long(), h, dst % page] = pages[st["table"][b, src // page].long(), h, src % page]
    w2, ids2 = w.clone(), ids.clone()
    w2[b, h, dst], ids2[b, h, dst] = w[b, h, src], ids[b, h, src]
    w2 = torch.where(low, w2, torch.zeros_like(w2))
    ids2 = torch.where(low, ids2, torch.full_like(ids2, -1))
    return st["k_pages"], st["v_pages"], w2, ids2, after


# ---------------------------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------------------------
def run(st):
    c = st["case"]
    if not own:
        if st["op"] == "rotary":
            return _turn(st["x"], st["pos"], st["freq"], st["lengthen"], c["layout"])
        return dict(append=_plain_append, attend=_plain_attend, weigh=_plain_weigh, evict=_plain_evict)[st["op"]](st)
    vs = _framework()
    if st["op"] == "rotary":
        return vs.rotary(st["x"], st["pos"], st["freq"], layout=c["layout"], lengthen=st["lengthen"])
    if st["op"] == "append":
        after = vs.paged_append(st["k"], st["v"], st["k_pages"], st["v_pages"], st["table"], st["before"], st["starts"],
                                positions=st["pos"], frequencies=st["freq"], layout=c["layout"],
                                lengthen=st["lengthen"], ids=st["ids"], new_ids=st["pos"], weights=st["weights"],
                                new_weights=st["init"])
        return st["k_pages"], st["v_pages"], st["ids"], st["weights"], after
    if st["op"] == "attend":
        return vs.paged_attention(st["q"], st["k_pages"], st["v_pages"], st["table"], st["after"], st["starts"],
                                  max_new=st["max_new"], max_len=st["max_len"], causal=c["causal"])
    if st["op"] == "weigh":
        return vs.paged_weights(st["q"], st["lse"], st["k_pages"], st["table"], st["after"], st["starts"],
                                st["weights"], max_new=st["max_new"], max_len=st["max_len"], causal=c["causal"])
    w, ids, after = vs.paged_evict(st["weights"], st["ids"], st["k_pages"], st["v_pages"], st["table"], st["before"],
                                   c["budget"], max_len=st["max_len"], recent_from=st["recent"])
    return st["k_pages"], st["v_pages"], w, ids, after


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
    size = 4 if case["dtype"] == "fp32" else 2
    op = case["op"]
    if op == "rotary":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * size + 4 * case["tokens"] * case["axes"], "flops": 3 * n * case["rot"]}
    before, heads, dim = _lengths(case), case["heads"], case["dim"]
    if op == "evict":
        # weights and numbers read and written; an evicted key's slot below the budget is refilled: at least the moved
        # rows' share if evicted keys lie evenly over the slots, but for the newest, which stay
        kept = [min(n, case["budget"]) for n in before]
        loose = [max(0, n - case["recent"]) for n in before]
        moved = sum(k * (n - k) / n * min(1.0, lo / n) for k, n, lo in zip(kept, before, loose))
        return {"bytes": heads * (8 * sum(before) + 8 * sum(kept) + moved * 4 * dim * size), "flops": heads * sum(before)}
    new = _new(case)
    if op == "append":
        total = sum(new)
        return {"bytes": total * heads * (4 * dim * size + 8) + 12 * total, "flops": 3 * total * heads * case["rot"]}
    pairs = sum(n * a + (n * (n + 1) // 2 if case["causal"] else n * n) for n, a in zip(new, before))
    keys = sum(n + a for n, a in zip(new, before)) * heads
    rows = sum(new) * case["q_heads"]
    if op == "attend":
        return {"bytes": keys * dim * size * 2 + rows * (2 * dim * size + 4), "flops": 4 * pairs * case["q_heads"] * dim}
    return {"bytes": keys * (dim * size + 8) + rows * (dim * size + 4), "flops": 2 * pairs * case["q_heads"] * dim}


# ---------------------------------------------------------------------------------------------
# the definitions, in 64 bits
# ---------------------------------------------------------------------------------------------
def _exact_turn(x, pos, freq, lengthen, layout):
    x = x.double().clone()
    n = freq.numel()
    for axis in range(pos.shape[1]):
        for i in range(n):
            a, b = (2 * axis * n + i, 2 * axis * n + n + i) if layout == "half" else (2 * (axis * n + i), 2 * (axis * n + i) + 1)
            z = torch.polar(torch.full_like(pos[:, axis], lengthen, dtype=torch.float64), pos[:, axis].double() * freq[i])
            turned = torch.complex(x[:, :, a], x[:, :, b]) * z[:, None]
            x[:, :, a], x[:, :, b] = turned.real, turned.imag
    return x


def _slots_of(st, b, n):
    """Page numbers and places within the page of a sequence's first n slots."""
    slot = torch.arange(n, device=st["table"].device)
    page = st["case"]["page"]
    return st["table"][b, slot // page].long(), slot % page


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "rotary":
        return _exact_turn(st["x"], st["pos"], st["freq"], st["lengthen"], case["layout"])
    before = _lengths(case)
    if op == "evict":
        return _exact_evict(st, case, before)
    new, first = _new(case), 0
    if op == "append":
        kp, vp = st["k_pages"].double(), st["v_pages"].double()
        turned = _exact_turn(st["k"], st["pos"][:, None], st["freq"], st["lengthen"], case["layout"])
        w = st["weights"].double()
        for b, (n, m) in enumerate(zip(before, new)):
            page, at = _slots_of(st, b, n + m)
            kp[page[n:], :, at[n:]] = turned[first:first + m]
            vp[page[n:], :, at[n:]] = st["v"][first:first + m].double()
            w[b, :, n:n + m] = st["init"][first:first + m].double()
            first += m
        return kp, vp, None, w, None
    group = case["q_heads"] // case["heads"]
    q = st["q"].double()
    out, lse = torch.zeros_like(q), torch.zeros(q.shape[:2], device=q.device, dtype=torch.float64)
    w = st["weights"].double() if op == "weigh" else None
    for b, (n, m) in enumerate(zip(before, new)):
        page, at = _slots_of(st, b, n + m)
        for h in range(case["q_heads"]):
            s = q[first:first + m, h] @ st["k_pages"][page, h // group, at].double().T / math.sqrt(case["dim"])
            if case["causal"]:
                s += torch.full_like(s, -math.inf).triu(n + 1)
            if op == "weigh":
                w[b, h // group, :n + m] += torch.exp(s - st["lse"][first:first + m, h, None].double()).sum(0)
                continue
            lse[first:first + m, h] = torch.logsumexp(s, 1)
            out[first:first + m, h] = torch.softmax(s, 1) @ st["v_pages"][page, h // group, at].double()
        first += m
    return w if op == "weigh" else (out, lse)


def _exact_evict(st, case, before):
    """The moves found on the host, key by key; what moves is copied, so the values are those of the inputs."""
    kp, vp = st["k_pages"].clone(), st["v_pages"].clone()
    w, ids = st["weights"].cpu().double(), st["ids"].cpu()
    w2 = torch.zeros_like(w)
    for b, n in enumerate(before):
        page, at = _slots_of(st, b, n)
        page, at = page.tolist(), at.tolist()
        keep = min(n, case["budget"])
        newest = before[b] - case["recent"]
        for h in range(case["heads"]):
            value, number = w[b, h, :n].tolist(), ids[b, h, :n].tolist()
            rank = sorted(range(n), key=lambda j: (-(math.inf if number[j] >= newest else value[j]), j))
            kept = set(rank[:keep])
            holes = [j for j in range(keep) if j not in kept]
            movers = [j for j in range(keep, n) if j in kept]
            source = list(range(keep))
            for dst, src in zip(holes, movers):
                source[dst] = src
            w2[b, h, :keep] = w[b, h, source]
            if holes:
                to = (torch.tensor([page[j] for j in holes]), torch.tensor(h), torch.tensor([at[j] for j in holes]))
                of = (torch.tensor([page[j] for j in movers]), torch.tensor(h), torch.tensor([at[j] for j in movers]))
                to, of = (tuple(t.to(kp.device) for t in v) for v in (to, of))
                kp[to], vp[to] = kp[of], vp[of]
    return kp.double(), vp.double(), w2.to(kp.device), None, None
