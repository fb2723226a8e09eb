"""The streaming cache's operators on the GPU against plain 64-bit code.

Bounds (u: unit roundoff of the element type, 2^-8 bf16, 2^-11 fp16):
* rotary: one rounding of a value that fp32 holds to 2^-22 of the pair's length;
* attention: the output's own rounding u |o|, the rounding of each probability
  u sum p |v|, and 2^-13 sum p |v| for exponentials and scores in fp32;
* log-sum-exp: scores in fp32 (2^-20 of the largest magnitudes summed) and
  exponentials good to 2^-16;
* weights: probabilities good to 2e-5, added over n rows in fp32 (n 2^-24);
* ids, lengths, moved rows and their weights: exact.
"""
import math

import pytest
import torch

import vggt_sparse
from vggt_sparse import _lib

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
BF, FP = torch.bfloat16, torch.float16


def ints(v, dev):
    return torch.tensor(v, dtype=torch.int32, device=dev)


class Case:
    """A cache whose unowned slots hold NaN, and the new tokens' queries."""

    def __init__(self, dev, lengths, new, heads=2, group=2, dim=64, page=16, dtype=BF, seed=0,
                 layout="hnd", spare=3, width=None, scale_q=2.0):
        g = torch.Generator().manual_seed(seed)
        self.dev, self.lengths, self.new, self.group = dev, lengths, new, group
        self.dim, self.page, self.heads, self.dtype = dim, page, heads, dtype
        need = [-(-n // page) for n in lengths]
        order = torch.randperm(sum(need) + spare, generator=g)
        width = max(1, max(need)) if width is None else width
        table = torch.full((len(lengths), width), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n].to(torch.int32)
            at += n
        n_pages = order.numel()
        shape = (n_pages, heads, page, dim)
        if layout == "hnd":
            k, v = (torch.full(shape, math.nan, dtype=dtype) for _ in range(2))
        elif layout == "nhd":  # [pages, page, heads, dim]
            k, v = (torch.full((n_pages, page, heads, dim), math.nan, dtype=dtype).transpose(1, 2)
                    for _ in range(2))
        else:  # keys and values of a page side by side
            kv = torch.full((n_pages, 2) + shape[1:], math.nan, dtype=dtype)
            k, v = kv[:, 0], kv[:, 1]
        self.k, self.v = [], []
        for b, n in enumerate(lengths):
            kb, vb = (torch.randn(n, heads, dim, generator=g).to(dtype) for _ in range(2))
            for s in range(n):
                p = int(table[b, s // page])
                k[p, :, s % page] = kb[s]
                v[p, :, s % page] = vb[s]
            self.k.append(kb.to(dev))
            self.v.append(vb.to(dev))
        move = lambda t: torch.empty_strided(t.shape, t.stride(), dtype=dtype, device=dev).copy_(t)  # noqa: E731
        if layout == "both":
            kv = kv.to(dev)
            self.kp, self.vp = kv[:, 0], kv[:, 1]
        else:
            self.kp, self.vp = move(k), move(v)
        self.table = table.to(dev)
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        self.starts_l = starts
        self.starts, self.len = ints(starts, dev), ints(lengths, dev)
        self.q = (scale_q * torch.randn(starts[-1], heads * group, dim, generator=g)).to(dtype).to(dev)
        self.status = torch.zeros(1, dtype=torch.int32, device=dev)

    def rows(self, b):
        return slice(self.starts_l[b], self.starts_l[b + 1])

    def seen(self, b, causal):
        n, m = self.new[b], self.lengths[b]
        j = torch.arange(m, device=self.dev)
        last = m - n + torch.arange(n, device=self.dev) + 1 if causal else \
            torch.full((n,), m, device=self.dev)
        return j[None] < last[:, None]

    def scores(self, b, causal, scale=None):
        """[heads * group, n, m] in 64 bits, -inf where a row does not see."""
        scale = self.dim ** -0.5 if scale is None else scale
        q = self.q[self.rows(b)].double()
        k = self.k[b].double().repeat_interleave(self.group, 1)
        s = torch.einsum("nhd,mhd->hnm", q, k) * scale
        size = torch.einsum("nhd,mhd->hnm", q.abs(), k.abs()) * scale
        return s.masked_fill(~self.seen(b, causal), -math.inf), size

    def check(self, out, lse, causal, scale=None, skip=()):
        assert int(self.status) == 0
        for b in range(len(self.new)):
            if self.new[b] == 0 or b in skip:
                continue
            s, size = self.scores(b, causal, scale)
            want_l = torch.logsumexp(s, -1).T
            p = torch.nan_to_num(torch.exp(s - torch.logsumexp(s, -1, keepdim=True)), nan=0.0)
            v = self.v[b].double().repeat_interleave(self.group, 1)
            want = torch.einsum("hnm,mhd->nhd", p, v)
            mag = torch.einsum("hnm,mhd->nhd", p, v.abs())
            got = out[self.rows(b)].double()
            u = U[self.dtype]
            bound = u * want.abs() + (u + 2.0 ** -13) * mag + 1e-7
            err = (got - want).abs()
            assert bool((err <= bound).all()), (b, float((err - bound).max()), float(err.max()))
            got_l = lse[self.rows(b)].double()
            empty = want_l == -math.inf
            assert bool((got_l[empty] == -math.inf).all())
            assert bool((got[empty] == 0).all())
            lim = 2.0 ** -16 + 2.0 ** -20 * size.amax(-1).T if s.shape[-1] else torch.zeros_like(want_l)
            err = (got_l - want_l).abs()[~empty]
            assert bool((err <= lim[~empty]).all()), (b, float(err.max()))

    def attend(self, causal=True, **kw):
        kw.setdefault("max_new", max(1, max(self.new)))
        return vggt_sparse.paged_attention(self.q, self.kp, self.vp, self.table, self.len,
                                           self.starts, causal=causal, status=self.status, **kw)


# ------------------------------------------------------------------ rotary
def turned(x, pos, freq, lengthen, layout, inverse=False):
    x = x.double().clone()
    n = freq.numel()
    pos = pos.reshape(pos.shape[0], -1)
    for a in range(pos.shape[1]):
        ang = pos[:, a].double()[:, None] * freq[None] * (-1 if inverse else 1)
        c, s = (torch.cos(ang) * lengthen)[:, None], (torch.sin(ang) * lengthen)[:, None]
        part = x[..., 2 * a * n:2 * (a + 1) * n]
        u, w = (part[..., :n], part[..., n:]) if layout == "half" else (part[..., 0::2], part[..., 1::2])
        y, z = u * c - w * s, u * s + w * c
        if layout == "half":
            part = torch.cat((y, z), -1)
        else:
            part = torch.stack((y, z), -1).flatten(-2)
        x[..., 2 * a * n:2 * (a + 1) * n] = part
    return x


ROTARY = [  # tokens, heads, dim, rotary_dim, axes, layout, dtype
    (1, 1, 64, 64, 1, "half", BF), (1, 32, 128, 128, 1, "interleaved", FP),
    (7, 3, 64, 64, 2, "half", BF), (33, 5, 128, 32, 1, "interleaved", BF),
    (33, 5, 128, 96, 1, "half", FP), (5, 2, 72, 12, 2, "interleaved", BF),
    (3, 2, 6, 2, 1, "half", torch.float32), (257, 16, 64, 16, 1, "half", torch.float32),
    (19, 4, 80, 40, 4, "half", BF), (1, 7, 128, 128, 2, "interleaved", torch.float32),
    (2000, 2, 128, 64, 1, "half", BF)]


@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("t,h,d,rot,axes,layout,dtype", ROTARY)
def test_rotary(cuda, t, h, d, rot, axes, layout, dtype, inverse):
    g = torch.Generator().manual_seed(t + d)
    wide = torch.randn(t, 2 * h, d + 8, generator=g).to(dtype).to(cuda)
    x = wide[:, h:, :d] if t % 2 else wide[:, :h, :d].contiguous()
    pos = torch.randint(-3, 2 ** 31 - 1, (t, axes), generator=g, dtype=torch.int64)
    pos[::2] %= 5000
    pos = pos.to(torch.int32).to(cuda)
    freq, lengthen = vggt_sparse.rotary_frequencies(rot, axes=axes, scaling="by_parts", factor=4.0,
                                                    original_length=2048)
    got = vggt_sparse.rotary(x, pos if axes > 1 else pos[:, 0].contiguous(), freq, layout=layout,
                             lengthen=lengthen, inverse=inverse).double()
    want = turned(x, pos, freq, lengthen, layout, inverse)
    # at 2^31 radians a 64-bit angle itself is off by 2^-22
    size = lengthen * 1.5 * x.double().abs().amax(-1, keepdim=True)
    bound = U[dtype] * want.abs() + 2.0 ** -20 * size
    assert bool(((got - want).abs() <= bound).all())
    assert torch.equal(got[..., rot:], x[..., rot:].double())


@pytest.mark.parametrize("t,h,d,rot,axes,layout,dtype", [
    (40003, 1, 64, 64, 1, "half", BF), (40003, 1, 64, 32, 1, "interleaved", FP),
    (20001, 2, 128, 128, 2, "half", torch.float32), (9999, 2, 72, 12, 2, "interleaved", BF),
    (160000, 1, 6, 2, 1, "half", FP), (37886, 1, 64, 64, 1, "half", BF)])
def test_rotary_many_tokens_of_few_heads(cuda, t, h, d, rot, axes, layout, dtype):
    """Several tokens to a thread, and odd numbers of them; every eighth of a
    turn and its neighbours are among the angles."""
    g = torch.Generator().manual_seed(t)
    wide = torch.randn(t, h + 1, d + 8, generator=g).to(dtype).to(cuda)
    x = wide[:, 1:, :d]
    pos = torch.randint(-70000, 70000, (t, axes), generator=g)
    pos[:4096] = torch.arange(-2048, 2048)[:, None]
    pos = pos.to(torch.int32).to(cuda)
    freq, lengthen = vggt_sparse.rotary_frequencies(rot, axes=axes)
    freq = freq.clone()
    freq[0] = 2 * math.pi / 8
    freq[-1] = 2 * math.pi / 4096
    pos = pos if axes > 1 else pos[:, 0].contiguous()
    want = turned(x, pos, freq, lengthen, layout)
    got = vggt_sparse.rotary(x, pos, freq, layout=layout, lengthen=lengthen)
    size = 1.5 * x.double().abs().amax(-1, keepdim=True)
    err = (got.double() - want).abs()
    assert bool((err <= U[dtype] * want.abs() + 2.0 ** -21 * size).all())
    assert torch.equal(got[..., rot:], x[..., rot:])
    assert torch.equal(vggt_sparse.rotary(x, pos, freq, layout=layout, lengthen=lengthen, out=x), got)
    assert not torch.isnan(wide).any()


def test_rotary_in_place_and_gradient(cuda):
    """In place gives the same bits; the inverse is the transposed map (the
    gradient), checked by a difference quotient: the map is linear."""
    g = torch.Generator().manual_seed(1)
    x, y = (torch.randn(9, 3, 64, generator=g).to(cuda) for _ in range(2))
    pos = torch.randint(0, 4000, (9,), generator=g).to(torch.int32).to(cuda)
    freq, lengthen = vggt_sparse.rotary_frequencies(48, scaling="by_parts", factor=8.0,
                                                    original_length=512)
    run = lambda v, **k: vggt_sparse.rotary(v, pos, freq, lengthen=lengthen, **k)  # noqa: E731
    fx = run(x)
    grad = run(y, inverse=True)  # of sum(y * rotary(x))
    assert abs(float((fx.double() * y).sum() - (x.double() * grad).sum())) <= 2.0 ** -18 * x.numel()
    step = torch.zeros_like(x)
    for at in ((0, 0, 0), (4, 1, 23), (8, 2, 47), (3, 0, 60)):
        step.zero_()
        step[at] = 0.5
        quotient = ((run(x + step).double() - run(x - step).double()) * y).sum()
        assert abs(float(quotient - grad[at])) <= 2.0 ** -16 * 64
    z = x.clone()
    assert torch.equal(run(z, out=z), fx)


# ------------------------------------------------------------------ append
@pytest.mark.parametrize("layout", ["hnd", "nhd", "both"])
@pytest.mark.parametrize("dim,page,dtype,rot", [(64, 16, BF, "half"), (128, 64, FP, "interleaved"),
                                                (64, 128, FP, None)])
def test_append(cuda, layout, dim, page, dtype, rot):
    new = [3, 0, 1, 40, 17]
    c = Case(cuda, [5, 9, 0, 64, 15], [0] * 5, heads=3, dim=dim, page=page, dtype=dtype,
             layout=layout, spare=20, width=8)
    # pages for the new tokens
    used = set(c.table[c.table >= 0].tolist())
    free = [p for p in range(c.kp.shape[0]) if p not in used]
    for b, n in enumerate(c.lengths):
        for i in range(-(-n // page), -(-(n + new[b]) // page)):
            c.table[b, i] = free.pop()
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    total, slots = starts[-1], 8 * page
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(total, 3, 3, dim, generator=g).to(dtype).to(cuda)
    k, v = qkv[:, 1], qkv[:, 2]
    pos = torch.randint(0, 9000, (total,), generator=g).to(torch.int32).to(cuda)
    freq, lengthen = vggt_sparse.rotary_frequencies(dim // 2)
    ids = torch.full((5, 3, slots), -1, dtype=torch.int32, device=cuda)
    weights = torch.zeros(5, 3, slots, device=cuda)
    init = torch.rand(total, generator=g).to(cuda)
    init[0] = math.inf
    kw = dict(positions=pos, frequencies=freq, layout=rot) if rot else {}
    kp0, vp0 = c.kp.clone(), c.vp.clone()
    after = vggt_sparse.paged_append(k, v, c.kp, c.vp, c.table, c.len, ints(starts, cuda), ids=ids,
                                     new_ids=pos, weights=weights, new_weights=init,
                                     status=c.status, **kw)
    assert after.tolist() == [n + m for n, m in zip(c.lengths, new)] and int(c.status) == 0
    want_k = turned(k, pos, freq, 1.0, rot) if rot else k.double()
    for b, n in enumerate(c.lengths):
        for i in range(new[b]):
            s, row = n + i, starts[b] + i
            p = int(c.table[b, s // page])
            got = c.kp[p, :, s % page].double()
            assert bool(((got - want_k[row]).abs() <= U[dtype] * want_k[row].abs() + 2.0 ** -18).all())
            assert torch.equal(c.vp[p, :, s % page], v[row])
            assert ids[b, :, s].tolist() == [int(pos[row])] * 3
            assert weights[b, :, s].tolist() == [float(init[row])] * 3
            kp0[p, :, s % page] = c.kp[p, :, s % page]
            vp0[p, :, s % page] = c.vp[p, :, s % page]
    same = lambda x, y: torch.equal(torch.nan_to_num(x, nan=7.0), torch.nan_to_num(y, nan=7.0))  # noqa: E731
    assert same(kp0, c.kp) and same(vp0, c.vp)  # nothing else was written
    assert int((ids >= 0).sum()) == 3 * total


def test_append_past_the_end_and_bad_pages(cuda):
    """A full sequence drops the rest, an unusable page is not written; both
    set a status bit."""
    c = Case(cuda, [30, 5], [0, 0], heads=1, page=16, width=2)
    k = torch.randn(6, 1, 64, device=cuda).to(BF)
    c.table[1, 0] = 10 ** 6
    kp0 = c.kp.clone()
    after = vggt_sparse.paged_append(k, k, c.kp, c.vp, c.table, c.len, ints([0, 4, 6], cuda),
                                     status=c.status)
    assert after.tolist() == [32, 7]
    assert int(c.status) == _lib.STATUS_BAD_LENGTH | _lib.STATUS_BAD_PAGE
    p = int(c.table[0, 1])
    assert torch.equal(c.kp[p, :, 14:], k[:2].transpose(0, 1))
    kp0[p, :, 14:] = k[:2].transpose(0, 1)
    assert torch.equal(torch.nan_to_num(kp0, nan=7.0), torch.nan_to_num(c.kp, nan=7.0))
    with pytest.raises(ValueError, match="sequence is full"):
        vggt_sparse.check_cache_status(c.status)


# ------------------------------------------------------------------ attention
ATTEND = [  # lengths, new, heads, group, dim, page, dtype, layout
    ([1], [1], 1, 1, 64, 16, BF, "hnd"),
    ([130], [1], 2, 4, 128, 64, BF, "hnd"),
    ([64, 65, 1, 700, 0, 33], [1, 1, 1, 1, 0, 1], 2, 1, 64, 32, FP, "nhd"),
    ([300, 17, 2000], [3, 5, 2], 2, 7, 128, 16, BF, "both"),
    ([500, 44], [9, 8], 2, 3, 64, 64, FP, "hnd"),
    ([90, 260], [33, 70], 1, 2, 64, 16, BF, "hnd"),
    ([513, 129, 1024], [200, 129, 1], 2, 1, 64, 64, BF, "hnd"),
    ([515, 77, 300], [250, 77, 3], 1, 5, 128, 32, FP, "both"),
    ([1000], [1], 1, 48, 128, 128, BF, "hnd"),
    ([2300], [300], 1, 3, 128, 1024, BF, "nhd"),
    ([5000, 4000], [130, 1], 2, 2, 64, 256, FP, "hnd"),
]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,new,heads,group,dim,page,dtype,layout", ATTEND)
def test_attention(cuda, lengths, new, heads, group, dim, page, dtype, layout, causal):
    c = Case(cuda, lengths, new, heads, group, dim, page, dtype, seed=len(lengths), layout=layout)
    c.check(*c.attend(causal), causal)


@pytest.mark.parametrize("max_new,max_len", [(1, 1), (1, 10 ** 6), (4000, 64), (64, 4096)])
def test_attention_holds_for_any_expectation(cuda, max_new, max_len):
    """max_new and max_len choose the kernel and the split, not the result."""
    c = Case(cuda, [700, 3, 1500], [90, 1, 20], 2, 2, 64, 16)
    c.check(*c.attend(True, max_new=max_new, max_len=max_len), True)


@pytest.mark.parametrize("new", [40, 300])
def test_attention_rows_without_keys(cuda, new):
    """More new tokens than the cache holds: the first rows see nothing."""
    c = Case(cuda, [new - 17, 0, 50], [new, new, 2], 2, 2, 64, 16)
    out, lse = c.attend(True)
    c.check(out, lse, True)
    assert bool((lse[:17] == -math.inf).all()) and bool((out[new:2 * new] == 0).all())


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [5, 200])
def test_attention_later_tokens_do_not_reach_earlier_rows(cuda, new, dim):
    """NaN and infinity in the keys and values of the chunk's later tokens:
    rows that do not see them are as if they were not there."""
    c = Case(cuda, [450, 200], [new, new], 1, 2, dim, 16, FP)
    bad = 450 - new // 2
    out0, lse0 = c.attend(True)
    p = int(c.table[0, bad // 16])
    c.kp[p, :, bad % 16] = math.nan
    c.vp[p, :, bad % 16, 3] = math.inf
    c.vp[p, :, bad % 16, 5] = math.nan
    out, lse = c.attend(True)
    first = bad - (450 - new)  # the first row that sees it
    assert bool(torch.isnan(lse[first:new]).all())
    assert bool(torch.isfinite(out[:first]).all()) and bool(torch.isfinite(lse[:first]).all())
    c.k[0], c.v[0] = c.k[0].clone(), c.v[0].clone()
    full = c.new[0]
    # rows below `first` against the plain form of the clean inputs
    u = U[FP]
    diff = (out[:first].double() - out0[:first].double()).abs()
    assert bool((diff <= 2 * (u + 2.0 ** -12) * 8).all())
    assert bool(((lse[:first] - lse0[:first]).abs() <= 2.0 ** -14).all())
    assert torch.equal(out[full:], out0[full:])


@pytest.mark.parametrize("new", [4, 70])
def test_attention_infinite_score_spoils_its_row(cuda, new):
    """A score of +inf makes the row's probabilities inf - inf, in whichever
    column of a tile it stands; rows that do not see the key stay as they are."""
    c = Case(cuda, [100], [new], 1, 1, 64, 16, FP)
    c.q[..., 0] = c.q[..., 0].abs() + 1
    clean, _ = c.attend(True)
    for j in [*range(20), 63, 64, 97, 99]:
        at = int(c.table[0, j // 16]), 0, j % 16, 0
        old = c.kp[at].clone()
        c.kp[at] = math.inf
        out, lse = c.attend(True)
        c.kp[at] = old
        first = max(0, j - (100 - new))
        assert bool(torch.isnan(out[first:]).all()), j
        assert not torch.isfinite(lse[first:]).any(), j
        assert torch.equal(out[:first], clean[:first]), j


def test_attention_infinite_value_is_seen(cuda):
    c = Case(cuda, [100], [1], 1, 1, 64, 16, FP)
    p = int(c.table[0, 2])
    c.vp[p, 0, 5, 7] = math.inf
    out, _ = c.attend(True)
    assert float(out[0, 0, 7]) == math.inf
    assert int(torch.isfinite(out[0, 0]).sum()) == 63


@pytest.mark.parametrize("new", [3, 180])
def test_attention_large_scores(cuda, new):
    """Scores of several hundred, in rising and falling order over the keys."""
    c = Case(cuda, [900, 400], [new, new], 1, 2, 64, 64, BF, scale_q=40.0)
    c.check(*c.attend(True), True)
    c = Case(cuda, [900, 400], [new, new], 1, 2, 64, 64, BF)
    ramp = torch.linspace(-3, 3, 900, device=cuda)
    for b, n in enumerate(c.lengths):
        for flip in (False, True):
            r = ramp[:n].flip(0) if flip else ramp[:n]
            k = (c.k[b].float() + r[:, None, None]).to(BF)
            for s in range(n):
                c.kp[int(c.table[b, s // 64]), :, s % 64] = k[s]
            c.k[b] = k
    c.q = (c.q.float().abs()).to(BF)
    c.check(*c.attend(True), True)


def test_attention_scale_strides_and_out(cuda):
    c = Case(cuda, [200, 31], [70, 1], 2, 2, 64, 16)
    wide = torch.zeros(71, 3, 4, 64, device=cuda, dtype=BF)
    wide[:, 1] = c.q
    c.q = wide[:, 1]
    out = torch.full((71, 4, 128), 9.0, device=cuda, dtype=BF)[:, :, 64:]
    got, lse = c.attend(False, scale=0.03, out=out)
    assert got.data_ptr() == out.data_ptr()
    c.check(got, lse, False, 0.03)


def test_attention_bad_pages_and_lengths(cuda):
    c = Case(cuda, [100, 100], [1, 40], 1, 1, 64, 16)
    c.table[0, 1] = -5
    c.table[1, 2] = 10 ** 7
    c.attend(True)
    assert int(c.status) == _lib.STATUS_BAD_PAGE
    for bad_len, bad_starts in (([-3, 10 ** 9], None), (None, [5, 2, 60]), (None, [-4, 1, 10 ** 6])):
        c = Case(cuda, [100, 100], [1, 40], 1, 1, 64, 16)
        if bad_len:
            c.len = ints(bad_len, cuda)
            c.kp.zero_()
            c.vp.zero_()
        if bad_starts:
            c.starts = ints(bad_starts, cuda)
        c.attend(True)
        assert int(c.status) & _lib.STATUS_BAD_LENGTH


@pytest.mark.parametrize("new", [1, 150])
def test_attention_repeats_bit_for_bit_and_in_a_graph(cuda, new):
    c = Case(cuda, [3000, 1700], [new, new], 2, 2, 64, 64)
    out, lse = c.attend(True)
    for _ in range(5):
        again = c.attend(True)
        assert torch.equal(again[0], out) and torch.equal(again[1], lse)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        again = c.attend(True)
    torch.cuda.current_stream().wait_stream(other)
    assert torch.equal(again[0], out)
    o2, l2 = torch.empty_like(out), torch.empty_like(lse)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.attend(True, out=o2, lse=l2)
    for _ in range(3):
        o2.zero_()
        graph.replay()
        assert torch.equal(o2, out) and torch.equal(l2, lse)


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("lengths,new,heads,group,dim,page,dtype,layout", ATTEND)
def test_weights(cuda, lengths, new, heads, group, dim, page, dtype, layout, causal):
    c = Case(cuda, lengths, new, heads, group, dim, page, dtype, seed=len(lengths), layout=layout)
    slots = c.table.shape[1] * page
    w0 = torch.rand(len(new), heads, slots, device=cuda)
    lse = torch.full((c.q.shape[0], heads * group), -math.inf, device=cuda)
    want = w0.double()
    total = torch.zeros_like(want)
    for b in range(len(new)):
        n = lengths[b]
        want[b, :, :n] *= 0.75
        if new[b] == 0 or n == 0:
            continue
        s, _ = c.scores(b, causal)
        l = torch.logsumexp(s, -1)
        lse[c.rows(b)] = l.T.float()
        p = torch.nan_to_num(torch.exp(s - lse[c.rows(b)].T[..., None].double()), nan=0.0)
        add = p.sum(1).unflatten(0, (heads, group)).sum(1)
        want[b, :, :n] += add
        total[b, :, :n] += add
    w = w0.clone()
    got = vggt_sparse.paged_weights(c.q, lse, c.kp, c.table, c.len, c.starts, w, causal=causal,
                                    max_new=max(new), decay=0.75, status=c.status)
    assert got.data_ptr() == w.data_ptr() and int(c.status) == 0
    rows = max(new) * group
    bound = (2e-5 + rows * 2.0 ** -24) * total + 2.0 ** -23 * want
    assert bool(((got.double() - want).abs() <= bound).all()), \
        float(((got.double() - want).abs() - bound).max())
    for b, n in enumerate(lengths):
        assert torch.equal(got[b, :, n:], w0[b, :, n:])
    w2 = w0.clone()
    vggt_sparse.paged_weights(c.q, lse, c.kp, c.table, c.len, c.starts, w2, causal=causal,
                              max_new=max(new), decay=0.75)
    assert torch.equal(w, w2)


@pytest.mark.parametrize("max_new", [1, 500])
def test_weights_rows_without_keys_and_odd_keys(cuda, max_new):
    """Empty rows add nothing; a NaN key spoils its own weight alone."""
    c = Case(cuda, [25, 40], [40, 3], 1, 2, 64, 16)
    _, lse = c.attend(True)
    c.kp[int(c.table[0, 0]), :, 2] = math.nan
    w = torch.zeros(2, 1, c.table.shape[1] * 16, device=cuda)
    vggt_sparse.paged_weights(c.q, lse, c.kp, c.table, c.len, c.starts, w, max_new=max_new)
    assert bool(torch.isnan(w[0, 0, 2])) and int(torch.isnan(w).sum()) == 1
    assert abs(float(w[1].sum()) - 3 * 2) <= 1e-4


@pytest.mark.parametrize("max_new", [1, 500])
def test_weights_odd_rows_and_scores(cuda, max_new):
    """A NaN row spoils the weights of all keys that it sees, a score of +inf
    that of its key, in whichever column of a tile they stand."""
    c = Case(cuda, [100], [60], 1, 1, 64, 16)
    c.q[..., 0] = c.q[..., 0].abs() + 1
    _, lse = c.attend(True)

    def weights(q, lse):
        w = torch.zeros(1, 1, c.table.shape[1] * 16, device=cuda)
        vggt_sparse.paged_weights(q, lse, c.kp, c.table, c.len, c.starts, w, max_new=max_new)
        return torch.isnan(w[0, 0, :100])

    j = torch.arange(100, device=cuda)
    for r in range(60):
        q = c.q.clone()
        q[r] = math.nan
        assert torch.equal(weights(q, lse), j <= 40 + r), r
    at = int(c.table[0, 99 // 16]), 0, 99 % 16, 0
    c.kp[at] = math.inf  # only the last row sees it
    lse[59] = math.inf
    assert torch.equal(weights(c.q, lse), j == 99)


# ------------------------------------------------------------------ eviction
def evicted(w, ids, n, budget, recent):
    """(sources of the slots below the new length, holes, movers) of one head."""
    rank = [math.inf if recent is not None and i >= recent else x for x, i in zip(w, ids)]
    rank = [(-math.inf, 0) if x != x else (x, 1) for x in rank]
    order = sorted(range(n), key=lambda j: (-rank[j][0], -rank[j][1], j))
    keep = min(n, budget)
    kept = set(order[:keep])
    holes = [j for j in range(keep) if j not in kept]
    movers = [j for j in range(keep, n) if j in kept]
    src = list(range(keep))
    for to, of in zip(holes, movers):
        src[to] = of
    return src


EVICT = [  # lengths, budget, heads, dim, page, dtype, layout, recent, kind
    ([1], 1, 1, 64, 16, BF, "hnd", None, "rand"), ([2], 1, 1, 64, 16, BF, "hnd", None, "rand"),
    ([40, 7, 0, 33], 20, 3, 64, 16, BF, "nhd", 5, "rand"),
    ([40, 7, 0, 33], 0, 2, 64, 16, BF, "hnd", None, "rand"),
    ([100, 90], 100, 2, 128, 32, FP, "hnd", 3, "rand"),
    ([1500, 2049], 1024, 2, 128, 64, BF, "both", 100, "rand"),
    ([1500, 2049], 1200, 1, 64, 64, BF, "hnd", None, "ties"),
    ([3000], 17, 2, 64, 128, FP, "hnd", 40, "inf"),  # more recent tokens than room
    ([1100, 64], 700, 2, 64, 16, FP, "hnd", 9, "odd"),
    ([9000], 5000, 1, 64, 256, BF, "hnd", 300, "tiny"),
]


@pytest.mark.parametrize("lengths,budget,heads,dim,page,dtype,layout,recent,kind", EVICT)
def test_evict(cuda, lengths, budget, heads, dim, page, dtype, layout, recent, kind):
    c = Case(cuda, lengths, [0] * len(lengths), heads, 1, dim, page, dtype, layout=layout)
    slots = c.table.shape[1] * page
    g = torch.Generator().manual_seed(budget)
    w = torch.rand(len(lengths), heads, slots, generator=g)
    if kind == "ties":
        w = (w * 3).floor()
    elif kind == "inf":
        w[:, :, ::7] = math.inf
    elif kind == "tiny":  # subnormal, zero, and of close exponents
        w = torch.where(w < 0.3, w * 1e-40, w * 1e-3 + 0.5)
    elif kind == "odd":
        w[:, :, ::3] = math.nan
        w[:, :, 1::5] = -math.inf
        w[:, :, 2::11] *= -1
        w[:, :, 3::13] = -0.0
        w[:, :, 4::13] = 0.0
    ids = torch.argsort(torch.rand(len(lengths), heads, slots, generator=g), -1).to(torch.int32)
    newest = None if recent is None else [n - recent for n in lengths]
    kw = {} if recent is None else dict(recent_from=ints(newest, cuda))
    kp0, vp0 = c.kp.clone(), c.vp.clone()
    got_w, got_i, got_n = vggt_sparse.paged_evict(w.to(cuda), ids.to(cuda), c.kp, c.vp, c.table,
                                                  c.len, budget, status=c.status, **kw)
    assert int(c.status) == 0
    assert got_n.tolist() == [min(n, budget) for n in lengths]
    got_w, got_i = got_w.cpu(), got_i.cpu()
    same = lambda x, y: torch.equal(torch.nan_to_num(x, nan=7.0), torch.nan_to_num(y, nan=7.0))  # noqa: E731
    for b, n in enumerate(lengths):
        for h in range(heads):
            src = evicted(w[b, h, :n].tolist(), ids[b, h, :n].tolist(), n, budget,
                          None if recent is None else newest[b])
            at = torch.tensor(src, dtype=torch.long)
            keep = len(src)
            assert same(got_w[b, h, :keep], w[b, h][at])
            assert torch.equal(got_i[b, h, :keep], ids[b, h][at])
            assert bool((got_w[b, h, keep:] == 0).all()) and bool((got_i[b, h, keep:] == -1).all())
            for to, of in enumerate(src):
                if to != of:
                    pt, po = int(c.table[b, to // page]), int(c.table[b, of // page])
                    kp0[pt, h, to % page] = c.k[b][of, h]
                    vp0[pt, h, to % page] = c.v[b][of, h]
    assert same(kp0, c.kp) and same(vp0, c.vp)


def test_evict_bad_pages(cuda):
    c = Case(cuda, [64], [0], 1, 1, 64, 16)
    w = torch.arange(64, device=cuda, dtype=torch.float32)[None, None].contiguous()
    ids = torch.arange(64, device=cuda, dtype=torch.int32)[None, None].contiguous()
    c.table[0, 3] = 99999
    kp0 = c.kp.clone()
    vggt_sparse.paged_evict(w, ids, c.kp, c.vp, c.table, c.len, 32, status=c.status)
    assert int(c.status) == _lib.STATUS_BAD_PAGE
    third, second = int(c.table[0, 2]), int(c.table[0, 0])
    kp0[second] = kp0[third]
    assert torch.equal(torch.nan_to_num(kp0, nan=7.0), torch.nan_to_num(c.kp, nan=7.0))


# ------------------------------------------------------------------ the parts together
def test_cache_serves_ragged_sequences(cuda):
    """Prompts, decode steps, an eviction and more steps over two sequences,
    grouped heads, causal: each step against plain attention over the tokens
    that the cache says it holds (its ids), with the turned keys in 64 bits."""
    g = torch.Generator().manual_seed(9)
    heads, group, dim = 2, 2, 64
    cache = vggt_sparse.PagedKVCache(2, heads, dim, pages=24, max_length=160, page=16, device=cuda)
    freq, _ = vggt_sparse.rotary_frequencies(dim)
    kept_k, kept_v = [[], []], [[], []]
    free = len(cache._free)
    for step, counts in enumerate(([70, 9], [1, 1], [1, 1], [5, 40], [1, 1], [1, 0], [30, 1])):
        total = sum(counts)
        q, k, v = (torch.randn(total, h, dim, generator=g).to(BF).to(cuda)
                   for h in (heads * group, heads, heads))
        ids = torch.cat([torch.arange(cache.seen[b], cache.seen[b] + n) for b, n in enumerate(counts)])
        ids = ids.to(torch.int32).to(cuda)
        kept = [cache.lengths[b] for b in range(2)]
        cache.append(k, v, counts, frequencies=freq)
        q = vggt_sparse.rotary(q, ids, freq)
        out, _ = cache.attend(q, causal=True)
        turned_k = turned(k, ids, freq, 1.0, "half").to(BF)
        row = 0
        for b, n in enumerate(counts):
            kept_k[b].append(turned_k[row:row + n])
            kept_v[b].append(v[row:row + n])
            all_k, all_v = torch.cat(kept_k[b]), torch.cat(kept_v[b])
            m = cache.lengths[b]
            for h in range(heads * group):
                at = cache.ids[b, h // group, :m].long()
                s = q[row:row + n, h].double() @ all_k[at, h // group].double().T * dim ** -0.5
                limit = kept[b] + torch.arange(n, device=cuda)[:, None]
                s = s.masked_fill(torch.arange(m, device=cuda)[None] > limit, -math.inf)
                p, val = torch.softmax(s, -1), all_v[at, h // group].double()
                # the keys differ by a rounding step from the kernel's own: u per score unit
                bound = U[BF] * (p @ val).abs() + 3 * U[BF] * (p @ val.abs()) + 1e-6
                assert bool(((out[row:row + n, h].double() - p @ val).abs() <= bound).all()), (step, b, h)
            row += n
        if step == 3:
            want = [cache.weights[b, :, :cache.lengths[b]].sum(-1) for b in range(2)]
            cache.evict(50, recent=4)
            assert cache.lengths == [50, 50] and int(cache.length.sum()) == 100
            assert len(cache._free) == free - 2 * 4
            for b in range(2):
                held = cache.ids[b, :, :50]
                for h in range(heads):  # the newest stay, nothing twice, weights move along
                    assert set(range(cache.seen[b] - 4, cache.seen[b])) <= set(held[h].tolist())
                    assert len(set(held[h].tolist())) == 50
                assert bool((cache.weights[b].sum(-1) <= want[b] + 1e-3).all())
            with pytest.raises(ValueError, match="append comes before"):
                cache.attend(q)
    cache.check()
    cache.release(0)
    cache.release(1)
    assert sorted(cache._free) == list(range(24))


def test_streaming_layer_keeps_specials_and_equals_full_attention(cuda):
    """Frames of 5 special and 36 patch tokens.  While nothing is evicted the
    layer is attention over all frames so far; afterwards the specials of every
    frame and the whole last frame are still there."""
    g = torch.Generator().manual_seed(4)
    heads, dim, per, frames = 3, 64, 41, 6
    layer = vggt_sparse.StreamingGlobalLayer(heads, dim, per, 4 * per, page=32, device=cuda)
    yy, xx = torch.meshgrid(torch.arange(6), torch.arange(6), indexing="ij")
    pos = torch.cat((torch.zeros(5, 2), torch.stack((yy.flatten() + 1, xx.flatten() + 1), -1)))
    pos = pos.to(torch.int32).to(cuda)
    keys, vals = [], []
    for f in range(frames):
        q, k, v = (torch.randn(per, heads, dim, generator=g).to(BF).to(cuda) for _ in range(3))
        out = layer(q, k, v, pos)
        keys.append(turned(k, pos, layer.frequencies, 1.0, "half").to(BF).double())
        vals.append(v.double())
        if f < 4:
            tq = turned(q, pos, layer.frequencies, 1.0, "half").to(BF).double()
            s = torch.einsum("nhd,mhd->hnm", tq, torch.cat(keys)) * dim ** -0.5
            p, val = torch.softmax(s, -1), torch.cat(vals)
            want = torch.einsum("hnm,mhd->nhd", p, val)
            mag = torch.einsum("hnm,mhd->nhd", p, val.abs())
            assert bool(((out.double() - want).abs() <= U[BF] * want.abs() + 3 * U[BF] * mag).all())
    layer.cache.check()
    assert layer.cache.lengths == [4 * per]
    for h in range(heads):
        held = set(layer.cache.ids[0, h, :4 * per].tolist())
        assert len(held) == 4 * per
        assert {f * per + i for f in range(frames) for i in range(5)} <= held
        assert set(range((frames - 1) * per, frames * per)) <= held


@pytest.mark.parametrize("new,lengths", [(300, 3000), (1, 3000), (70, 64)])
def test_wait_limit_is_reported(cuda, new, lengths):
    """The self-test switch lets one warp of every CTA wait on a barrier that
    nothing completes; with a limit of 2 ms each CTA gives up through its
    ordinary path, the status says so, and the next calls are right."""
    c = Case(cuda, [lengths], [new], 2, 1, 64, 64)
    w = torch.zeros(1, 2, c.table.shape[1] * 64, device=cuda)

    def weigh(lse):
        vggt_sparse.paged_weights(c.q, lse, c.kp, c.table, c.len, c.starts, w, max_new=new,
                                  status=c.status)
    prev_limit = _lib.set_wait_limit_ns(2_000_000)
    prev_test = _lib.set_wait_selftest(True)
    try:
        for call in (lambda: c.attend(True),
                     lambda: weigh(torch.zeros(new, 2, device=cuda))):
            c.status.zero_()
            call()
            torch.cuda.synchronize()
            assert int(c.status) == _lib.STATUS_TIMEOUT
            with pytest.raises(ValueError, match="timed out"):
                vggt_sparse.check_cache_status(c.status)
    finally:
        _lib.set_wait_selftest(prev_test)
        _lib.set_wait_limit_ns(prev_limit)
    c.status.zero_()
    w.zero_()
    out, lse = c.attend(True)
    c.check(out, lse, True)
    weigh(lse)
    seen = int((lse > -math.inf).sum())
    assert abs(float(w.sum()) - seen) <= 1e-4 * seen
