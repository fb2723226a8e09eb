"""The streaming cache's operators at the edges of their types, layouts and
arguments, on the GPU against plain 64-bit code.  The bounds are those of
test_gpu_kv_cache.py; what a test adds to them it derives where it stands.
"""
import math

import pytest
import torch

import vggt_sparse
from vggt_sparse import _lib
from test_gpu_kv_cache import BF, FP, Case, ints, turned

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ attention
@pytest.mark.parametrize("where", [0, 11990])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [1, 70])
def test_attention_keeps_the_tail_in_fp16(cuda, new, dim, where):
    """One key 17.6 nats (2^25.4) above 12,000 others, with values of zero: the
    output is what the others add up to.  A probability goes to the product
    with V in fp16, shifted by 2^15 (single tokens) or 2^7 against a reference
    that may lie 2^8 low: within the type's rounding, or half its least step."""
    c = Case(cuda, [12000], [new], 1, 1, dim, 64, FP)
    weak, strong = 0.5, 18.125
    page = c.table[0, torch.arange(12000, device=cuda) // 64].long()
    row = torch.arange(12000, device=cuda) % 64
    k = torch.zeros(12000, 1, dim, device=cuda, dtype=FP)
    k[:, :, 0] = weak
    k[where, :, 0] = strong
    v = (torch.rand(12000, 1, dim, generator=torch.Generator().manual_seed(1)) + 0.5).to(FP).to(cuda)
    v[where] = 0
    c.kp[page, :, row], c.vp[page, :, row] = k, v
    c.q.zero_()
    c.q[:, :, 0] = 1
    out, lse = c.attend(True, scale=1.0)
    for i in range(new):
        n = 12000 - new + i + 1
        sees = where < n
        s = k[:n, 0, 0].double()
        want_l = torch.logsumexp(s, 0)
        p = torch.exp(s - want_l)
        want = p @ v[:n, 0].double()
        step = 2.0 ** -(25 + (15 if new == 1 else 7)) * 1.5 * n if sees else 0.0
        bound = (2 * 2.0 ** -11 + 2.0 ** -13) * want + step
        err = (out[i, 0].double() - want).abs()
        assert bool((err <= bound).all()), (i, float((err / want).max()))
        assert abs(float(lse[i, 0]) - float(want_l)) <= 2.0 ** -16 + 2.0 ** -20 * strong


def test_attention_of_scores_beyond_fp16(cuda):
    """Scores of 10^8, whose exponents fp32 holds to several units: the shifted
    probabilities stay within the type, and the largest scores (exact in fp32,
    the next ones 960,000 below) share the row."""
    for new in (1, 70):
        c = Case(cuda, [300], [new], 1, 1, 64, 16, FP)
        c.q.zero_()
        c.q[..., 0] = 30000
        at = torch.arange(300, device=cuda)
        c.kp[c.table[0, at // 16].long(), :, at % 16] = 0
        c.kp[c.table[0, at // 16].long(), 0, at % 16, 0] = (4 * (at % 97) + 10).to(FP)
        out, lse = c.attend(False, scale=8.0)
        top = [j for j in range(300) if j % 97 == 96]
        want = c.v[0][top, 0].double().mean(0)
        assert bool(((out[:, 0].double() - want).abs() <= 2.0 ** -10 * want.abs() + 2.0 ** -10 * 4).all())
        assert torch.isfinite(lse).all()


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new", [5, 200])
def test_attention_large_values_of_later_tokens(cuda, new, dim):
    """Values of 1e38 (bf16) in the chunk's later tokens, in every column of a
    tile: rows that do not see them are the same bits as with zeros there."""
    c = Case(cuda, [450, 200], [new, new], 1, 2, dim, 16, BF)
    first = new // 2
    at = torch.arange(450 - new + first, 450, device=cuda)
    page = c.table[0, at // 16].long()
    c.vp[page, :, at % 16] = 0
    want, want_lse = c.attend(True)
    c.vp[page, :, at % 16] = 1e38
    out, lse = c.attend(True)
    assert torch.equal(out[:first], want[:first]) and torch.equal(lse[:first], want_lse[:first])
    assert torch.equal(out[new:], want[new:])
    assert bool((out[first:new].abs() > 1e30).all())


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,length", [(5, 450), (200, 450), (200, 3000)])
def test_attention_values_of_later_tokens_that_are_not_finite(cuda, new, length, dim, bad):
    """bf16: one such value in the chunk, in one run of the keys or in the last of
    several.  Rows that see it get it, the others are as if it were zero."""
    c = Case(cuda, [length, 70], [new, new], 1, 2, dim, 16)
    first = new // 2
    j = length - new + first
    at = int(c.table[0, j // 16]), 0, j % 16, 9
    c.vp[at] = 0
    want, want_lse = c.attend(True)
    c.vp[at] = bad
    out, lse = c.attend(True)
    assert torch.equal(out[new:], want[new:]) and torch.equal(lse[new:], want_lse[new:])
    seen = out[first:new, :, 9]
    assert bool(torch.isnan(seen).all()) if bad != bad else bool((seen == bad).all())
    others = torch.ones_like(out[:new], dtype=torch.bool)
    others[first:, :, 9] = False
    # both sides round the probabilities (or not) and the output: two bounds apart
    size = 4 * c.v[0].abs().max().double()
    diff = (out[:new].double() - want[:new].double()).abs()[others]
    assert bool((diff <= 2 * (2 * 2.0 ** -8 + 2.0 ** -13) * size).all())
    assert bool(((lse[:new] - want_lse[:new]).abs() <= 2.0 ** -14).all())


# ------------------------------------------------------------------ weights
@pytest.mark.parametrize("decay", [0.0, 0.5, -1.0])
@pytest.mark.parametrize("max_new", [1, 500])
def test_weights_of_infinity_stay(cuda, max_new, decay):
    """+inf keeps a token from eviction whatever the decay, in a sequence
    without new tokens too and where the token's key is NaN; the other weights
    are decay * weight + sum as ever."""
    c = Case(cuda, [300, 40], [60, 0], 2, 1, 64, 16)
    out, lse = c.attend(True)
    w0 = torch.rand(2, 2, c.table.shape[1] * 16, device=cuda)
    w0[:, :, 1:300:7] = math.inf
    c.kp[int(c.table[0, 0]), :, 8] = math.nan
    w = w0.clone()
    vggt_sparse.paged_weights(c.q, lse, c.kp, c.table, c.len, c.starts, w, max_new=max_new,
                              decay=decay, status=c.status)
    added = torch.zeros_like(w0)
    vggt_sparse.paged_weights(c.q, lse, c.kp, c.table, c.len, c.starts, added, max_new=max_new)
    pinned = w0 == math.inf
    assert bool((w[pinned] == math.inf).all()) and int(c.status) == 0
    for b, n in enumerate(c.lengths):
        want = (w0[b, :, :n] * decay + added[b, :, :n])[~pinned[b, :, :n]]
        got = w[b, :, :n][~pinned[b, :, :n]]
        assert bool(((got - want).abs() <= 2.0 ** -22 * (1 + added.nan_to_num().max())).all())
    ids = torch.arange(w.shape[2], device=cuda, dtype=torch.int32).expand(2, 2, -1).contiguous()
    _, kept, n = vggt_sparse.paged_evict(w, ids, c.kp, c.vp, c.table, c.len, 50)
    assert n.tolist() == [50, 40]
    for h in range(2):
        assert set(range(1, 300, 7)) <= set(kept[0, h, :50].tolist())


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("max_new", [1, 500])
@pytest.mark.parametrize("new,group", [(1, 1), (2, 7), (40, 7), (90, 3), (70, 65), (17, 1)])
def test_weights_of_keys_that_nobody_looks_at(cuda, new, group, max_new, causal):
    """Keys with an infinite element whose scores are all -inf receive nothing,
    whatever fills up the tiles of rows: their weights stay, and the others are
    what they are without such keys."""
    c = Case(cuda, [300], [new], 1, group, 64, 16)
    c.q[..., 5] = -(c.q[..., 5].abs() + 0.5)
    at = torch.arange(0, 300, 3, device=cuda)
    where = c.table[0, at // 16].long(), 0, at % 16, 5
    c.kp[where] = 1e4  # scores of -600 and less: exponentials of zero
    out, lse = c.attend(causal)

    def weights():
        w = torch.full((1, 1, c.table.shape[1] * 16), 0.25, device=cuda)
        return vggt_sparse.paged_weights(c.q, lse, c.kp, c.table, c.len, c.starts, w,
                                         max_new=max_new, causal=causal, status=c.status)[0, 0]
    want = weights()
    assert bool((want[at] == 0.25).all())
    c.kp[where] = math.inf
    assert torch.equal(weights(), want) and int(c.status) == 0


# ------------------------------------------------------------------ the streaming layer
@pytest.mark.parametrize("budget,special", [(41, 5), (50, 5), (60, 5), (82, 5), (70, 0), (45, 1)])
def test_streaming_layer_keeps_what_it_promises(cuda, budget, special):
    """Streams far past the point where the special tokens of all frames no
    longer fit: after each frame the cache holds the whole frame and the special
    tokens of the first frames, as many as there is room for."""
    g = torch.Generator().manual_seed(budget)
    per = 41
    layer = vggt_sparse.StreamingGlobalLayer(2, 64, per, budget, special=special, page=16, device=cuda)
    pos = torch.arange(2 * per).reshape(per, 2).to(torch.int32).to(cuda)
    pinned = (budget - per) // special if special else 0
    for f in range(pinned + 8):
        layer(*(torch.randn(per, 2, 64, generator=g).to(BF).to(cuda) for _ in range(3)), pos)
        n = layer.cache.lengths[0]
        assert n == min(budget, (f + 1) * per)
        for h in range(2):
            held = set(layer.cache.ids[0, h, :n].tolist())
            assert len(held) == n
            assert set(range(f * per, (f + 1) * per)) <= held, f
            assert {e * per + i for e in range(min(f + 1, pinned)) for i in range(special)} <= held, f
    layer.cache.check()
    assert layer.pinned_frames == pinned


# ------------------------------------------------------------------ arguments
@pytest.mark.parametrize("new,heads,group", [(1, 2, 2), (1, 1, 1), (20, 1, 1), (60, 2, 2)])
def test_rows_of_any_stride_and_address(cuda, new, heads, group):
    """q as a contiguous tensor that is not 16-byte aligned, with an odd stride
    of its one token or its one head, and with a strided last dimension: copied
    where need be, the same bits.  So are outputs of one token or head."""
    c = Case(cuda, [200], [new], heads, group, 64, 16)
    n, h, d = c.q.shape
    out, lse = c.attend(True)

    def weights(q):
        w = torch.zeros(1, heads, c.table.shape[1] * 16, device=cuda)
        return vggt_sparse.paged_weights(q, lse, c.kp, c.table, c.len, c.starts, w, max_new=new)
    want_w, q0 = weights(c.q), c.q
    shifted = torch.empty(q0.numel() + 1, device=cuda, dtype=BF)[1:].view(n, h, d)
    wide = torch.empty(n, h * d + 5, device=cuda, dtype=BF)[:, :h * d].unflatten(1, (h, d))
    odd = torch.empty(n, h, d + 3, device=cuda, dtype=BF)[:, :, :d]
    apart = torch.empty(n, h, d, 2, device=cuda, dtype=BF)[..., 0]
    for q in (shifted, wide, odd, apart):
        q.copy_(q0)
        c.q = q
        got, got_lse = c.attend(True)
        assert torch.equal(got, out) and torch.equal(got_lse, lse)
        assert torch.equal(weights(q), want_w)
    c.q = q0
    if n == 1:
        o = torch.empty(1, h * d + 5, device=cuda, dtype=BF)[:, :h * d].unflatten(1, (h, d))
        assert torch.equal(c.attend(True, out=o)[0], out) and torch.equal(o, out)
    if h == 1:
        o = torch.empty(n, d, 1, device=cuda, dtype=BF).transpose(1, 2)
        o = o.as_strided((n, 1, d), (d, 3, 1))
        assert torch.equal(c.attend(True, out=o)[0], out) and torch.equal(o, out)
    for k in (shifted, wide) if group == 1 else ():
        kp, vp = c.kp.clone(), c.vp.clone()
        vggt_sparse.paged_append(q0, q0, c.kp, c.vp, c.table, c.len - new, c.starts)
        vggt_sparse.paged_append(k, k, kp, vp, c.table, c.len - new, c.starts)
        same = lambda x, y: torch.equal(x.nan_to_num(7.0), y.nan_to_num(7.0))  # noqa: E731
        assert same(kp, c.kp) and same(vp, c.vp)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("new,length", [(1, 70), (3, 5000), (90, 300), (90, 5000)])
def test_attention_rows_of_no_sequence(cuda, new, length, dim):
    """Rows before the first start and behind the last one give zeros and -inf
    and set a status bit; those of the sequences are what they are alone."""
    c = Case(cuda, [length, length // 2], [new, new], 1, 2, dim, 16)
    out, lse = c.attend(True)
    c.check(out, lse, True)
    q = torch.randn(2 * new + 5, 2, dim, device=cuda).to(BF)
    q[3:-2] = c.q
    o, l = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=cuda)
    vggt_sparse.paged_attention(q, c.kp, c.vp, c.table, c.len, c.starts + 3, max_new=new, out=o,
                                lse=l, status=c.status)
    assert int(c.status) == _lib.STATUS_BAD_LENGTH
    rest = torch.tensor([0, 1, 2, 2 * new + 3, 2 * new + 4], device=cuda)
    assert bool((o[rest] == 0).all()) and bool((l[rest] == -math.inf).all())
    # the split goes by the rows, so that sums may be cut elsewhere
    c.status.zero_()
    c.check(o[3:-2], l[3:-2], True)
    o, l = vggt_sparse.paged_attention(q, c.kp, c.vp, c.table, c.len, torch.zeros_like(c.starts),
                                       max_new=new, status=c.status)
    assert bool((o == 0).all()) and bool((l == -math.inf).all())
    assert int(c.status) == _lib.STATUS_BAD_LENGTH
    c.status.zero_()
    word = torch.zeros(4, dtype=torch.int32, device=cuda)[::2]
    o, l = vggt_sparse.paged_attention(q, c.kp, c.vp, c.table[:0], c.len[:0], c.starts[:1],
                                       max_new=new, out=torch.full_like(q, 7.0), status=word)
    assert bool((o == 0).all()) and bool((l == -math.inf).all())
    assert word.tolist() == [_lib.STATUS_BAD_LENGTH, 0]


# ------------------------------------------------------------------ gradients
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, BF])
def test_rotary_in_a_graph(cuda, dtype, inverse, layout):
    """The gradient of a weighted sum against the formula's, in place too."""
    g = torch.Generator().manual_seed(2)
    x, y = (torch.randn(9, 3, 64, generator=g).to(dtype).to(cuda) for _ in range(2))
    pos = torch.randint(0, 4000, (9, 2), generator=g).to(torch.int32).to(cuda)
    freq, lengthen = vggt_sparse.rotary_frequencies(48, axes=2, scaling="by_parts", factor=8.0,
                                                    original_length=512)
    kw = dict(layout=layout, lengthen=lengthen, inverse=inverse)
    want = turned(y, pos, freq, lengthen, layout, not inverse)
    u = {torch.float32: 2.0 ** -24, BF: 2.0 ** -8}[dtype]
    bound = u * want.abs() + 2.0 ** -20 * 1.5 * lengthen * y.double().abs().amax(-1, keepdim=True)
    for form in ("out", "in place", "other out", "strided gradient"):
        leaf = x.clone().requires_grad_()
        z = leaf * 1
        if form == "out":
            r = vggt_sparse.rotary(z, pos, freq, **kw)
        else:
            into = z if form == "in place" else torch.empty_like(x)
            r = vggt_sparse.rotary(z, pos, freq, out=into, **kw)
            assert r.data_ptr() == into.data_ptr()
        assert r.requires_grad
        assert torch.equal(r.detach(), vggt_sparse.rotary(x, pos, freq, **kw))
        if form == "strided gradient":
            r.backward(y.transpose(1, 2).contiguous().transpose(1, 2))
        else:
            (r * y).sum().backward()
        assert bool(((leaf.grad.double() - want).abs() <= bound).all()), form
    with torch.no_grad():
        assert not vggt_sparse.rotary(leaf, pos, freq, **kw).requires_grad


@pytest.mark.parametrize("new", [1, 40])
def test_attention_says_that_it_has_no_gradient(cuda, new):
    """Inputs that require gradients give the same numbers, with a graph whose
    backward pass raises instead of none."""
    c = Case(cuda, [200], [new], 1, 2, 64, 16)
    out, lse = c.attend(True)
    leaf = c.q.clone().requires_grad_()
    c.q = leaf * 1
    for kw in ({}, dict(out=torch.empty_like(out), lse=torch.empty_like(lse))):
        got, got_lse = c.attend(True, **kw)
        assert torch.equal(got, out) and torch.equal(got_lse, lse)
        for t in (got, got_lse):
            assert t.requires_grad
            with pytest.raises(RuntimeError, match="no gradient"):
                t.sum().backward()
        if kw:
            assert got.data_ptr() == kw["out"].data_ptr()
    w = torch.zeros(1, 1, c.table.shape[1] * 16, device=cuda)
    vggt_sparse.paged_weights(c.q, got_lse, c.kp, c.table, c.len, c.starts, w, max_new=new)
    assert not w.requires_grad and abs(float(w.sum()) - 2 * new) <= 1e-4 * new
    with torch.no_grad():
        assert not c.attend(True)[0].requires_grad


# ------------------------------------------------------------------ expectations
HINTS = [(1, 1), (1, 2 ** 62), (2 ** 62, 1), (2 ** 62, 2 ** 62), (2 ** 63 - 1, 2 ** 63 - 1), (40, 300)]


@pytest.mark.parametrize("max_new,max_len", HINTS)
@pytest.mark.parametrize("new", [1, 40])
def test_attention_and_weights_hold_for_any_expectation(cuda, new, max_new, max_len):
    """Many sequences and heads (132 of them), and hints from far too low to
    far too high: the same weights but for the order of sums."""
    c = Case(cuda, [33 * b + 60 for b in range(11)], [new] * 11, 12, 1, 64, 16)
    out, lse = c.attend(True, max_new=max_new, max_len=max_len)
    c.check(out, lse, True)
    w = torch.zeros(11, 12, c.table.shape[1] * 16, device=cuda)
    vggt_sparse.paged_weights(c.q, lse, c.kp, c.table, c.len, c.starts, w, max_new=max_new,
                              max_len=max_len, status=c.status)
    assert int(c.status) == 0
    for b, n in enumerate(c.lengths):
        s, _ = c.scores(b, True)
        p = torch.exp(s - lse[c.rows(b)].T[..., None].double())
        bound = (2e-5 + new * 2.0 ** -24) * p.sum(1) + 2.0 ** -23 * p.sum(1)
        assert bool(((w[b, :, :n].double() - p.sum(1)).abs() <= bound).all())
        assert bool((w[b, :, n:] == 0).all())


@pytest.mark.parametrize("max_len", [0, 40, 500, 3000, 2 ** 62])
@pytest.mark.parametrize("dim", [64, 128])
def test_evict_holds_for_any_expectation(cuda, dim, max_len):
    """max_len below the lengths (the shares do not fit what was set aside for
    them, and are read again) and above: the same choice, the same bits."""
    c = Case(cuda, [2900, 700], [0, 0], 2, 1, dim, 16)
    g = torch.Generator().manual_seed(3)
    w = (torch.rand(2, 2, c.table.shape[1] * 16, generator=g) * 50).floor().to(cuda)
    ids = torch.arange(w.shape[2], dtype=torch.int32, device=cuda).expand(2, 2, -1).contiguous()
    recent = ints([2800, 650], cuda)
    kp, vp = c.kp.clone(), c.vp.clone()
    want = vggt_sparse.paged_evict(w, ids, kp, vp, c.table, c.len, 600, recent_from=recent)
    got = vggt_sparse.paged_evict(w, ids, c.kp, c.vp, c.table, c.len, 600, max_len=max_len,
                                  recent_from=recent, status=c.status)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(c.status) == 0
    assert torch.equal(kp.nan_to_num(7.0), c.kp.nan_to_num(7.0))
    assert torch.equal(vp.nan_to_num(7.0), c.vp.nan_to_num(7.0))
    rank = torch.where(ids[0] >= 2800, math.inf, w[0])[:, :2900]
    keep = torch.sort(rank, dim=-1, descending=True, stable=True).indices[:, :600]
    for h in range(2):
        assert set(got[1][0, h, :600].tolist()) == set(keep[h].tolist())
