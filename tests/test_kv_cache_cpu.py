"""The streaming cache without a GPU: the C ABI's declarations and refusals
(argument errors return before any CUDA call), the Python refusals, the
frequencies and the page accounting."""
import math
import os
import re
import shutil
import subprocess

import pytest
import torch

import vggt_sparse
from conftest import REPO

HEADER = os.path.join(REPO, "include", "vggt_cache.h")


@pytest.fixture(scope="module")
def lib():
    from vggt_sparse import _lib, build
    if not os.path.exists(_lib.LIB_PATH) or not os.path.exists(build.BINDING_PATH):
        build.build()
    return _lib.load()


def declared():
    return sorted(set(re.findall(r"^\w[\w\s\*]*?\b(vggt_\w+)\s*\(", open(HEADER).read(), re.M)))


def test_header_and_library_agree(lib):
    from vggt_sparse import _lib
    assert declared() == ["vggt_paged_append", "vggt_paged_attention",
                          "vggt_paged_attention_workspace_size", "vggt_paged_evict",
                          "vggt_paged_evict_workspace_size", "vggt_paged_weights", "vggt_rotary"]
    for name in declared():
        assert hasattr(lib, name) and name in _lib.SIGNATURES


@pytest.mark.parametrize("lang,std", [("c", "-std=c99"), ("c++", "-std=c++17")])
def test_header_compiles_alone(lang, std):
    cc = shutil.which("gcc" if lang == "c" else "g++")
    if cc is None:
        pytest.skip("no host compiler")
    res = subprocess.run([cc, "-fsyntax-only", "-x", lang, std, "-Wall", "-Wextra", "-pedantic",
                          "-Werror", HEADER], capture_output=True, text=True)
    assert res.returncode == 0, res.stderr


def refused(lib, call, cases):
    for bad, text in cases:
        assert call(**bad) < 0, bad
        assert text in lib.vggt_sparse_last_error().decode(), (bad, lib.vggt_sparse_last_error())


def test_rotary_refusals(lib):
    call = lambda **kw: lib.vggt_rotary(*dict(dict(  # noqa: E731
        x=16, dtype=0, tokens=4, heads=2, dim=64, xt=128, xh=64, pos=16, axes=1, freq=16, pairs=32,
        layout=0, lengthen=1.0, inverse=0, out=16, ot=128, oh=64, stream=None), **kw).values())
    refused(lib, call, [
        (dict(dtype=3), "BF16, FP16 or FP32"), (dict(dim=63), "even"), (dict(tokens=-1), "negative"),
        (dict(layout=2), "layout"), (dict(axes=0), "axes"), (dict(axes=5), "axes"),
        (dict(pairs=0), "rotate"), (dict(pairs=33), "rotate"), (dict(axes=2), "rotate"),
        (dict(lengthen=float("inf")), "finite"), (dict(pos=None), "non-NULL"),
        (dict(freq=None), "non-NULL"), (dict(x=None), "non-NULL")])
    assert call(tokens=0) == 0 and call(heads=0) == 0


POOL = dict(pages=4, heads=2, page=16, dim=64, ps=2048, hs=1024, rs=64, table=16, width=2, seqs=1)
BAD_POOL = [
    (dict(dtype=2), "BF16 or FP16"), (dict(dim=96), "head dim"), (dict(page=8), "page size"),
    (dict(page=48), "page size"), (dict(page=2048), "page size"), (dict(heads=0), "kv_heads"),
    (dict(pages=-1), "negative"), (dict(seqs=70000), "too large"), (dict(width=1 << 30), "too large"),
    (dict(rs=60), "strides"), (dict(hs=1020), "strides")]


def test_append_refusals(lib):
    call = lambda **kw: lib.vggt_paged_append(*dict(dict(  # noqa: E731
        k=16, v=16, dtype=0, total=3, kt=128, kh=64, vt=128, vh=64, kp=16, vp=16, **POOL,
        before=16, starts=16, pos=None, axes=0, freq=None, pairs=0, layout=0, lengthen=1.0,
        ids=None, new_ids=None, w=None, nw=None, after=16, status=None, stream=None), **kw).values())
    refused(lib, call, BAD_POOL + [
        (dict(total=-1), "negative"), (dict(k=None), "non-NULL"), (dict(before=None), "non-NULL"),
        (dict(after=None), "non-NULL"), (dict(table=None), "non-NULL"), (dict(ids=16), "new_ids"),
        (dict(pos=16, freq=None, axes=1, pairs=4), "non-NULL"),
        (dict(pos=16, freq=16, axes=1, pairs=40), "rotate")])
    assert call(seqs=0) == 0


def test_attention_refusals(lib):
    call = lambda **kw: lib.vggt_paged_attention(*dict(dict(  # noqa: E731
        q=16, dtype=0, total=3, qt=256, qh=64, kp=16, vp=16, **POOL, lengths=16, starts=16, group=2,
        causal=1, scale=0.1, max_new=3, max_len=20, out=16, ot=256, oh=64, lse=None, status=None,
        ws=16, bytes=1 << 30, stream=None), **kw).values())
    refused(lib, call, BAD_POOL + [
        (dict(group=0), "group"), (dict(group=40000), "group"), (dict(scale=0.0), "scale"),
        (dict(scale=float("nan")), "scale"), (dict(max_new=0), "max_new"),
        (dict(max_len=-1), "max_new"), (dict(q=None), "non-NULL"), (dict(ws=None), "non-NULL"),
        (dict(kp=None), "empty"), (dict(pages=0), "empty"), (dict(q=8), "aligned"),
        (dict(out=24), "aligned"), (dict(kp=40), "aligned"), (dict(qt=260), "multiples of 8"),
        (dict(bytes=100), "workspace")])
    assert call(total=0) == 0 and call(seqs=0) == 0
    size = lib.vggt_paged_attention_workspace_size
    assert size(0, 1, 1, 1, 64, 1, 1) == 0 and size(1, 1, 1, 1, 96, 1, 1) == 0
    for args in ((1, 1, 16, 1, 64, 1, 1375), (32, 32, 8, 4, 128, 1, 32769), (1374, 1, 16, 1, 64, 1374, 43968)):
        assert size(*args) > 16384


def test_weights_refusals(lib):
    call = lambda **kw: lib.vggt_paged_weights(*dict(dict(  # noqa: E731
        q=16, dtype=0, total=3, qt=256, qh=64, lse=16, kp=16, **POOL, lengths=16, starts=16,
        group=2, causal=1, scale=0.1, decay=1.0, max_new=3, max_len=20, w=16, status=None,
        stream=None), **kw).values())
    refused(lib, call, BAD_POOL + [
        (dict(group=0), "group"), (dict(scale=-1.0), "scale"), (dict(decay=float("inf")), "decay"),
        (dict(max_new=0), "max_new"), (dict(lse=None), "non-NULL"), (dict(w=None), "non-NULL"),
        (dict(pages=0), "empty"), (dict(q=20), "aligned"), (dict(qh=4), "multiples of 8")])
    assert call(seqs=0) == 0


def test_evict_refusals(lib):
    call = lambda **kw: lib.vggt_paged_evict(*dict(dict(  # noqa: E731
        w=16, ids=16, dtype=0, kp=16, vp=16, **POOL, lengths=16, budget=10, recent=None,
        max_len=20, w2=32, ids2=32, n2=32, status=None, ws=16, bytes=1 << 20, stream=None),
        **kw).values())
    refused(lib, call, BAD_POOL + [
        (dict(budget=-1), "negative"), (dict(max_len=-1), "negative"), (dict(n2=None), "non-NULL"),
        (dict(w=None), "non-NULL"), (dict(w2=16), "inputs"), (dict(n2=16), "inputs"),
        (dict(kp=24), "aligned"), (dict(bytes=8), "workspace"), (dict(ws=None), "workspace"),
        (dict(seqs=40000), "65535")])
    assert call(seqs=0) == 0
    size = lib.vggt_paged_evict_workspace_size
    assert size(2, 3, 100, 100) == 0 and size(2, 3, 100, 30) == 6 * 30 * 8
    assert size(2, 3, 100, 90) == 6 * 10 * 8


def test_python_refusals():
    x = torch.zeros(4, 8, 64, dtype=torch.bfloat16)
    ints = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    freq, _ = vggt_sparse.rotary_frequencies(64, device="cpu")
    pos = ints(4)
    rot = vggt_sparse.rotary
    for kw, text in ((dict(positions=pos.long()), "positions"), (dict(positions=ints(5)), "positions"),
                     (dict(frequencies=freq.float()), "frequencies"), (dict(layout="both"), "layout"),
                     (dict(x=x.double()), "BF16, FP16 or FP32"), (dict(x=x[0]), "tokens, heads"),
                     (dict(out=x[:2]), "out must"), (dict(x=None), "tensor"), ({}, "CUDA")):
        args = dict(dict(x=x, positions=pos, frequencies=freq), **kw)
        with pytest.raises(ValueError, match=text):
            rot(args.pop("x"), args.pop("positions"), args.pop("frequencies"), **args)

    pool = torch.zeros(6, 2, 16, 64, dtype=torch.bfloat16)
    table, n1, st = ints(1, 3), ints(1), ints(2)
    kv = torch.zeros(4, 2, 64, dtype=torch.bfloat16)
    base = dict(k=kv, v=kv, kp=pool, vp=pool, table=table, before=n1, starts=st)

    def append(**kw):
        a = dict(base, **kw)
        rest = {k: v for k, v in a.items() if k not in base}
        return vggt_sparse.paged_append(*[a[k] for k in base], **rest)
    for kw, text in ((dict(kp=pool.float(), vp=pool.float()), "BF16 or FP16"),
                     (dict(vp=pool[:3]), "same shape"), (dict(kp=pool[0]), "pools must"),
                     (dict(table=table.long()), "table"), (dict(k=kv[:, :1]), "k must"),
                     (dict(v=kv[:2]), "same shape"), (dict(before=ints(2)), "before"),
                     (dict(starts=n1), "starts"), (dict(ids=ints(1, 2, 48)), "new_ids"),
                     (dict(ids=ints(1, 2, 40), new_ids=pos), "ids must"),
                     (dict(weights=torch.zeros(1, 2, 40)), "weights must"),
                     (dict(positions=pos), "frequencies"), (dict(after=n1), "after must not"),
                     (dict(status=torch.zeros(1)), "status"), ({}, "CUDA")):
        with pytest.raises(ValueError, match=text):
            append(**kw)

    def attend(q=x, kp=pool, **kw):
        return vggt_sparse.paged_attention(q, kp, pool, table, n1, st,
                                           **dict(dict(max_new=1), **kw))
    for kw, text in ((dict(q=x[:, :7]), "multiple"), (dict(q=x.half()), "q must"),
                     (dict(out=x[:2]), "out must"), (dict(lse=torch.zeros(4, 2)), "lse must"),
                     (dict(scale="a"), "scale"), (dict(max_new=1.5), "max_new"), ({}, "CUDA")):
        with pytest.raises(ValueError, match=text):
            attend(**kw)

    w, lse = torch.zeros(1, 2, 48), torch.zeros(4, 8)
    for kw, text in ((dict(lse=lse[:2]), "lse must"), (dict(w=w[:, :1]), "weights must"),
                     (dict(q=x[:, :3]), "multiple"), ({}, "CUDA")):
        a = dict(dict(q=x, lse=lse, w=w), **kw)
        with pytest.raises(ValueError, match=text):
            vggt_sparse.paged_weights(a["q"], a["lse"], pool, table, n1, st, a["w"], max_new=1)

    ids = ints(1, 2, 48)
    for kw, text in ((dict(ids=ids.long()), "ids must"), (dict(recent_from=ints(2)), "recent_from"),
                     (dict(out=(w, ids[:, :1], n1)), "out"), (dict(n=ints(3)), "lengths"), ({}, "CUDA")):
        a = dict(dict(ids=ids, n=n1), **kw)
        with pytest.raises(ValueError, match=text):
            vggt_sparse.paged_evict(w, a.pop("ids"), pool, pool, table, a.pop("n"), 10, **a)


def test_missing_binding_fails_loudly(monkeypatch):
    from vggt_sparse import _lib, kv_cache
    monkeypatch.setattr(kv_cache, "_module", None)
    monkeypatch.setattr(kv_cache, "BINDING_PATH", "/nonexistent/_cache_binding.so")
    with pytest.raises(_lib.ExtensionMissing):
        vggt_sparse.rotary(None, None, None)


def test_frequencies():
    f, l = vggt_sparse.rotary_frequencies(8, base=100.0, device="cpu")
    assert l == 1.0 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75]).double())
    f2, _ = vggt_sparse.rotary_frequencies(16, base=100.0, axes=2, device="cpu")
    assert torch.equal(f2, f)
    g, _ = vggt_sparse.rotary_frequencies(8, base=100.0, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(g, f / 4)
    g, _ = vggt_sparse.rotary_frequencies(8, base=100.0, scaling="base", factor=4.0, device="cpu")
    assert g[0] == 1.0 and abs(float(f[3] / g[3]) - 4.0) < 1e-12
    g, l = vggt_sparse.rotary_frequencies(64, scaling="by_parts", factor=16.0, original_length=4096,
                                          device="cpu")
    f, _ = vggt_sparse.rotary_frequencies(64, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32])
    assert torch.allclose(g[turns <= 1], f[turns <= 1] / 16)
    between = (turns > 1) & (turns < 32)
    assert bool(between.any()) and bool(((g < f) & (g > f / 16))[between].all())
    assert abs(l - (0.1 * math.log(16.0) + 1.0)) < 1e-12
    for bad in (dict(rotary_dim=7), dict(rotary_dim=8, axes=3), dict(rotary_dim=8, scaling="other"),
                dict(rotary_dim=8, scaling="by_parts", factor=2.0), dict(rotary_dim=8, factor=0.0)):
        with pytest.raises(ValueError):
            vggt_sparse.rotary_frequencies(device="cpu", **bad)


def test_cache_page_accounting():
    """Page accounting happens on the host, before any operator is called."""
    cache = vggt_sparse.PagedKVCache(2, 1, 64, pages=5, max_length=64, page=16, device="cpu")
    k = torch.zeros(40, 1, 64, dtype=torch.bfloat16)
    for counts, text in (([40], "one number"), ([41, -1], "one number"), ([30, 5], "add up"),):
        with pytest.raises(ValueError, match=text):
            cache.append(k, k, counts)
    with pytest.raises(ValueError, match="max_length"):
        cache.append(torch.zeros(65, 1, 64), None, [65, 0])
    with pytest.raises(ValueError, match="out of pages"):
        cache.append(torch.zeros(82, 1, 64), None, [33, 49])
    assert len(cache._free) == 5
    with pytest.raises(ValueError, match="append comes before"):
        cache.attend(k)
    with pytest.raises(ValueError, match="budget"):
        cache.evict(-1)
    with pytest.raises(ValueError, match="hold a frame"):
        vggt_sparse.StreamingGlobalLayer(2, 64, 100, 99, device="cpu")
