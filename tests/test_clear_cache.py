"""The cache's operators without a GPU: what their entries refuse is decided before any device call, so the addresses are never
dereferenced; the argument structs are the header's."""
import ctypes as C
import re

import pytest

import perseus_amd as pa
from perseus_amd import clear
from perseus_amd._lib import LIB
from tests.test_clear import P, Fake, NoStream, attention_args, fill


@pytest.fixture
def ops():
    return pa.Clear(NoStream, workspace=0)


def header_fields(name):
    """a struct's field names in the header's order, each HeadsRef as three"""
    text = open(pa._lib.HEADER).read()
    end = text.index("} %s;" % name)
    body = re.sub(r"/\*.*?\*/", "", text[text.rindex("typedef struct", 0, end):end], flags=re.S)
    want = []
    for line in body.split("{", 1)[1].split(";"):
        names = re.findall(r"\*?(\w+)(?:\[\d+\])?\s*(?:,|$)", line.strip())
        for n in names:
            want += [n, n + "_token", n + "_head"] if line.strip().startswith("HeadsRef") and "[" not in line else [n]
    return want


def cache_ref(**kw):
    return fill(clear.CacheRef, **{**dict(pages=P, pages_seq=8, width=7, page_rows=16), **kw})


def paged_args(cache=None, **kw):
    a = clear.AttentionPagedArgs()
    a.attention = attention_args(**{**dict(k_start=None), **kw})
    a.cache = cache_ref(**(cache or {}))
    return a


@pytest.mark.parametrize("name", ["CacheRef", "AttentionPagedArgs"])
def test_the_header_s_structs(name):
    assert [f for f, _ in getattr(clear, name)._fields_] == header_fields(name)


@pytest.mark.parametrize("bad,cache,rc", [
    (dict(tokens=-1), {}, -1), (dict(seqs=-1), {}, -1), (dict(k_len=None), {}, -1), (dict(kv_heads=3), {}, -1),
    (dict(type=2), {}, -2), (dict(dim=60), {}, -2), (dict(k_token=129), {}, -2), (dict(k_token=1 << 40), {}, -2),
    (dict(work=P + 4, work_bytes=1024), {}, -2), ({}, dict(pages=None), -1), ({}, dict(width=0), -1), ({}, dict(width=-1), -1),
    ({}, dict(pages_seq=-1), -1), ({}, dict(pages_seq=6), -1), ({}, dict(start=P), -1), ({}, dict(page_rows=8), -2),
    ({}, dict(page_rows=0), -2), ({}, dict(page_rows=-16), -2), ({}, dict(page_rows=48), -2), (dict(tokens=0), {}, 0),
    (dict(seqs=0), dict(pages=None), 0), (dict(seqs=1, tokens=0), dict(pages_seq=0), 0), (dict(heads=0), {}, 0)])
def test_attention_paged_refusals(bad, cache, rc):
    a = paged_args(cache, **bad)
    assert LIB.pcx_attention_paged(C.byref(a), None) == rc
    if rc:
        assert LIB.pcx_attention_paged_workspace(C.byref(a)) == 0
    assert LIB.pcx_attention_paged(None, None) == -1 and LIB.pcx_attention_paged_workspace(None) == 0


def test_attention_paged_s_workspace_is_attention_s():
    kw = dict(seqs=1, tokens=1, max_q=1, max_k=100000, kv_rows=100000)
    want = LIB.pcx_attention_workspace(C.byref(attention_args(**kw)))
    assert want > 0 and LIB.pcx_attention_paged_workspace(C.byref(paged_args(dict(width=9000), **kw))) == want


def test_attention_paged_shapes_are_refused(ops):
    x, kv, q0, kl = Fake((4, 4, 64)), Fake((96, 2, 64)), Fake((3,), "i32"), Fake((2,), "i32")
    good = dict(q=x, k=kv, v=kv, q_start=q0, pages=Fake((2, 5), "i32"), page_rows=16, k_len=kl, out=x)
    for bad in (dict(pages=Fake((3, 5), "i32")), dict(pages=Fake((2, 5), "i64")), dict(pages=Fake((10,), "i32")),
                dict(pages=Fake((2, 5), "i32", strides=(1, 2))), dict(pages=Fake((2, 0), "i32")), dict(page_rows=8),
                dict(page_rows=24), dict(page_rows=0), dict(k=Fake((96, 2, 32))), dict(out=Fake((4, 4, 32))), dict(q_start=kl)):
        with pytest.raises(ValueError):
            ops.attention_paged(**{**good, **bad})


def test_attention_paged_arguments(ops):
    """the packed arguments are the struct's; the longest run expected is at most what a table holds"""
    x, kv = Fake((4, 6, 64)), Fake((96, 2, 64), ptr=P + 64)
    a = ops.attention_paged_args(x, kv, kv, Fake((3,), "i32"), Fake((2, 5), "i32", strides=(8, 1), ptr=P + 16), 32, Fake((2,), "i32"), x)
    assert {n: getattr(a.cache, n) for n, _ in clear.CacheRef._fields_} == dict(start=None, pages=P + 16, pages_seq=8, width=5,
                                                                               page_rows=32)
    assert (a.attention.k_start, a.attention.kv_rows, a.attention.max_k, a.attention.max_q) == (None, 96, 160, 4)
    a = ops.attention_paged_args(x, kv, kv, Fake((3,), "i32"), Fake((2, 5), "i32"), 32, Fake((2,), "i32"), x, max_k=7, max_q=2)
    assert (a.attention.max_k, a.attention.max_q, a.cache.pages_seq) == (7, 2, 5)


@pytest.mark.parametrize("cls,packed", [("EvictArgs", "_EVICT"), ("MoveRowsArgs", "_MOVE_ROWS")])
def test_evict_s_structs(cls, packed):
    """the header's fields, and struct.pack's layout the same: the same bytes give the same fields"""
    assert [f for f, _ in getattr(clear, cls)._fields_] == header_fields(cls)

    def flat(x):
        for n, _ in x._fields_:
            v = getattr(x, n)
            for y in v if hasattr(v, "__len__") else [v]:
                yield from flat(y) if isinstance(y, C.Structure) else [y]

    layout = getattr(clear, packed)
    n = sum(1 for _ in flat(getattr(clear, cls)()))
    assert list(flat(getattr(clear, cls).from_buffer_copy(layout.pack(*range(1, n + 1))))) == list(range(1, n + 1))


def evict_args(cache=None, **kw):
    base = dict(weights=P, weights_token=1, weights_head=200, k_len=P, moves=P, count=P, rows=200, seqs=2, kv_heads=2, keep=8, most=4,
                max_k=50)
    a = fill(clear.EvictArgs, **{**base, **kw})
    a.cache = cache_ref(**(cache or {}))
    return a


@pytest.mark.parametrize("bad,cache,rc", [
    (dict(seqs=-1), {}, -1), (dict(kv_heads=-1), {}, -1), (dict(keep=-1), {}, -1), (dict(recent=-1), {}, -1), (dict(first=-1), {}, -1),
    (dict(most=-1), {}, -1), (dict(max_k=-1), {}, -1), (dict(rows=-1), {}, -1), (dict(k_len=None), {}, -1), (dict(count=None), {}, -1),
    (dict(moves=None), {}, -1), (dict(weights=None), {}, -1), (dict(weights_token=-1), {}, -1), (dict(places=P, places_head=-1), {}, -1),
    (dict(kept_len=P), {}, -1), (dict(recent=8, first=1), {}, -1), (dict(recent=2 ** 31 - 1, first=2 ** 31 - 1), {}, -1),
    ({}, dict(pages=None), -1), ({}, dict(start=P), -1), ({}, dict(width=0), -1), ({}, dict(page_rows=8), -2),
    ({}, dict(page_rows=17), -2), (dict(weights=P + 2), {}, -2), (dict(places=P + 1), {}, -2), (dict(kv_heads=65536), {}, -2),
    (dict(seqs=0), dict(pages=None), 0), (dict(kv_heads=0), {}, 0), (dict(kv_heads=0, weights=None, k_len=None), dict(start=P, pages=None), 0)])
def test_evict_refusals(bad, cache, rc):
    assert LIB.pcx_evict(C.byref(evict_args(cache, **bad)), None) == rc
    assert LIB.pcx_evict(None, None) == -1


def move_args(cache=None, base=P, token=128, head=64, size=2, dim=64, **kw):
    a = fill(clear.MoveRowsArgs, **{**dict(moves=P, count=P, rows=200, tensors=1, seqs=2, kv_heads=2, most=4), **kw})
    a.cache = cache_ref(**(cache or {}))
    a.t[0] = clear.HeadsRef(base, token, head)
    a.size[0], a.dim[0] = size, dim
    return a


@pytest.mark.parametrize("bad,cache,rc", [
    (dict(seqs=-1), {}, -1), (dict(kv_heads=-1), {}, -1), (dict(most=-1), {}, -1), (dict(tensors=-1), {}, -1), (dict(tensors=5), {}, -1),
    (dict(rows=-1), {}, -1), (dict(moves=None), {}, -1), (dict(count=None), {}, -1), (dict(moves=P + 4), {}, -1), (dict(base=None), {}, -1),
    (dict(token=-1), {}, -1), (dict(size=1), {}, -2), (dict(size=3), {}, -2), (dict(dim=0), {}, -2), (dict(dim=2 ** 21), {}, -2),
    (dict(base=P + 1), {}, -2), (dict(token=63), {}, -2), (dict(head=32), {}, -2), (dict(kv_heads=65536), {}, -2),
    ({}, dict(pages=None), -1), ({}, dict(start=P), -1), ({}, dict(page_rows=8), -2), (dict(seqs=0), dict(pages=None), 0),
    (dict(most=0, moves=None), {}, 0), (dict(tensors=0), {}, 0), (dict(kv_heads=0), {}, 0)])
def test_move_rows_refusals(bad, cache, rc):
    assert LIB.pcx_move_rows(C.byref(move_args(cache, **bad)), None) == rc
    assert LIB.pcx_move_rows(None, None) == -1


def test_evict_s_shapes_are_refused(ops):
    w, n, mv, ct = Fake((96, 3), "f32"), Fake((2,), "i32"), Fake((2, 3, 4, 2), "i32"), Fake((2, 3), "i32")
    good = dict(weights=w, k_len=n, keep=8, moves=mv, count=ct, pages=Fake((2, 5), "i32"), page_rows=16)
    for bad in (dict(weights=Fake((96, 3))), dict(weights=Fake((96, 3, 1), "f32")), dict(places=Fake((96, 2), "i32")),
                dict(places=Fake((96, 3), "f32")), dict(moves=Fake((2, 3, 4), "i32")), dict(moves=Fake((2, 2, 4, 2), "i32")),
                dict(moves=Fake((2, 3, 4, 2), "i64")), dict(count=Fake((3, 3), "i32")), dict(k_len=Fake((2,), "i64")), dict(keep=-1),
                dict(recent=5, first=4), dict(recent=-1), dict(next_place=Fake((3,), "i32")), dict(kept_len=Fake((3,), "i32")),
                dict(k_start=Fake((2,), "i64")), dict(pages=None), dict(page_rows=None), dict(pages=None, page_rows=None),
                dict(pages=Fake((3, 5), "i32")), dict(page_rows=20)):
        with pytest.raises(ValueError):
            ops.evict(**{**good, **bad})
    k = Fake((96, 3, 64))
    good = dict(moves=mv, count=ct, tensors=(k, w), pages=Fake((2, 5), "i32"), page_rows=16)
    for bad in (dict(tensors=()), dict(tensors=(k,) * 5), dict(tensors=(k, Fake((95, 3), "f32"))), dict(tensors=(Fake((96, 2, 64)),)),
                dict(tensors=(Fake((96, 3, 64), strides=(384, 128, 2)),)), dict(tensors=(Fake((96,), "f32"),)),
                dict(moves=Fake((2, 3, 4, 1), "i32")), dict(moves=Fake((2, 3, 4, 2), "f32")), dict(count=Fake((2, 2), "i32")),
                dict(k_start=Fake((2,), "i64"))):
        with pytest.raises(ValueError):
            ops.move_rows(**{**good, **bad})


def test_key_weights_s_struct():
    assert [f for f, _ in clear.KeyWeightsArgs._fields_] == header_fields("KeyWeightsArgs")
    names = [f for f, _ in clear.KeyWeightsArgs._fields_]
    a = clear.KeyWeightsArgs.from_buffer_copy(clear._KEY_WEIGHTS.pack(*range(1, 40)))
    got = []
    for n in names:
        got += [getattr(a.cache, x) for x, _ in clear.CacheRef._fields_] if n == "cache" else [getattr(a, n)]
    assert got == list(range(1, 40))


def weights_args(cache=None, **kw):
    base = dict(lse=P, q_start=P, k_len=P, kv_rows=96, tokens=4, seqs=2, heads=4, kv_heads=2, dim=64, causal=1, max_q=2, max_k=50, scale=0.125,
                decay=0.9)
    for r, row, head in (("q", 256, 64), ("k", 128, 64), ("weights", 1, 96), ("before", 1, 96)):
        base.update({r: P, r + "_token": row, r + "_head": head})
    a = fill(clear.KeyWeightsArgs, **{**base, **kw})
    a.cache = cache_ref(**(cache or {}))
    return a


@pytest.mark.parametrize("bad,cache,rc", [
    (dict(tokens=-1), {}, -1), (dict(seqs=-1), {}, -1), (dict(heads=-1), {}, -1), (dict(kv_heads=-1), {}, -1), (dict(kv_rows=-1), {}, -1),
    (dict(max_q=-1), {}, -1), (dict(max_k=-1), {}, -1), (dict(kv_heads=0), {}, -1), (dict(kv_heads=3), {}, -1), (dict(lse=None), {}, -1),
    (dict(q_start=None), {}, -1), (dict(k_len=None), {}, -1), (dict(q=None), {}, -1), (dict(k=None), {}, -1), (dict(weights=None), {}, -1),
    (dict(places=P), {}, -1), (dict(before_token=-1), {}, -1), (dict(places=P, next_place=P, places_head=-1), {}, -1),
    (dict(scale=0.0), {}, -1), (dict(scale=float("nan")), {}, -1), (dict(scale=2.4e38), {}, -1), (dict(decay=-0.5), {}, -1),
    (dict(decay=float("nan")), {}, -1), (dict(decay=float("inf")), {}, -1), ({}, dict(pages=None), -1), ({}, dict(start=P), -1),
    ({}, dict(width=0), -1), ({}, dict(pages_seq=2), -1), ({}, dict(page_rows=8), -2), (dict(type=2), {}, -2), (dict(type=-1), {}, -2),
    (dict(dim=60), {}, -2), (dict(dim=264), {}, -2), (dict(dim=0), {}, -2), (dict(q=P + 8), {}, -2), (dict(k_head=68), {}, -2),
    (dict(q_token=1 << 27), {}, -2), (dict(q_head=1 << 28), {}, -2), (dict(weights=P + 2), {}, -2), (dict(before=P + 1), {}, -2),
    (dict(weights_token=0), {}, -2), (dict(work=P + 4, work_bytes=1 << 20), {}, -2), (dict(heads=65536, kv_heads=65536), {}, -2),
    (dict(tokens=2 ** 30), {}, -2), (dict(seqs=0), dict(pages=None), 0), (dict(heads=0, kv_heads=0), {}, 0)])
def test_key_weights_refusals(bad, cache, rc):
    a = weights_args(cache, **bad)
    assert LIB.pcx_key_weights(C.byref(a), None) == rc
    if rc:
        b = weights_args(cache, **{n: v for n, v in bad.items() if n != "work"})
        assert "work" in bad or LIB.pcx_key_weights_workspace(C.byref(b)) == 0
    assert LIB.pcx_key_weights(None, None) == -1 and LIB.pcx_key_weights_workspace(None) == 0


def test_evict_s_workspace():
    """none for runs of up to 16384 keys, nor for more than 128 (sequence, key head) pairs; a share for each pair else"""
    size = lambda **kw: LIB.pcx_evict_workspace(C.byref(evict_args(**kw)))  # noqa: E731
    assert size(max_k=16384) == size(max_k=20000, seqs=43, kv_heads=3) == size(max_k=20000, seqs=0) == 0
    one, all = size(max_k=16385, seqs=1, kv_heads=1) - 4 * 4096, size(max_k=20000, seqs=64, kv_heads=2) - 4 * 4096
    assert one > 0 and all == 128 * one and LIB.pcx_evict_workspace(None) == 0


def test_key_weights_s_workspace():
    """none for a token; the parts' sums for a prompt, whatever work says"""
    assert LIB.pcx_key_weights_workspace(C.byref(weights_args(max_q=1))) == 0
    a = weights_args(tokens=8192, seqs=1, max_q=8192, max_k=4096, kv_rows=8192, work=3, work_bytes=1)
    n = LIB.pcx_key_weights_workspace(C.byref(a))
    assert n > 4 * 4096 and (n - 4 * 4096) % (2 * 4096 * 4) == 0
    # where no key is expected there is nothing to split
    assert LIB.pcx_key_weights_workspace(C.byref(weights_args(tokens=8192, seqs=1, max_q=8192, max_k=0, kv_rows=8192))) == 0


def test_key_weights_shapes_are_refused(ops):
    q, k, lse, w, n = Fake((4, 4, 64)), Fake((96, 2, 64)), Fake((4, 4), "f32"), Fake((96, 2), "f32"), Fake((2,), "i32")
    good = dict(q=q, k=k, lse=lse, q_start=Fake((3,), "i32"), k_len=n, weights=w, pages=Fake((2, 5), "i32"), page_rows=16)
    for bad in (dict(k=Fake((96, 2, 32))), dict(k=Fake((96, 2, 64), "f16")), dict(q=Fake((4, 4, 64), "i32")), dict(lse=Fake((4, 2), "f32")),
                dict(lse=Fake((4, 4))), dict(weights=Fake((95, 2), "f32")), dict(weights=Fake((96, 2))), dict(before=Fake((96, 4), "f32")),
                dict(places=Fake((96, 2), "i32")), dict(places=Fake((96, 2), "f32"), next_place=n), dict(next_place=Fake((3,), "i32")),
                dict(q_start=n), dict(k_len=Fake((2,), "i64")), dict(k_start=Fake((2,), "i64")), dict(pages=None), dict(page_rows=20)):
        with pytest.raises(ValueError):
            ops.key_weights(**{**good, **bad})
