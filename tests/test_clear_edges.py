"""The ends of the clear side's ranges without a GPU: what its entries refuse there is decided before any device call, so the
addresses are never dereferenced."""
import ctypes as C

import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import attention, clear
from perseus_amd._lib import LIB
from tests.test_clear import Fake, NoStream, attention_args


@pytest.mark.parametrize("tokens,heads,kv", [(2 ** 31 - 1, 1, 1), (2 ** 31 - 127, 1, 1), (2 ** 28, 8, 2), (2 ** 29 - 31, 4, 1)])
def test_attention_refuses_rows_near_2_31(tokens, heads, kv):
    """a tile of 128 rows that ends past 2^31 - 1"""
    a = attention_args(tokens=tokens, heads=heads, kv_heads=kv, q_token=64 * heads, out_token=64 * heads)
    assert LIB.pcx_attention(C.byref(a), None) == -2
    assert LIB.pcx_attention_workspace(C.byref(a)) == 0


@pytest.mark.parametrize("bad", [
    dict(seqs=2 ** 31 - 1), dict(seqs=2 ** 31 - 65535), dict(seqs=2 ** 31 - 2 ** 25, tokens=2 ** 29, heads=2, kv_heads=1, q_token=128, out_token=128),
    dict(heads=2 ** 23, kv_heads=2 ** 23, q_token=2 ** 29, out_token=2 ** 29, k_token=2 ** 22, k_head=0, v_token=2 ** 22, v_head=0)])
def test_attention_refuses_what_no_grid_holds(bad):
    """more (sequence, tile) pairs than 31 bits number, more key heads than 32 bits of threads take"""
    a = attention_args(**bad)
    assert LIB.pcx_attention(C.byref(a), None) == -2
    assert LIB.pcx_attention_workspace(C.byref(a)) == 0


@pytest.mark.parametrize("work", [1, 4, 2 ** 20 + 8])
def test_the_workspace_query_reads_no_workspace(work):
    """its bytes for a struct whose work is not set yet; the call itself refuses a workspace that is not aligned"""
    kw = dict(seqs=1, tokens=1, max_q=1, max_k=100000, kv_rows=100000)
    want = LIB.pcx_attention_workspace(C.byref(attention_args(**kw)))
    assert want > 0
    a = attention_args(work=work, work_bytes=12345, **kw)
    assert LIB.pcx_attention_workspace(C.byref(a)) == want
    assert LIB.pcx_attention(C.byref(a), None) == -2


@pytest.mark.parametrize("one", [
    dict(tokens=1, q_token=129, out_token=3), dict(kv_rows=1, k_token=2 ** 40, v_token=1),
    dict(heads=1, kv_heads=1, q_head=5, out_head=2 ** 41, k_head=2 ** 30 + 3, v_head=1),
    dict(heads=2, kv_heads=1, k_head=7, v_head=9)])
def test_strides_of_single_rows_are_not_refused(one):
    """a stride that no address is made with: the workspace query answers as for a dense tensor"""
    many = dict(tokens=2, seqs=1, max_q=1, max_k=100000, kv_rows=100000)
    shape = {n: x for n, x in one.items() if n in ("tokens", "heads", "kv_heads", "kv_rows")}
    want = LIB.pcx_attention_workspace(C.byref(attention_args(**{**many, **shape})))
    assert want > 0
    assert LIB.pcx_attention_workspace(C.byref(attention_args(**{**many, **one}))) == want
    for n in one:  # and still refused where there is a second row
        if n not in shape:
            assert LIB.pcx_attention(C.byref(attention_args(**{n: one[n] * 2 + 1})), None) == -2


@pytest.mark.parametrize("scale", [2.4e38, 2.9e38, 3e38])
def test_attention_refuses_a_scale_that_leaves_f32(scale):
    """scores are taken in powers of two: the scale times log2(e) has to be finite too"""
    assert LIB.pcx_attention(C.byref(attention_args(scale=scale)), None) == -1
    assert LIB.pcx_attention(C.byref(attention_args(scale=2.3e38, tokens=0)), None) == 0


class HostBuf:
    """a buffer of no memory, for arrays that are never read"""

    def __init__(self, words):
        self.words, self.ptr = int(words), C.c_void_p(1 << 20)

    def upload(self, a, stream=None, offset=0):
        assert offset + a.size <= self.words


@pytest.mark.parametrize("bad", [
    dict(dtype="f32"), dict(dtype="i32"), dict(dim=60), dict(dim=264), dict(dim=0), dict(heads=5), dict(heads=0, kv_heads=0),
    dict(kv_heads=0), dict(capacity=0), dict(layout="other"), dict(table=Fake((9, 32, 2), "f32")),
    dict(table=Fake((10, 33, 2), "f32")), dict(table=Fake((10, 64), "f32")), dict(table=Fake((10, 32, 2), "f16")),
    dict(q_weight=Fake((32,), "f32")), dict(k_weight=Fake((64,), "bf16"))])
def test_a_block_that_no_token_could_enter_is_refused(monkeypatch, bad):
    """when it is made: a table with fewer places than the block holds tokens would put NaN into the cache, a type or width that
    attention refuses would fail after the cache was written"""
    monkeypatch.setattr(clear, "DevBuf", HostBuf)
    good = dict(heads=4, kv_heads=2, dim=64, capacity=10, dtype="f16", table=Fake((10, 32, 2), "f32"))
    ops = pa.Clear(NoStream, workspace=0)
    block = attention.ClearBlock(ops, **good)
    assert block.length == 0 and block.k.shape == (10, 2, 64) and block.out.shape == (10, 4, 64)
    attention.ClearBlock(ops, **{**good, "table": None})
    with pytest.raises(ValueError):
        attention.ClearBlock(ops, **{**good, **bad})


def test_a_failed_append_leaves_the_block_s_length(monkeypatch):
    """a caller that tries again appends the same tokens at the same places"""
    monkeypatch.setattr(clear, "DevBuf", HostBuf)
    calls = []

    class Ops:
        stream = NoStream

        def qk_norm_rotary(self, *args, slots, **kw):
            calls.append(slots.offset)

        def attention(self, *args, max_k, **kw):
            calls.append(max_k)
            if len(calls) == 4:
                raise pa.HipError("attention")

    class Rows(Fake):
        def __getitem__(self, at):
            return self

    block, rows = attention.ClearBlock(Ops(), 4, 2, 64, 10), Rows((3, 8, 64))
    block.append(rows)
    with pytest.raises(pa.HipError):
        block.append(rows)
    assert block.length == 3
    block.append(rows)
    assert block.length == 6 and calls == [0, 3, 6, 6, 6, 6]


@pytest.mark.parametrize("kind,want", [("u1", "i32"), ("u2", "i32"), ("u4", "i64"), ("u8", "i64"), ("i1", "i32"), ("i4", "i32"), ("i8", "i64")])
def test_host_integers_stay_integers(monkeypatch, kind, want):
    """unsigned ones too, in a type that holds them"""
    got = []

    class Buf(HostBuf):
        def upload(self, a, stream=None, offset=0):
            got.append(a.copy())

    monkeypatch.setattr(clear, "DevBuf", Buf)
    x = np.array([0, 1, np.iinfo(kind).max if kind != "u8" else 2 ** 63 - 1, 77], kind)
    a = pa.Array.of(x)
    assert a.dtype == want
    assert (got[0].view({"i32": np.int32, "i64": np.int64}[want])[:4] == x.astype(np.int64)).all()
