"""The clear side without a GPU: the refusals of its entries (decided before any device call; the addresses are never
dereferenced), the rotation tables, the bfloat16 conversions, the argument structs."""
import ctypes as C
import math

import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import clear
from perseus_amd._lib import LIB


class Fake:
    """a tensor of addresses only"""
    is_cuda = True

    def __init__(self, shape, dtype="bf16", strides=None, ptr=1 << 20):
        self.shape, self.dtype, self._p = tuple(shape), dtype, ptr
        if strides is None:
            strides = [math.prod(self.shape[i + 1:]) for i in range(len(self.shape))]
        self._s = tuple(strides)

    def data_ptr(self):
        return self._p

    def stride(self):
        return self._s

    def numel(self):
        return math.prod(self.shape)

    def is_contiguous(self):
        return self._s == tuple(math.prod(self.shape[i + 1:]) for i in range(len(self.shape)))


class NoStream:
    h = None


@pytest.fixture
def ops():
    return pa.Clear(NoStream, workspace=0)


def test_bf16_rounds_to_nearest_even():
    x = np.array([1.0, -2.5, 0.0, -0.0, 1 + 2 ** -8, 1 + 3 * 2 ** -8, 1 + 2 ** -8 + 2 ** -20, np.inf, -np.inf, 3.4e38, 1e-40], np.float32)
    want = np.array([1.0, -2.5, 0.0, -0.0, 1.0, 1 + 2 ** -6, 1 + 2 ** -7, np.inf, -np.inf, np.inf, np.nan], np.float32)
    got = clear.from_bf16(clear.to_bf16(x))
    assert (got[:-1] == want[:-1]).all() and abs(got[-1] - 1e-40) < 2.0 ** -134
    assert np.signbit(got[3])
    assert np.isnan(clear.from_bf16(clear.to_bf16(np.float32([np.nan, -np.nan])))).all()


def test_rotation_tables():
    r = clear.rotary_rates(64)
    assert r.shape == (32,) and r[0] == 1 and abs(r[16] - 0.01) < 1e-15
    assert np.allclose(clear.rotary_rates(64, scaling=("linear", 4)), r / 4, rtol=1e-15)
    b = clear.rotary_rates(64, scaling=("base", 8))
    assert b[0] == 1 and abs(b[-1] / r[-1] - 1 / 8) < 1e-12
    t = clear.rotary_rates(64, scaling=("by_turns", 8, 2048, 1, 4))
    turns = 2048 * r / (2 * np.pi)
    assert (t[turns > 4] == r[turns > 4]).all() and np.allclose(t[turns < 1], r[turns < 1] / 8)
    mid = (turns > 1) & (turns < 4)
    assert mid.any() and ((t[mid] < r[mid]) & (t[mid] > r[mid] / 8)).all()
    tab = clear.rotary_table(100, 8, magnitude=2.0)
    assert tab.shape == (100, 4, 2) and tab.dtype == np.float32
    assert np.abs((tab.astype(np.float64) ** 2).sum(-1) - 4).max() < 1e-6
    for bad in (dict(rot=7), dict(rot=0), dict(rot=8, scaling=("linear", 0)), dict(rot=2, scaling=("base", 2)),
                dict(rot=8, scaling=("by_turns", 8, 2048, 4, 1)), dict(rot=8, scaling=("other", 2))):
        with pytest.raises(ValueError):
            clear.rotary_rates(**bad)


def test_shapes_and_types_are_refused(ops):
    x, pos, tab = Fake((4, 2, 64)), Fake((4,), "i32"), Fake((10, 32, 2), "f32")
    for args, kw in [
            ((Fake((4, 128)), pos, tab, x), {}), ((x, pos, tab, Fake((4, 2, 32))), {}), ((x, pos, tab, Fake((4, 2, 64), "f16")), {}),
            ((x, Fake((3,), "i32"), tab, x), {}), ((x, Fake((4,), "i64"), tab, x), {}), ((x, pos, Fake((10, 64), "f32"), x), {}),
            ((x, pos, Fake((10, 32, 2), "bf16"), x), {}), ((x, pos, tab, x), dict(layout="other")),
            ((Fake((4, 2, 64), strides=(256, 128, 2)), pos, tab, x), {}), ((Fake((4, 2, 64), "i32"), pos, tab, x), {})]:
        with pytest.raises(ValueError):
            ops.rotary(*args, **kw)
    off = Fake((4, 2, 64))
    off.is_cuda = False
    with pytest.raises(ValueError):
        ops.rotary(off, pos, tab, x)
    w = Fake((64,), "f32")
    good = dict(q=x, k=Fake((4, 1, 64)), q_weight=w, k_weight=w, positions=pos, table=tab, q_out=x, k_out=Fake((4, 1, 64)))
    for bad in (dict(k=Fake((3, 1, 64))), dict(k_out=Fake((5, 1, 64))), dict(q_weight=Fake((32,), "f32")),
                dict(k_weight=Fake((64,))), dict(v=Fake((4, 1, 64))), dict(k=Fake((4, 1, 64), "f16")),
                dict(slots=Fake((4,), "i32")), dict(v=Fake((4, 1, 64)), v_out=Fake((5, 1, 64)))):
        with pytest.raises(ValueError):
            ops.qk_norm_rotary(**{**good, **bad})
    q0, k0, kl = Fake((3,), "i32"), Fake((2,), "i64"), Fake((2,), "i32")
    kv = Fake((9, 1, 64))
    good = dict(q=x, k=kv, v=kv, q_start=q0, k_start=k0, k_len=kl, out=x)
    for bad in (dict(v=Fake((8, 1, 64))), dict(out=Fake((4, 2, 32))), dict(q_start=Fake((2,), "i32")), dict(k_start=kl),
                dict(k=Fake((9, 1, 32))), dict(lse=Fake((4, 3), "f32")), dict(lse=Fake((4, 2))), dict(k=Fake((9, 1, 64), "f16"))):
        with pytest.raises(ValueError):
            ops.attention(**{**good, **bad})


def fill(cls, **kw):
    a = cls()
    for name, _ in cls._fields_:
        if name in kw:
            setattr(a, name, kw[name])
    return a


P = 1 << 20


def rotary_args(**kw):
    base = dict(x=P, x_token=128, x_head=64, out=P, out_token=128, out_head=64, positions=P, table=P, places=10, tokens=4,
                heads=2, dim=64, rot=64)
    return fill(clear.RotaryArgs, **{**base, **kw})


def norm_args(**kw):
    base = dict(positions=P, table=P, places=10, cache_rows=9, tokens=4, heads=2, kv_heads=1, dim=64, rot=64, eps=1e-6)
    for r, st in (("q", 128), ("q_out", 128), ("k", 64), ("k_out", 64)):
        base.update({r: P, r + "_token": st, r + "_head": 64})
    return fill(clear.QkNormRotaryArgs, **{**base, **kw})


def attention_args(**kw):
    base = dict(q_start=P, k_start=P, k_len=P, lse=P, kv_rows=100, tokens=4, seqs=2, heads=4, kv_heads=2, dim=64, max_q=2,
                max_k=50, scale=0.125, causal=1)
    for r, st in (("q", 256), ("out", 256), ("k", 128), ("v", 128)):
        base.update({r: P, r + "_token": st, r + "_head": 64})
    return fill(clear.AttentionArgs, **{**base, **kw})


@pytest.mark.parametrize("bad,rc", [
    (dict(tokens=-1), -1), (dict(heads=-1), -1), (dict(x=None), -1), (dict(out=None), -1), (dict(positions=None), -1),
    (dict(table=None), -1), (dict(places=-1), -1), (dict(type=3), -1), (dict(type=-1), -1), (dict(x_token=-1), -1),
    (dict(dim=0), -2), (dict(dim=513), -2), (dict(rot=63), -2), (dict(rot=66), -2), (dict(rot=-2), -2),
    (dict(out_token=63), -2), (dict(out_head=32), -2), (dict(tokens=0), 0), (dict(heads=0), 0), (dict(tokens=0, x=None), 0)])
def test_rotary_refusals(bad, rc):
    assert LIB.pcx_rotary(C.byref(rotary_args(**bad)), None) == rc
    assert LIB.pcx_rotary(None, None) == -1


@pytest.mark.parametrize("bad,rc", [
    (dict(tokens=-1), -1), (dict(heads=-1), -1), (dict(kv_heads=-1), -1), (dict(q=None), -1), (dict(k=None), -1),
    (dict(q_out=None), -1), (dict(k_out=None), -1), (dict(v=P), -1), (dict(eps=-1.0), -1), (dict(eps=float("nan")), -1),
    (dict(positions=None), -1), (dict(slots=P, cache_rows=-1), -1), (dict(rot=1), -2), (dict(k_out_token=60), -2),
    (dict(v=P, v_out=P, v_out_token=1), -2), (dict(heads=0x7fffffff, kv_heads=1), -2), (dict(heads=0, kv_heads=0), 0),
    (dict(tokens=0, positions=None, table=None), 0)])
def test_qk_norm_rotary_refusals(bad, rc):
    assert LIB.pcx_qk_norm_rotary(C.byref(norm_args(**bad)), None) == rc
    assert LIB.pcx_qk_norm_rotary(None, None) == -1


@pytest.mark.parametrize("bad,rc", [
    (dict(tokens=-1), -1), (dict(seqs=-1), -1), (dict(heads=-1), -1), (dict(kv_rows=-1), -1), (dict(max_q=-1), -1),
    (dict(max_k=-1), -1), (dict(kv_heads=0), -1), (dict(kv_heads=3), -1), (dict(q_start=None), -1), (dict(k_start=None), -1),
    (dict(k_len=None), -1), (dict(q=None), -1), (dict(k=None), -1), (dict(v=None), -1), (dict(out=None), -1),
    (dict(scale=0.0), -1), (dict(scale=-1.0), -1), (dict(scale=float("nan")), -1), (dict(scale=float("inf")), -1),
    (dict(type=2), -2), (dict(type=-1), -2), (dict(dim=60), -2), (dict(dim=264), -2), (dict(dim=0), -2), (dict(q=P + 8), -2),
    (dict(k_token=129), -2), (dict(v_head=68), -2), (dict(out_head=32), -2), (dict(out_token=128, out_head=0), -2),
    (dict(work=P + 4, work_bytes=1024), -2), (dict(k_token=1 << 40), -2), (dict(tokens=0), 0), (dict(seqs=0), 0),
    (dict(heads=0), 0)])
def test_attention_refusals(bad, rc):
    a = attention_args(**bad)
    assert LIB.pcx_attention(C.byref(a), None) == rc
    assert LIB.pcx_attention(None, None) == -1
    if rc:
        assert LIB.pcx_attention_workspace(C.byref(a)) == 0
    assert LIB.pcx_attention_workspace(None) == 0


def test_the_header_s_structs():
    """the structs' fields in the header's order, each HeadsRef as three"""
    import re
    text = open(pa._lib.HEADER).read()
    for name in ("RotaryArgs", "QkNormRotaryArgs", "AttentionArgs"):
        end = text.index("} %s;" % name)
        body = re.sub(r"/\*.*?\*/", "", text[text.rindex("typedef struct", 0, end):end], flags=re.S)
        want = []
        for line in body.split("{", 1)[1].split(";"):
            line = line.strip()
            if not line:
                continue
            names = re.findall(r"\*?(\w+)\s*(?:,|$)", line)
            for n in names:
                want += [n, n + "_token", n + "_head"] if line.startswith("HeadsRef") else [n]
        assert [f for f, _ in getattr(clear, name)._fields_] == want


def test_packed_arguments_are_the_structs(ops):
    """struct.pack's layouts are the structs': the same bytes give the same fields"""
    x, kv = Fake((4, 6, 64), strides=(512, 64, 1)), Fake((9, 2, 64), ptr=P + 64)
    a = ops.attention_args(x, kv, kv, Fake((3,), "i32"), Fake((2,), "i64", ptr=P + 16), Fake((2,), "i32", ptr=P + 32), x,
                           Fake((4, 6), "f32", ptr=P + 48), scale=0.5, causal=False, max_q=3, max_k=7)
    got = {n: getattr(a, n) for n, _ in clear.AttentionArgs._fields_}
    want = dict(q=P, q_token=512, q_head=64, k=P + 64, k_token=128, k_head=64, v=P + 64, v_token=128, v_head=64, out=P,
                out_token=512, out_head=64, lse=P + 48, q_start=P, k_start=P + 16, k_len=P + 32, work=None, work_bytes=0,
                kv_rows=9, tokens=4, seqs=2, heads=6, kv_heads=2, dim=64, type=0, causal=0, max_q=3, max_k=7, scale=0.5)
    assert got == want
    for cls, packed in ((clear.RotaryArgs, clear._ROTARY), (clear.QkNormRotaryArgs, clear._QK_NORM_ROTARY)):
        n = len(cls._fields_)
        b = cls.from_buffer_copy(packed.pack(*range(1, n + 1)))
        assert [getattr(b, f) for f, _ in cls._fields_] == list(range(1, n + 1))
