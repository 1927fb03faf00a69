"""Attention over keys and values in pages against its definition in 64 bits (tests/clear_oracle.py), with the bounds of attention
over caches, and against attention over the same keys in one run, to the bit. Each test prints its case before the GPU runs."""
import ctypes as C
import sys

import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import clear
from perseus_amd._lib import LIB
from tests import clear_oracle as co
from tests.test_gpu_clear import placed

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ops():
    assert pa.device_count() >= 1, "no GPU visible"
    return pa.Clear(pa.Stream())


def paged(rng, lens, page_rows, spare=2, width=None):
    """(table, rows): pages of a pool in any order for sequences of these lengths, and each sequence's rows; unused entries far
    outside the pool"""
    need = [-(-n // page_rows) for n in lens]
    order = rng.permutation(sum(need) + spare)
    table = np.full((len(lens), width or max(max(need), 1)), 2 ** 31 - 1, np.int32)
    rows, at = [], 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
        j = np.arange(lens[b])
        rows.append(table[b, j // page_rows].astype(np.int64) * page_rows + j % page_rows if lens[b] else np.zeros(0, np.int64))
    return table, rows, (sum(need) + spare) * page_rows


def run_paged(ops, kind, dim, heads, kv, spans, causal, page_rows, order="rows", qscale=1.0, hints=None, seed=0, edit=None, scale=None,
              work=True, table_gap=0):
    """spans [(queries, keys)]; unused rows of the pool NaN; edit(q, k, v): keys of each sequence in their order"""
    rng = np.random.default_rng(seed + dim + heads + page_rows)
    qn, kn = [a for a, _ in spans], [b for _, b in spans]
    q0, k0 = (np.concatenate([[0], np.cumsum(x)]).astype(np.int64) for x in (qn, kn))
    T = int(q0[-1])
    q = co.rounded(rng.normal(size=(T, heads, dim)) * qscale, kind)
    k = co.rounded(rng.normal(size=(int(k0[-1]), kv, dim)), kind)
    v = co.rounded(rng.normal(size=(int(k0[-1]), kv, dim)) + 0.5, kind)
    if edit:
        edit(q, k, v, k0[:-1])
    table, rows, pool = paged(rng, kn, page_rows)
    kp, vp = (np.full((pool, kv, dim), np.nan, np.float32) for _ in range(2))
    for b, r in enumerate(rows):
        kp[r], vp[r] = k[k0[b]:k0[b + 1]], v[k0[b]:k0[b + 1]]
    scale = dim ** -0.5 if scale is None else scale
    dq, dk, dv = (placed(a, kind, order) for a in (q, kp, vp))
    wide = np.full((len(spans), table.shape[1] + table_gap), -7, np.int32)
    wide[:, :table.shape[1]] = table
    dt = pa.Array.of(wide)
    dt = pa.Array(table.shape, "i32", dt.buf, 0, (wide.shape[1], 1))
    hint = {} if hints is None else dict(max_q=hints[0], max_k=hints[1])
    got = []
    for pages in (True, False):
        out, lse = placed(np.full((T, heads, dim), 9.0), kind, order), pa.Array.of(np.full((T, heads), 9.0, np.float32))
        dq0, dn = pa.Array.of(q0, "i32"), pa.Array.of(np.array(kn), "i32")
        kw = dict(lse=lse, scale=scale, causal=causal, **hint)
        if pages:
            a = ops.attention_paged_args(dq, dk, dv, dq0, dt, page_rows, dn, out, **kw)
            inner, call = a.attention, LIB.pcx_attention_paged
            chosen = inner.max_q, inner.max_k
        else:  # the same keys in one run, by the kernels that were chosen
            ck, cv = (placed(x, kind, order) for x in (k, v))
            kw.update(max_q=chosen[0], max_k=chosen[1])
            a = ops.attention_args(dq, ck, cv, dq0, pa.Array.of(k0[:-1], "i64"), dn, out, **kw)
            inner, call = a, LIB.pcx_attention
        if not work:
            inner.work, inner.work_bytes = None, 0
        assert call(C.byref(a), ops.stream.h) == 0
        got.append((out.numpy(ops.stream), lse.numpy(ops.stream)))
    want, wl, spread, dlse = co.attention(q, k, v, [(int(a), n, int(b), m) for a, n, b, m in zip(q0, qn, k0, kn)], heads // kv, scale,
                                          causal)
    vmax = float(np.abs(v[np.isfinite(v)]).max()) if np.isfinite(v).any() else 1.0
    co.check(got[0][0], want, co.attention_bound(want, spread, dlse, kind, vmax), "out")
    co.check(got[0][1], wl, dlse, "lse")
    for x, y in zip(*got):
        assert np.array_equal(x, y, equal_nan=True), "not what one run of the same keys gives"
    return got[0]


SHAPES = [
    # dim, heads, kv heads, [(queries, keys)]
    (64, 12, 12, [(1, 1)]),
    (64, 12, 12, [(1, 512)]),
    (128, 8, 2, [(1, 33), (1, 64), (1, 1), (1, 0), (1, 700)]),
    (128, 32, 8, [(3, 130), (2, 2), (1, 65)]),
    (64, 4, 1, [(65, 65), (1, 1), (127, 127), (0, 0), (33, 33)]),
    (128, 4, 2, [(100, 333), (257, 257), (64, 64)]),
    (128, 3, 3, [(40, 10), (5, 0), (0, 70), (64, 63), (32, 31)]),
    (80, 5, 1, [(70, 150), (17, 17)]),
    (8, 2, 1, [(30, 60), (1, 5)]),
    (96, 14, 2, [(1, 257), (2, 129), (140, 300)]),
    (256, 2, 1, [(65, 200), (1, 77), (150, 150)]),
    (200, 4, 4, [(33, 40), (1, 300)]),
    (192, 3, 1, [(43, 43), (300, 300)]),
    (128, 64, 1, [(1, 400), (2, 50)]),
    (64, 2, 2, [(512, 512)]),
]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("page_rows", [16, 32, 128])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention_paged(ops, kind, page_rows, shape):
    dim, heads, kv, spans = SHAPES[shape]
    say(f"[clear] attention_paged {kind} dim {dim} heads {heads}/{kv} pages of {page_rows} {spans}")
    for causal in (True, False):
        run_paged(ops, kind, dim, heads, kv, spans, causal, page_rows)


@pytest.mark.parametrize("order", ["padded", "heads"])
@pytest.mark.parametrize("dim,heads,kv,spans", [
    (128, 8, 2, [(1, 100), (1, 33), (1, 64)]), (64, 4, 4, [(90, 90), (30, 200)]), (80, 6, 2, [(50, 70), (1, 40)])])
def test_attention_paged_layouts(ops, order, dim, heads, kv, spans):
    say(f"[clear] attention_paged {order}, tables with a gap, dim {dim} {spans}")
    run_paged(ops, "bf16", dim, heads, kv, spans, True, 16, order=order, table_gap=3)
    run_paged(ops, "f16", dim, heads, kv, spans, False, 64, order=order, table_gap=1)


@pytest.mark.parametrize("dim,heads,kv,spans,causal", [
    (128, 8, 1, [(1, 5000)], True), (64, 12, 12, [(1, 3001), (1, 100)], True), (128, 16, 2, [(40, 4000)], True),
    (80, 10, 2, [(19, 3500), (83, 1200)], False), (256, 4, 1, [(1, 2500)], True), (128, 2, 2, [(700, 1500)], True)])
def test_attention_paged_over_long_caches(ops, dim, heads, kv, spans, causal):
    """the keys split over the chip and joined; with a workspace that holds few splits, and without one"""
    say(f"[clear] attention_paged over long caches dim {dim} heads {heads}/{kv} {spans}")
    run_paged(ops, "bf16", dim, heads, kv, spans, causal, 16)
    run_paged(pa.Clear(ops.stream, workspace=300_000), "f16", dim, heads, kv, spans, causal, 256)
    run_paged(ops, "bf16", dim, heads, kv, spans, causal, 16, work=False)


@pytest.mark.parametrize("dim,heads,kv,spans", [(128, 4, 2, [(150, 150), (2, 100)]), (64, 6, 2, [(8, 200)]), (256, 2, 2, [(80, 80)])])
def test_attention_paged_infinite_and_nan_values(ops, dim, heads, kv, spans):
    """infinities and NaN at keys that only later queries see, and infinite values that are seen"""
    say(f"[clear] attention_paged with infinities and NaN, dim {dim} {spans}")

    def edit(q, k, v, k0):
        for s, (n, m) in zip(k0, spans):
            v[s + m - 1, 0, 3] = np.nan
            v[s + m - 2, -1, 0] = np.inf
            k[s + m - 3, 0, 1] = np.nan
            v[s + 3, -1, 5] = np.inf

    run_paged(ops, "bf16", dim, heads, kv, spans, True, 16, edit=edit)
    run_paged(ops, "f16", dim, heads, kv, spans, False, 32, edit=edit)


@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (1, 100000), (100000, 7)])
def test_attention_paged_hints_choose_no_result(ops, hints):
    say(f"[clear] attention_paged hints {hints}")
    for dim, heads, kv, spans in ((128, 8, 2, [(1, 900), (1, 3)]), (64, 6, 2, [(40, 1200), (3, 3), (9, 100)])):
        run_paged(ops, "bf16", dim, heads, kv, spans, True, 32, hints=hints)


def test_attention_paged_many_sequences(ops):
    say("[clear] attention_paged of 300 sequences, some empty")
    rng = np.random.default_rng(9)
    spans = [(int(rng.integers(0, 4)), int(rng.integers(0, 50))) for _ in range(300)]
    run_paged(ops, "bf16", 64, 2, 1, spans, True, 16)
    run_paged(ops, "f16", 64, 2, 2, [(5 * n, 2 * m) for n, m in spans[:130]], True, 32)


@pytest.mark.parametrize("queries", [1, 3, 200])
@pytest.mark.parametrize("page_rows", [16, 64])
def test_attention_paged_cuts_and_pages_outside_the_pool(ops, queries, page_rows):
    """keys past the table's width are not there; those on a page outside the pool read as zeros; sequences may share pages"""
    say(f"[clear] attention_paged: bad pages, lengths past the table, shared pages, {queries} queries, pages of {page_rows}")
    rng = np.random.default_rng(queries)
    H, KV, D, width, pool = 4, 2, 64, 5, 6
    q = co.rounded(rng.normal(size=(3 * queries, H, D)), "bf16")
    k, v = (co.rounded(rng.normal(size=(pool * page_rows, KV, D)), "bf16") for _ in range(2))
    table = np.array([[2, 0, 5, 1, 3], [2, 0, -1, 6, 4], [-2 ** 31, 2 ** 31 - 1, 2, 2, 7]], np.int32)
    lens = np.array([2 ** 31 - 1, width * page_rows - 3, 4 * page_rows - 1])
    out, lse = pa.Array.of(np.full(q.shape, 9.0), "bf16"), pa.Array.of(np.zeros((3 * queries, H), np.float32))
    for causal in (True, False):
        ops.attention_paged(pa.Array.of(q, "bf16"), pa.Array.of(k, "bf16"), pa.Array.of(v, "bf16"),
                            pa.Array.of(np.arange(4) * queries, "i32"), pa.Array.of(table), page_rows, pa.Array.of(lens, "i32"),
                            out, lse, causal=causal)
        seen = np.minimum(lens, width * page_rows)
        K, V, spans = [], [], []
        for b in range(3):
            j = np.arange(seen[b])
            page = table[b, j // page_rows].astype(np.int64)
            there = (page >= 0) & (page < pool)
            row = np.where(there, page, 0) * page_rows + j % page_rows
            spans.append((b * queries, queries, sum(len(x) for x in K), len(j)))
            K.append(k[row] * there[:, None, None])
            V.append(v[row] * there[:, None, None])
        K, V = np.concatenate(K), np.concatenate(V)
        want, wl, spread, dlse = co.attention(q, K, V, spans, H // KV, D ** -0.5, causal)
        co.check(out.numpy(ops.stream), want, co.attention_bound(want, spread, dlse, "bf16", 5.0), "out")
        co.check(lse.numpy(ops.stream), wl, dlse, "lse")


def test_attention_paged_offsets_past_32_bits(ops):
    """pages past 2^32 bytes and 2^31 values into a pool"""
    say("[clear] attention_paged far into a pool of 5.4 GB")
    rows, kv, dim, n = 1_300_000, 8, 128, 200
    rng = np.random.default_rng(2)
    k, v = (co.rounded(rng.normal(size=(n, kv, dim)), "bf16") for _ in range(2))
    pools = []
    first = rows // 16 - 13  # the last 13 pages, from the last on
    table = np.arange(first + 12, first - 1, -1).astype(np.int32)[None]
    order = np.concatenate([np.arange(16 * p, 16 * p + 16) for p in range(12, -1, -1)])[:n]
    for a in (k, v):
        tail = np.full((13 * 16, kv, dim), np.nan, np.float32)
        tail[order] = a
        buf = pa.DevBuf(rows * kv * dim // 2)
        buf.upload(clear.to_bf16(tail).view(np.uint32), offset=first * 16 * kv * dim // 2)
        pools.append(pa.Array((rows, kv, dim), "bf16", buf))
    for queries in (1, 90):
        q = co.rounded(rng.normal(size=(queries, 16, dim)), "bf16")
        out, lse = pa.Array((queries, 16, dim), "bf16"), pa.Array((queries, 16), "f32")
        ops.attention_paged(pa.Array.of(q, "bf16"), *pools, pa.Array.of(np.array([0, queries]), "i32"), pa.Array.of(table), 16,
                            pa.Array.of(np.array([n]), "i32"), out, lse)
        want, wl, spread, dlse = co.attention(q, k, v, [(0, queries, 0, n)], 2, dim ** -0.5, True)
        co.check(out.numpy(ops.stream), want, co.attention_bound(want, spread, dlse, "bf16", 5.0), "out")
        co.check(lse.numpy(ops.stream), wl, dlse, "lse")
