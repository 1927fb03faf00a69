"""The clear side's operators on the GPU against their definitions in 64 bits (tests/clear_oracle.py), at the sizes, layouts and
masks where they can go wrong. Bounds are those of f32 arithmetic and one rounding to the stored type. Each test prints its
case before the GPU runs."""
import ctypes as C
import sys

import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import clear
from perseus_amd._lib import LIB
from tests import clear_oracle as co

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ops():
    assert pa.device_count() >= 1, "no GPU visible"
    return pa.Clear(pa.Stream())


def placed(a, kind, order="rows", fill=None):
    """host values [T][H][D] on the device in a layout: "rows" dense; "padded": a gap after each head and each row; "heads":
    [H][T][D] in memory"""
    T, H, D = a.shape
    pad = 8
    if order == "rows":
        shape, st = (T, H, D), (H * D, D, 1)
    elif order == "padded":
        shape, st = (T, H, D), (H * (D + pad) + 2 * pad, D + pad, 1)
    else:
        shape, st = (T, H, D), (D, T * D, 1)
    x = pa.Array(shape, kind, strides=st)
    size = {"bf16": 2, "f16": 2, "f32": 4}[kind]
    flat = np.full(4 * x.buf.words // size, np.nan if fill is None else fill, np.float32)
    view = np.lib.stride_tricks.as_strided(flat, shape, [s * 4 for s in st])
    view[...] = a
    raw = clear.to_bf16(flat) if kind == "bf16" else flat.astype(np.float16 if kind == "f16" else np.float32)
    x.buf.upload(raw.view(np.uint32))
    return x


# ---------------------------------------------------------------------------------------------------- rotary


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot,heads,tokens,order", [
    (64, 64, 24, 1, "rows"), (128, 128, 5, 37, "rows"), (128, 32, 3, 70, "padded"), (80, 80, 4, 9, "heads"),
    (96, 48, 7, 33, "rows"), (256, 64, 2, 5, "padded"), (40, 24, 3, 17, "rows"), (6, 2, 3, 11, "rows"), (33, 14, 5, 6, "rows"),
    (512, 512, 1, 3, "rows"), (72, 8, 2, 130, "heads"), (128, 0, 4, 3, "rows"), (1, 0, 3, 5, "rows"), (64, 62, 2, 4, "rows")])
def test_rotary(ops, kind, layout, dim, rot, heads, tokens, order):
    say(f"[clear] rotary {kind} {layout} dim {dim} rot {rot} heads {heads} tokens {tokens} {order}")
    rng = np.random.default_rng(dim * 1000 + rot + tokens)
    x = co.rounded(rng.normal(size=(tokens, heads, dim)) * 3, kind)
    table = clear.rotary_table(50, rot, 1000.0) if rot else np.zeros((50, 0, 2), np.float32)
    pos = rng.integers(0, 50, tokens)
    pos[-1] = 49
    dx, dp = placed(x, kind, order), pa.Array.of(pos, "i32")
    dt = pa.Array.of(table) if rot else None
    for inverse in (False, True):
        y, mag = co.rotary(x, pos, table, layout, inverse)
        out = placed(np.full_like(x, 7), kind, order)
        ops.rotary(dx, dp, dt, out, layout=layout, inverse=inverse)
        co.check(out.numpy(ops.stream), y, co.rotary_bound(y, mag, kind), f"inverse {inverse}")
    y, mag = co.rotary(x, pos, table, layout)
    ops.rotary(dx, dp, dt, dx, layout=layout)  # in place
    co.check(dx.numpy(ops.stream), y, co.rotary_bound(y, mag, kind), "in place")


@pytest.mark.parametrize("kind", ["bf16", "f32"])
def test_rotary_gaps_and_positions_outside_the_table(ops, kind):
    say(f"[clear] rotary {kind}: positions outside the table, gaps of the output untouched")
    rng = np.random.default_rng(3)
    x = co.rounded(rng.normal(size=(6, 3, 64)), kind)
    table = clear.rotary_table(10, 32)
    pos = np.array([0, -1, 9, 10, 2 ** 31 - 1, -2 ** 31])
    out = placed(np.zeros_like(x), kind, "padded", fill=5.0)
    ops.rotary(placed(x, kind), pa.Array.of(pos, "i32"), pa.Array.of(table), out)
    y, mag = co.rotary(x, pos, table, "half")
    co.check(out.numpy(ops.stream), y, co.rotary_bound(y, mag, kind))
    flat = out.buf.download(stream=ops.stream).view(np.uint16 if kind == "bf16" else np.float32)
    flat = clear.from_bf16(flat) if kind == "bf16" else flat
    mask = np.ones(flat.size, bool)
    view = np.lib.stride_tricks.as_strided(mask, out.shape, out.stride())
    view[...] = False
    assert (flat[mask] == 5.0).all(), "a gap was written"


def test_rotary_undone_returns_the_values(ops):
    """the inverse is the rotation's transpose: in 32 bits both together move a value by a few units of the last place"""
    say("[clear] rotary f32 and back")
    rng = np.random.default_rng(5)
    x = rng.normal(size=(200, 4, 128)).astype(np.float32)
    a, pos = pa.Array.of(x), pa.Array.of(rng.integers(0, 4096, 200), "i32")
    table = pa.Array.of(clear.rotary_table(4096, 128))
    ops.rotary(a, pos, table, a)
    ops.rotary(a, pos, table, a, inverse=True)
    pairs = np.hypot(x[..., :64], x[..., 64:])
    co.check(a.numpy(ops.stream), x, 16 * co.E * np.concatenate([pairs, pairs], -1))


# ---------------------------------------------------------------------------------------------------- norms


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,rot,heads,kv,tokens,order", [
    (128, 128, 32, 8, 3, "rows"), (64, 64, 4, 4, 65, "padded"), (96, 32, 6, 2, 20, "rows"), (80, 80, 5, 1, 9, "heads"),
    (256, 256, 3, 1, 4, "rows"), (40, 40, 0, 3, 7, "rows"), (128, 64, 7, 0, 130, "rows"), (30, 10, 2, 1, 5, "rows"),
    (512, 512, 2, 1, 2, "rows"), (128, 0, 2, 2, 3, "rows"), (72, 16, 9, 3, 1, "padded")])
def test_qk_norm_rotary(ops, kind, layout, dim, rot, heads, kv, tokens, order):
    say(f"[clear] qk_norm_rotary {kind} {layout} dim {dim} rot {rot} heads {heads}/{kv} tokens {tokens} {order}")
    rng = np.random.default_rng(dim + rot + heads)
    q = co.rounded(rng.normal(size=(tokens, heads, dim)) * 10, kind)
    k = co.rounded(rng.normal(size=(tokens, kv, dim)) * 1e-2, kind)
    v = co.rounded(rng.normal(size=(tokens, kv, dim)), kind)
    wq, wk = (1 + 0.3 * rng.normal(size=dim)).astype(np.float32), None if tokens == 3 else rng.normal(size=dim).astype(np.float32)
    table = clear.rotary_table(300, rot) if rot else np.zeros((300, 0, 2), np.float32)
    pos = rng.integers(0, 300, tokens)
    eps = 1e-5
    dq, dk, dv = (placed(a, kind, order) for a in (q, k, v))
    dp, dt = pa.Array.of(pos, "i32"), pa.Array.of(table) if rot else None
    dwq, dwk = pa.Array.of(wq), None if wk is None else pa.Array.of(wk)
    wants = [co.rotary(co.norm(a, w, eps), pos, table, layout) for a, w in ((q, wq), (k, wk))]
    qo, ko = placed(np.zeros_like(q), kind, order), placed(np.zeros_like(k), kind, order)
    ops.qk_norm_rotary(dq, dk, dwq, dwk, dp, dt, qo, ko, eps=eps, layout=layout)
    for got, (y, mag), what in ((qo, wants[0], "q"), (ko, wants[1], "k")):
        co.check(got.numpy(ops.stream), y, co.norm_rotary_bound(y, mag, kind, dim), what)
    # into a cache: rows by slot, some outside it, values beside the keys
    rows = tokens + 9
    slots = rng.permutation(rows)[:tokens].astype(np.int64)
    slots[0] = -1
    if tokens > 2:
        slots[2] = rows
    kc, vc = (placed(np.full((rows, kv, dim), 3.0), kind, order) for _ in range(2))
    ops.qk_norm_rotary(dq, dk, dwq, dwk, dp, dt, dq, kc, eps=eps, layout=layout, v=dv, v_out=vc, slots=pa.Array.of(slots))
    y, mag = wants[0]
    co.check(dq.numpy(ops.stream), y, co.norm_rotary_bound(y, mag, kind, dim), "q in place")
    (y, mag), full, fmag, fv = wants[1], np.full((rows, kv, dim), 3.0), np.zeros((rows, kv, dim)), np.full((rows, kv, dim), 3.0)
    for t, r in enumerate(slots):
        if 0 <= r < rows:
            full[r], fmag[r], fv[r] = y[t], mag[t], v[t]
    co.check(kc.numpy(ops.stream), full, co.norm_rotary_bound(full, fmag, kind, dim) * (fmag > 0), "cache keys")
    assert (vc.numpy(ops.stream) == fv).all(), "cache values"


def test_norm_of_zeros_and_large_heads(ops):
    """a head of zeros stays zero (eps alone under the root); eps 0 too is a division by zero as defined: NaN; squares near
    f32's range"""
    say("[clear] qk_norm_rotary: zero heads, large values")
    x = np.zeros((2, 2, 64), np.float32)
    x[1] = 1e17
    pos, table = pa.Array.of(np.zeros(2, np.int32)), pa.Array.of(clear.rotary_table(1, 64))
    q, k = pa.Array.of(x), pa.Array.of(x[:, :1])
    ops.qk_norm_rotary(q, k, None, None, pos, table, q, k, eps=1e-6)
    want = np.zeros((2, 2, 64))
    want[1] = 1
    co.check(q.numpy(ops.stream), want, 64 * co.E, "q")
    q = pa.Array.of(x)
    ops.qk_norm_rotary(q, k, None, None, pos, table, q, k, eps=0.0)
    assert np.isnan(q.numpy(ops.stream)[0]).all()


# ---------------------------------------------------------------------------------------------------- attention


def run_attention(ops, kind, dim, heads, kv, spans, causal, order="rows", gap=0, qscale=1.0, lse=True, hints=None, seed=0,
                  tail=0, edit=None, scale=None, work=True):
    """spans [(queries, keys)]; gap: unused key rows between sequences, NaN; tail: query rows of no sequence"""
    rng = np.random.default_rng(seed + dim + heads)
    qn, kn = [a for a, _ in spans], [b for _, b in spans]
    q0 = np.concatenate([[0], np.cumsum(qn)]).astype(np.int64)
    k0 = np.concatenate([[0], np.cumsum([b + gap for b in kn])])[:-1].astype(np.int64) + gap
    T, R = int(q0[-1]) + tail, int(sum(kn) + gap * (len(kn) + 1))
    q = co.rounded(rng.normal(size=(T, heads, dim)) * qscale, kind)
    k = np.full((R, kv, dim), np.nan, np.float32)
    v = k.copy()
    for s, n in zip(k0, kn):
        k[s:s + n] = co.rounded(rng.normal(size=(n, kv, dim)), kind)
        v[s:s + n] = co.rounded(rng.normal(size=(n, kv, dim)) + 0.5, kind)
    if edit:
        edit(q, k, v, k0)
    scale = dim ** -0.5 if scale is None else scale
    dq, dk, dv = (placed(a, kind, order) for a in (q, k, v))
    out = placed(np.full((T, heads, dim), 9.0), kind, order)
    dl = pa.Array.of(np.full((T, heads), 9.0, np.float32))
    args = (dq, dk, dv, pa.Array.of(q0, "i32"), pa.Array.of(k0, "i64"), pa.Array.of(np.array(kn), "i32"), out)
    kw = dict(lse=dl if lse else None, scale=scale, causal=causal)
    if hints is not None:
        kw.update(max_q=hints[0], max_k=hints[1])
    a = ops.attention_args(*args, **kw)
    if not work:
        a.work, a.work_bytes = None, 0
    assert LIB.pcx_attention(C.byref(a), ops.stream.h) == 0
    want, wl, spread, dlse = co.attention(q, k, v, [(int(a), n, int(b), m) for a, n, b, m in zip(q0, qn, k0, kn)],
                                          heads // kv, scale, causal)
    got, gl = out.numpy(ops.stream), dl.numpy(ops.stream)
    if tail:
        assert (got[T - tail:] == 9.0).all(), "rows of no sequence were written"
        got, gl, want, wl, spread, dlse = (x[:T - tail] for x in (got, gl, want, wl, spread, dlse))
    vmax = float(np.abs(v[np.isfinite(v)]).max()) if np.isfinite(v).any() else 1.0
    co.check(got, want, co.attention_bound(want, spread, dlse, kind, vmax), "out")
    if lse:
        co.check(gl, wl, dlse, "lse")
    return got


SHAPES = [
    # dim, heads, kv heads, [(queries, keys)]
    (64, 12, 12, [(1, 1)]),
    (64, 12, 12, [(1, 512)]),
    (128, 8, 2, [(1, 33), (1, 64), (1, 1), (1, 0), (1, 700)]),
    (128, 32, 8, [(3, 130), (2, 2), (1, 65)]),
    (64, 2, 2, [(512, 512)]),
    (64, 4, 1, [(65, 65), (1, 1), (127, 127), (0, 0), (33, 33)]),
    (128, 4, 2, [(100, 333), (257, 257), (64, 64)]),
    (128, 3, 3, [(40, 10), (5, 0), (0, 70), (64, 63), (32, 31)]),
    (80, 5, 1, [(70, 150), (17, 17)]),
    (40, 6, 3, [(1, 90), (1, 31), (20, 20)]),
    (8, 2, 1, [(30, 60), (1, 5)]),
    (72, 7, 1, [(1, 300), (9, 40)]),
    (96, 14, 2, [(1, 257), (2, 129)]),
    (256, 2, 1, [(65, 200), (1, 77)]),
    (200, 4, 4, [(33, 40), (1, 300)]),
    (256, 8, 1, [(1, 513), (1, 2)]),
    (128, 64, 1, [(1, 400), (2, 50)]),
    (64, 48, 2, [(3, 100)]),
    (16, 1, 1, [(300, 300)]),
]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_attention(ops, kind, causal, shape):
    dim, heads, kv, spans = SHAPES[shape]
    say(f"[clear] attention {kind} causal {causal} dim {dim} heads {heads}/{kv} {spans}")
    run_attention(ops, kind, dim, heads, kv, spans, causal)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim,heads,kv,spans", [
    (128, 8, 2, [(32, 900)]), (128, 8, 2, [(16, 1500), (9, 33)]), (192, 4, 1, [(30, 500), (7, 64)]), (136, 4, 2, [(150, 330)]),
    (192, 3, 1, [(43, 43), (300, 300)]), (256, 4, 1, [(25, 700)]), (64, 8, 1, [(100, 1300)]), (32, 4, 1, [(128, 128)] * 3)])
def test_attention_between_few_rows_and_many(ops, kind, dim, heads, kv, spans):
    """33 to 128 rows of a key head and a little more, with the keys split and whole; widths between 129 and 192"""
    say(f"[clear] attention {kind} dim {dim} heads {heads}/{kv} {spans}")
    for causal in (True, False):
        run_attention(ops, kind, dim, heads, kv, spans, causal)


@pytest.mark.parametrize("order", ["padded", "heads"])
@pytest.mark.parametrize("dim,heads,kv,spans", [
    (128, 8, 2, [(1, 100), (1, 33), (1, 64)]), (64, 4, 4, [(90, 90), (30, 200)]), (80, 6, 2, [(50, 70), (1, 40)])])
def test_attention_layouts_and_gaps(ops, order, dim, heads, kv, spans):
    """strided tensors; NaN in every gap of the tensors, between sequences and after them; rows of no sequence unwritten"""
    say(f"[clear] attention {order}, NaN gaps, dim {dim} heads {heads}/{kv} {spans}")
    run_attention(ops, "bf16", dim, heads, kv, spans, True, order=order, gap=37, tail=3)
    run_attention(ops, "f16", dim, heads, kv, spans, False, order=order, gap=5, lse=False)


@pytest.mark.parametrize("dim,heads,kv,spans", [
    (128, 4, 2, [(150, 150), (70, 100)]), (64, 6, 2, [(8, 200)]), (64, 3, 3, [(300, 300)]), (256, 2, 2, [(80, 80)])])
def test_attention_unseen_values_do_not_reach_a_query(ops, dim, heads, kv, spans):
    """the last keys hold infinities and NaN: only the queries that see them become NaN"""
    say(f"[clear] attention with NaN and infinities in unseen keys, dim {dim} {spans}")

    def edit(q, k, v, k0):
        for s, (n, m) in zip(k0, spans):
            v[s + m - 1, 0, 3] = np.nan
            v[s + m - 2, -1, 0] = np.inf
            k[s + m - 3, 0, 1] = np.nan

    run_attention(ops, "bf16", dim, heads, kv, spans, True, edit=edit)


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim,heads,kv,spans", [
    (128, 4, 2, [(1, 900), (3, 100)]), (64, 2, 2, [(1, 40), (2, 3000)]), (256, 4, 2, [(2, 300)]), (128, 4, 2, [(150, 150)]),
    (64, 2, 2, [(300, 300)])])
def test_attention_infinite_values_that_are_seen(ops, kind, dim, heads, kv, spans):
    """an infinite value makes that dimension of the queries that see it infinite, two of different sign NaN"""
    say(f"[clear] attention with infinite values {kind} dim {dim} {spans}")

    def edit(q, k, v, k0):
        for s in k0:
            v[s + 3, 0, 1] = np.inf
            v[s + 4:s + 30, -1, 2] = -np.inf
            v[s + 9, 0, 5], v[s + 17, 0, 5] = np.inf, -np.inf

    for causal in (True, False):
        run_attention(ops, kind, dim, heads, kv, spans, causal, edit=edit)


@pytest.mark.parametrize("dim,heads,kv,spans", [(128, 4, 2, [(5, 900)]), (64, 2, 2, [(1, 40), (2, 3000)]), (128, 4, 4, [(200, 200)])])
def test_attention_of_nan_queries(ops, dim, heads, kv, spans):
    """a query of NaN has NaN for its sums and no finite log: its neighbours in the tile and the split do not"""
    say(f"[clear] attention with a NaN query, dim {dim} {spans}")

    def edit(q, k, v, k0):
        q[0, 0] = np.nan

    got = run_attention(ops, "bf16", dim, heads, kv, spans, True, edit=edit)
    assert np.isnan(got[0, 0]).all() and not np.isnan(got[0, 1:]).any()


def test_attention_large_scores(ops):
    """scores in the thousands: one key takes the whole weight, each f32 exponential's argument stays exact enough"""
    say("[clear] attention, scores up to thousands; growing maxima")
    run_attention(ops, "bf16", 64, 4, 2, [(100, 100), (1, 300)], True, qscale=200.0, scale=1.0)

    def rising(q, k, v, k0):  # every key's score above the last: the running maximum grows at each step
        q[...] = 1
        for s in k0:
            k[s:s + 400] = co.rounded(np.linspace(-4, 4, 400), "bf16")[:, None, None]

    run_attention(ops, "bf16", 64, 4, 2, [(60, 400), (1, 400)], True, edit=rising, scale=0.5)
    run_attention(ops, "f16", 128, 4, 1, [(2, 400), (1, 400)], False, edit=rising, scale=0.125)


@pytest.mark.parametrize("hints", [(0, 0), (1, 1), (1, 100000), (100000, 7)])
@pytest.mark.parametrize("work", [True, False])
def test_attention_hints_choose_no_result(ops, hints, work):
    """max_q and max_k below, above and far from the lengths, with and without a workspace"""
    say(f"[clear] attention hints {hints} workspace {work}")
    for dim, heads, kv, spans in ((128, 8, 2, [(1, 900), (1, 3)]), (64, 6, 2, [(40, 1200), (3, 3), (9, 100)])):
        run_attention(ops, "bf16", dim, heads, kv, spans, True, hints=hints, work=work)


@pytest.mark.parametrize("dim,heads,kv,spans,causal", [
    (128, 8, 1, [(1, 5000)], True), (64, 12, 12, [(1, 3001), (1, 100)], True), (128, 16, 2, [(40, 4000)], True),
    (80, 10, 2, [(19, 3500), (83, 1200)], False), (256, 4, 1, [(1, 2500)], True), (128, 2, 2, [(700, 1500)], True)])
def test_attention_over_long_caches(ops, dim, heads, kv, spans, causal):
    """few rows over many keys: the keys split over the chip and joined; with a workspace that holds few splits too"""
    say(f"[clear] attention over long caches dim {dim} heads {heads}/{kv} {spans}")
    run_attention(ops, "bf16", dim, heads, kv, spans, causal)
    small = pa.Clear(ops.stream, workspace=300_000)
    run_attention(small, "f16", dim, heads, kv, spans, causal)


def test_attention_many_sequences(ops):
    say("[clear] attention of 300 sequences, some empty")
    rng = np.random.default_rng(9)
    spans = [(int(rng.integers(0, 4)), int(rng.integers(0, 50))) for _ in range(300)]
    run_attention(ops, "bf16", 64, 2, 1, spans, True)
    run_attention(ops, "bf16", 64, 2, 1, [(1, m) for _, m in spans], True, hints=(1, 50))
    run_attention(ops, "f16", 64, 2, 2, [(5 * n, 2 * m) for n, m in spans[:130]], True, gap=1)


def test_attention_lengths_past_the_buffers_are_cut(ops):
    """device lengths that leave the buffers: key runs end with the rows, query runs with the tokens; sequences that begin
    outside see nothing"""
    say("[clear] attention with lengths past the buffers")
    rng = np.random.default_rng(1)
    q, k, v = (co.rounded(rng.normal(size=(n, 2, 64)), "bf16") for n in (6, 50, 50))
    dq, dk, dv = (pa.Array.of(a, "bf16") for a in (q, k, v))
    for causal in (False, True):
        for starts, runs, spans in (
                ([0, 3, 9], ([40, 10], [60, 5]), [(0, 3, 40, 10), (3, 3, 10, 5)]),
                ([0, 2, 6], ([-5, 51], [10, 10]), [(0, 2, 0, 0), (2, 4, 0, 0)]),
                ([0, 5, 6], ([0, 49], [-7, 2 ** 31 - 1]), [(0, 5, 0, 0), (5, 1, 49, 1)])):
            out, lse = pa.Array.of(np.full((6, 2, 64), 9.0), "bf16"), pa.Array.of(np.zeros((6, 2), np.float32))
            ops.attention(dq, dk, dv, pa.Array.of(np.array(starts), "i32"), pa.Array.of(np.array(runs[0]), "i64"),
                          pa.Array.of(np.array(runs[1]), "i32"), out, lse, causal=causal)
            want, wl, spread, dlse = co.attention(q, k, v, spans, 1, 0.125, causal)
            co.check(out.numpy(ops.stream), want, co.attention_bound(want, spread, dlse, "bf16", 5.0), "out")
            co.check(lse.numpy(ops.stream), wl, dlse, "lse")


def test_attention_offsets_past_32_bits(ops):
    """keys past 2^32 bytes and 2^31 values into a cache, and a token stride of a whole cache row"""
    say("[clear] attention far into a cache of 5.4 GB")
    rows, kv, dim, n = 1_300_000, 8, 128, 200
    words = rows * kv * dim // 2
    rng = np.random.default_rng(2)
    k, v = (co.rounded(rng.normal(size=(n, kv, dim)), "bf16") for _ in range(2))
    caches = []
    first = rows - n
    for a in (k, v):
        buf = pa.DevBuf(words)
        buf.upload(clear.to_bf16(a).view(np.uint32), offset=first * kv * dim // 2)
        caches.append(pa.Array((rows, kv, dim), "bf16", buf))
    for queries in (1, 90):
        q = co.rounded(rng.normal(size=(queries, 16, dim)), "bf16")
        out, lse = pa.Array((queries, 16, dim), "bf16"), pa.Array((queries, 16), "f32")
        ops.attention(pa.Array.of(q, "bf16"), *caches, pa.Array.of(np.array([0, queries]), "i32"),
                      pa.Array.of(np.array([first]), "i64"), pa.Array.of(np.array([n]), "i32"), out, lse)
        want, wl, spread, dlse = co.attention(q, k, v, [(0, queries, 0, n)], 2, dim ** -0.5, True)
        co.check(out.numpy(ops.stream), want, co.attention_bound(want, spread, dlse, "bf16", 5.0), "out")
        co.check(lse.numpy(ops.stream), wl, dlse, "lse")


def test_attention_repeats_to_the_bit(ops):
    """sums are taken in one order: the same call gives the same words"""
    say("[clear] attention three times, to the bit")
    a = [run_attention(ops, "bf16", 128, 8, 1, [(1, 3000), (2, 900)], True) for _ in range(3)]
    assert (a[0] == a[1]).all() and (a[0] == a[2]).all()


def test_a_decode_step_replays_as_a_graph(ops):
    """a step captured once (norms, rotation and the cache rows, then attention over the cache) follows the device's lengths,
    positions and slots: three replays with eager work between them equal the eager steps"""
    say("[clear] a decode step as a graph, 3 replays")
    rng = np.random.default_rng(4)
    B, H, KV, D, cap = 3, 8, 2, 64, 150
    st = ops.stream
    lens = np.array([100, 7, 60])
    table = pa.Array.of(clear.rotary_table(cap, D))
    fill = [co.rounded(rng.normal(size=(B * cap, KV, D)), "bf16") for _ in range(2)]

    def fresh():
        return [pa.Array.of(a, "bf16") for a in fill]

    dpos, dslot, dlen = pa.Array((B,), "i32"), pa.Array((B,), "i64"), pa.Array((B,), "i32")
    dq0, dk0 = pa.Array.of(np.arange(B + 1), "i32"), pa.Array.of(np.arange(B) * cap, "i64")
    rows = pa.Array((B, H + 2 * KV, D), "bf16")
    qn, out, lse = pa.Array((B, H, D), "bf16"), pa.Array((B, H, D), "bf16"), pa.Array((B, H), "f32")

    def load(step, x):
        rows.buf.upload(clear.to_bf16(x).view(np.uint32), st)
        dpos.buf.upload((lens + step).astype(np.int32).view(np.uint32), st)
        dslot.buf.upload((np.arange(B) * cap + lens + step).astype(np.int64).view(np.uint32), st)
        dlen.buf.upload((lens + step + 1).astype(np.int32).view(np.uint32), st)

    def step(kc, vc):
        ops.qk_norm_rotary(rows.heads(0, H), rows.heads(H, KV), None, None, dpos, table, qn, kc, v=rows.heads(H + KV, KV),
                           v_out=vc, slots=dslot)
        ops.attention(qn, kc, vc, dq0, dk0, dlen, out, lse, max_q=1, max_k=cap)

    xs = [co.rounded(rng.normal(size=(B, H + 2 * KV, D)), "bf16") for _ in range(3)]
    eager = []
    kc, vc = fresh()
    for i, x in enumerate(xs):
        load(i, x)
        step(kc, vc)
        eager.append((out.numpy(st), lse.numpy(st)))
    end = kc.numpy(st), vc.numpy(st)
    kc, vc = fresh()
    load(0, xs[0])
    other = fresh()
    graph = pa.Graph(st, lambda: step(kc, vc))
    for i, x in enumerate(xs):
        load(i, x)
        step(*other)  # eager work between the replays, on other caches
        st.sync()
        graph.launch(st)
        got, gl = out.numpy(st), lse.numpy(st)
        assert (got == eager[i][0]).all() and (gl == eager[i][1]).all(), i
    assert (kc.numpy(st) == end[0]).all() and (vc.numpy(st) == end[1]).all()
