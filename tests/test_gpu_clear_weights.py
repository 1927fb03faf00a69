"""The weight that keys gather on the GPU against its definition in 64 bits (tests/clear_oracle.py), bounded by f32 arithmetic. Each
test prints its case before the GPU runs."""
import sys

import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import clear
from tests import clear_oracle as co
from tests.test_gpu_clear import placed
from tests.test_gpu_clear_evict import per_key
from tests.test_gpu_clear_paged import paged

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ops():
    assert pa.device_count() >= 1, "no GPU visible"
    return pa.Clear(pa.Stream())


def true_lse(q, k, spans, group, scale, causal):
    out = np.full(q.shape[:2], -np.inf)
    for q0, n, k0, m in spans:
        for h in range(q.shape[1] if n and m else 0):
            with np.errstate(invalid="ignore", divide="ignore"):
                z = scale * (np.asarray(q[q0:q0 + n, h], np.float64) @ np.asarray(k[k0:k0 + m, h // group], np.float64).T)
                z = np.where(np.arange(m) <= m - n + np.arange(n)[:, None], z, -np.inf) if causal else z
                top = z.max(1, initial=-1e300)
                out[q0:q0 + n, h] = top + np.log(np.exp(z - top[:, None]).sum(1))
    return np.where(out < -1e299, -np.inf, out).astype(np.float32)


def run_weights(ops, kind, dim, heads, kv, spans, causal, page_rows, order="rows", keys="heads", hints=None, seed=0, edit=None, scale=None,
                decay=0.9, inplace=False, new=False, qscale=1.0, edit_lse=None):
    """spans [(queries, keys)]; unused rows NaN; edit(q, k, starts), edit_lse(lse): before the call"""
    rng = np.random.default_rng(seed + dim + heads + page_rows)
    qn, kn = [a for a, _ in spans], [b for _, b in spans]
    q0, k0 = (np.concatenate([[0], np.cumsum(x)]).astype(np.int64) for x in (qn, kn))
    T, group, scale = int(q0[-1]), heads // kv, dim ** -0.5 if scale is None else scale
    q = co.rounded(rng.normal(size=(T, heads, dim)) * qscale, kind)
    k = co.rounded(rng.normal(size=(int(k0[-1]), kv, dim)), kind)
    if edit:
        edit(q, k, k0[:-1])
    runs = [(int(a), n, int(b), m) for a, n, b, m in zip(q0, qn, k0, kn)]
    lse = true_lse(q, k, runs, group, scale, causal)
    if edit_lse:
        edit_lse(lse)
    if page_rows:
        table, rows, pool = paged(rng, kn, page_rows)
        where = dict(pages=pa.Array.of(table), page_rows=page_rows)
    else:
        starts = np.concatenate([[0], np.cumsum([n + 3 for n in kn])])
        rows, pool = [np.arange(s, s + n) for s, n in zip(starts, kn)], int(starts[-1]) + 1
        where = dict(k_start=pa.Array.of(starts[:-1].astype(np.int64)))
    kp, old = np.full((pool, kv, dim), np.nan, np.float32), np.full((pool, kv), 5.0, np.float32)
    places, nxt = np.full((pool, kv), -3), np.array([m + int(rng.integers(0, 9)) for m in kn])
    for b, r in enumerate(rows):
        kp[r] = k[k0[b]:k0[b + 1]]
        old[r] = rng.random((len(r), kv))
        if new:
            old[r[max(0, len(r) - qn[b]):]] = np.nan  # what evicted keys left there
    dw = per_key(np.full((pool, kv), 9.0, np.float32), "f32", keys)
    do = per_key(old, "f32", keys)
    dp = per_key(places, "i32", keys)
    kw = dict(before=do, decay=decay, scale=scale, causal=causal, **where)
    if inplace:
        dw = do
    if new:
        kw.update(places=dp, next_place=pa.Array.of(nxt.astype(np.int32)))
    if hints is not None:
        kw.update(max_q=hints[0], max_k=hints[1])
    ops.key_weights(placed(q, kind, order), placed(kp, kind, order), pa.Array.of(lse), pa.Array.of(q0, "i32"),
                    pa.Array.of(np.array(kn), "i32"), dw, **kw)
    want, bound = co.key_weights(q, k, lse, runs, group, scale, causal)
    got, gp = dw.numpy(ops.stream), dp.numpy(ops.stream)
    untouched = np.ones(pool, bool)
    for b, r in enumerate(rows):
        x, e = want[k0[b]:k0[b + 1]], bound[k0[b]:k0[b + 1]]
        base = decay * old[r].astype(np.float64) if decay else np.zeros((len(r), kv))
        if new:
            first = max(0, len(r) - qn[b])
            base[first:] = 0
            places[r[first:]] = (nxt[b] - len(r) + np.arange(first, len(r)))[:, None]
        co.check(got[r], base + x, e + 4 * co.E * (np.abs(base) + np.abs(x)) + 2.0 ** -140, f"sequence {b}")
        untouched[r] = False
    assert (got[untouched] == (old if inplace else np.full_like(old, 9.0))[untouched]).all(), "rows of no sequence were written"
    assert (gp == places).all()
    return got


SHAPES = [
    # dim, heads, kv heads, [(queries, keys)]
    (64, 12, 12, [(1, 512)]),
    (64, 1, 1, [(1, 1)]),
    (128, 8, 2, [(1, 33), (1, 64), (1, 1), (1, 0), (0, 40), (1, 700)]),
    (128, 32, 8, [(3, 130), (2, 2), (1, 65)]),
    (64, 4, 1, [(65, 65), (1, 1), (127, 127), (0, 0), (33, 33)]),
    (128, 6, 2, [(100, 333), (257, 257), (64, 64)]),
    (128, 3, 3, [(40, 10), (5, 0), (0, 70), (64, 63), (32, 31)]),
    (80, 5, 1, [(70, 150), (17, 17)]),
    (8, 2, 1, [(30, 60), (1, 5)]),
    (96, 14, 2, [(1, 257), (2, 129), (140, 300)]),
    (256, 2, 1, [(65, 200), (1, 77), (150, 150)]),
    (200, 4, 4, [(33, 40), (1, 300)]),
    (192, 7, 1, [(43, 43), (300, 300)]),
    (128, 64, 1, [(1, 400), (2, 50)]),
    (64, 71, 1, [(1, 300), (3, 40)]),
    (64, 300, 2, [(2, 270), (1, 9)]),
    (72, 48, 1, [(5, 90), (1, 600)]),
    (64, 2, 2, [(513, 513)]),
]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("page_rows", [0, 16, 64])
@pytest.mark.parametrize("shape", range(len(SHAPES)))
def test_key_weights(ops, kind, page_rows, shape):
    dim, heads, kv, spans = SHAPES[shape]
    say(f"[clear] key_weights {kind} dim {dim} heads {heads}/{kv} pages of {page_rows} {spans}")
    for causal in (True, False):
        run_weights(ops, kind, dim, heads, kv, spans, causal, page_rows)


@pytest.mark.parametrize("order,keys", [("padded", "rows"), ("heads", "padded"), ("rows", "rows"), ("heads", "heads")])
def test_key_weights_layouts(ops, order, keys):
    say(f"[clear] key_weights {order} {keys}")
    for dim, heads, kv, spans in ((128, 8, 2, [(1, 100), (3, 33), (70, 64)]), (80, 6, 2, [(50, 70), (1, 40)])):
        run_weights(ops, "bf16", dim, heads, kv, spans, True, 16, order=order, keys=keys)
        run_weights(ops, "f16", dim, heads, kv, spans, False, 0, order=order, keys=keys, inplace=True)


@pytest.mark.parametrize("page_rows", [0, 32])
def test_key_weights_of_new_keys(ops, page_rows):
    """the queries' own keys begin at 0, whatever lies there, and get their places; in place and not"""
    say(f"[clear] key_weights of new keys, pages of {page_rows}")
    for spans in ([(1, 90), (3, 3), (40, 300), (0, 20), (9, 4)], [(400, 400)]):
        run_weights(ops, "bf16", 64, 6, 2, spans, True, page_rows, new=True)
        run_weights(ops, "f16", 128, 4, 4, spans, True, page_rows, new=True, inplace=True, keys="rows")
        run_weights(ops, "bf16", 64, 6, 2, spans, False, page_rows, new=True, decay=0.0)


def test_key_weights_without_the_weights_before(ops):
    """decay 0 reads none, NaN or not; nor does before None"""
    say("[clear] key_weights without weights before")
    run_weights(ops, "bf16", 64, 2, 2, [(3, 70)], True, 16, decay=0.0)
    rng = np.random.default_rng(0)
    q, k = (co.rounded(rng.normal(size=(n, 2, 64)), "bf16") for n in (3, 70))
    lse = true_lse(q, k, [(0, 3, 0, 70)], 1, 0.125, True)
    out = pa.Array.of(np.full((70, 2), np.nan, np.float32))
    ops.key_weights(pa.Array.of(q, "bf16"), pa.Array.of(k, "bf16"), pa.Array.of(lse), pa.Array.of(np.array([0, 3]), "i32"),
                    pa.Array.of(np.array([70]), "i32"), out, k_start=pa.Array.of(np.zeros(1, np.int64)))
    want, bound = co.key_weights(q, k, lse, [(0, 3, 0, 70)], 1, 0.125, True)
    co.check(out.numpy(ops.stream), want, bound + 4 * co.E * want)


@pytest.mark.parametrize("dim,heads,kv,spans", [(128, 8, 2, [(700, 1500)]), (64, 4, 4, [(900, 900), (1, 300)]), (80, 20, 4, [(200, 4000), (80, 100)]),
                                                (64, 71, 1, [(30, 500)])])
def test_key_weights_with_the_rows_split(ops, dim, heads, kv, spans):
    """many rows over few keys: parts of the rows and their join; with room for few parts, and hints that are wrong"""
    say(f"[clear] key_weights split, dim {dim} heads {heads}/{kv} {spans}")
    for causal in (True, False):
        run_weights(ops, "bf16", dim, heads, kv, spans, causal, 16)
        run_weights(ops, "f16", dim, heads, kv, spans, causal, 0, new=True)
    run_weights(pa.Clear(ops.stream, workspace=40_000), "bf16", dim, heads, kv, spans, True, 16)
    run_weights(pa.Clear(ops.stream, workspace=0), "bf16", dim, heads, kv, spans, True, 16)
    for hints in ((0, 0), (1, 1), (10000, 200), (1, 100000), (100000, 100000)):
        run_weights(ops, "bf16", dim, heads, kv, spans, True, 16, hints=hints)


def test_key_weights_of_rows_that_see_nothing(ops):
    """a query whose log-sum-exp is -infinity adds nothing; infinities and NaN in keys reach those keys' weights alone"""
    say("[clear] key_weights: rows that see nothing, NaN keys and queries")

    def edit(q, k, k0):
        k[k0[0] + 5, 0, 3] = np.nan
        k[k0[0] + 99, 1, 0] = np.nan  # the last query alone sees it

    def edit_lse(lse):
        lse[2, 1] = -np.inf
        lse[np.isnan(lse)] = 3.0

    for page in (0, 16):
        got = run_weights(ops, "bf16", 64, 4, 2, [(20, 100), (40, 30)], True, page, edit=edit, edit_lse=edit_lse)
        assert np.isnan(got).sum() == 2


def test_key_weights_large_scores(ops):
    say("[clear] key_weights, scores up to thousands")
    run_weights(ops, "bf16", 64, 4, 2, [(100, 100), (1, 300)], True, 16, qscale=200.0, scale=1.0)
    run_weights(ops, "f16", 128, 4, 1, [(2, 400)], False, 0, qscale=30.0, scale=1.0)


def test_key_weights_many_sequences(ops):
    say("[clear] key_weights of 300 sequences, some empty")
    rng = np.random.default_rng(9)
    spans = [(int(rng.integers(0, 4)), int(rng.integers(0, 50))) for _ in range(300)]
    run_weights(ops, "bf16", 64, 2, 1, spans, True, 16, new=True)
    run_weights(ops, "f16", 64, 2, 2, [(5 * n, 2 * m) for n, m in spans[:130]], True, 0)


def test_key_weights_of_many_key_heads(ops):
    """more key heads than waves take at once"""
    say("[clear] key_weights of 5000 key heads")
    run_weights(ops, "f16", 8, 5000, 5000, [(1, 40), (2, 9)], True, 16, new=True)
    run_weights(ops, "bf16", 8, 600, 300, [(40, 50), (0, 3)], True, 0)


def test_key_weights_replay_as_a_graph(ops):
    """rows split and joined, and a token's, captured: replays with eager calls between them equal the eager sums"""
    say("[clear] key_weights as a graph, 3 replays")
    st, H, KV, D, n = ops.stream, 8, 2, 64, 700
    rng = np.random.default_rng(2)
    q, k = pa.Array((n, H, D), "bf16"), pa.Array((n, KV, D), "bf16")
    lse, w, q0 = pa.Array((n, H), "f32"), pa.Array((n, KV), "f32", strides=(1, n)), pa.Array((2,), "i32")
    k0, kl = pa.Array.of(np.zeros(1, np.int64)), pa.Array((1,), "i32")
    cases = [(rng.normal(size=(n, H, D)), rng.normal(size=(n, KV, D)), rng.random((n, H)) + 6, m) for m in (700, 500, 123)]

    def load(c):
        for x, y in ((q, c[0]), (k, c[1])):
            x.buf.upload(clear.to_bf16(y).view(np.uint32), st)
        lse.buf.upload(c[2].astype(np.float32).view(np.uint32), st)
        w.buf.upload(np.zeros(w.buf.words, np.uint32), st)
        q0.buf.upload(np.array([0, c[3]], np.uint32), st)
        kl.buf.upload(np.array([c[3]], np.uint32), st)

    def step():
        ops.key_weights(q, k, lse, q0, kl, w, k_start=k0, before=w, max_q=n, max_k=n)
        ops.key_weights(q, k, lse, q0, kl, w, k_start=k0, before=w, decay=0.5, max_q=1, max_k=n)

    eager = []
    for c in cases:
        load(c)
        step()
        eager.append(w.numpy(st))
    load(cases[0])
    graph = pa.Graph(st, step)
    for i, c in enumerate(cases):
        load(cases[(i + 1) % 3])
        step()
        st.sync()
        load(c)
        graph.launch(st)
        assert (w.numpy(st) == eager[i]).all(), i


def test_key_weights_cuts_and_bad_pages(ops):
    """lengths past the table or the cache end there, keys on pages outside the pool have no row"""
    say("[clear] key_weights with lengths past the cache and bad pages")
    rng = np.random.default_rng(5)
    H, KV, D, pool = 4, 2, 64, 6
    q, k = (co.rounded(rng.normal(size=(n, x, D)), "bf16") for n, x in ((6, H), (pool * 16, KV)))
    lse = rng.normal(size=(6, H)).astype(np.float32) + 5
    table = np.array([[2, 0, -1, 6, 4], [-2 ** 31, 2 ** 31 - 1, 5, 3, 7]])
    for paged_, lens, runs in ((True, [2 ** 31 - 1, 60], None), (False, [2 ** 31 - 1, 10, -4], [90, -1, 5])):
        n = len(lens)
        q0 = np.array([0, 2, 6, 9][:n + 1])
        out = pa.Array.of(np.full((pool * 16, KV), 9.0, np.float32))
        where = dict(pages=pa.Array.of(table, "i32"), page_rows=16) if paged_ else dict(k_start=pa.Array.of(np.array(runs), "i64"))
        ops.key_weights(pa.Array.of(q, "bf16"), pa.Array.of(k, "bf16"), pa.Array.of(lse), pa.Array.of(q0, "i32"),
                        pa.Array.of(np.array(lens), "i32"), out, **where)
        want, bound = np.full((pool * 16, KV), 9.0), np.zeros((pool * 16, KV))
        for b in range(n):
            if paged_:
                j = np.arange(min(lens[b], 80))
                p = table[b][j // 16].astype(np.int64)
                rows = np.where((p >= 0) & (p < pool), p * 16 + j % 16, -1)
            else:
                rows = np.arange(runs[b], min(runs[b] + lens[b], pool * 16)) if 0 <= runs[b] and lens[b] > 0 else np.zeros(0, int)
            n_q = min(q0[b + 1], 6) - min(q0[b], 6)
            K = np.where(rows[:, None, None] < 0, 0, k[rows]) if len(rows) else np.zeros((0, KV, D))
            w, e = co.key_weights(q, K, lse, [(q0[b], n_q, 0, len(rows))], H // KV, D ** -0.5, True)
            there = rows >= 0
            want[rows[there]], bound[rows[there]] = w[there], e[there] + 4 * co.E * w[there] + 2.0 ** -140
        co.check(out.numpy(ops.stream), want, bound)


def test_key_weights_repeat_to_the_bit(ops):
    say("[clear] key_weights three times, to the bit")
    a = [run_weights(ops, "bf16", 128, 8, 1, [(300, 3000), (2, 900)], True, 16) for _ in range(3)]
    assert np.array_equal(a[0], a[1]) and np.array_equal(a[0], a[2])


def test_the_weights_of_a_call_sum_to_its_heads(ops):
    """with attention's own log-sum-exps every (query, head) gives away 1"""
    say("[clear] attention_paged's log-sum-exps and key_weights")
    rng = np.random.default_rng(1)
    H, KV, D, lens, new = 8, 2, 128, [300, 77], [40, 1]
    table, rows, pool = paged(rng, lens, 16)
    q, k, v = (pa.Array.of(rng.normal(size=(n, h, D)), "bf16") for n, h in ((sum(new), H), (pool, KV), (pool, KV)))
    q0, n = pa.Array.of(np.concatenate([[0], np.cumsum(new)]), "i32"), pa.Array.of(np.array(lens), "i32")
    out, lse, w = pa.Array(q.shape, "bf16"), pa.Array(q.shape[:2], "f32"), pa.Array.of(np.zeros((pool, KV), np.float32))
    ops.attention_paged(q, k, v, q0, pa.Array.of(table), 16, n, out, lse)
    ops.key_weights(q, k, lse, q0, n, w, pages=pa.Array.of(table), page_rows=16, before=w)
    got = w.numpy(ops.stream)
    for b, r in enumerate(rows):
        assert np.allclose(got[r].sum(0, dtype=np.float64), new[b] * H // KV, rtol=2e-5)


@pytest.mark.parametrize("page_rows", [0, 16])
def test_key_weights_of_prompts_where_no_key_is_expected(ops, page_rows):
    """max_q of a prompt beside max_k 0, longer runs than that and none"""
    say(f"[clear] key_weights, prompts with max_k 0, pages of {page_rows}")
    run_weights(ops, "bf16", 64, 4, 2, [(300, 700), (40, 40)], True, page_rows, hints=(4096, 0))
    run_weights(ops, "bf16", 64, 4, 2, [(300, 0), (40, 0)], True, page_rows, hints=(4096, 0))


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_key_weights_of_keys_at_minus_infinity(ops, dim, causal):
    """keys that every query scores -infinity weigh what they did: rows that a tile has room for but the call has none of make no
    NaN of them (heads of a group that fill no tile, one token, odd prompts)"""
    say(f"[clear] key_weights, keys at -infinity, {dim} dimensions, causal {causal}")

    def edit(q, k, k0):
        q[:, :, dim - 3] = co.rounded(np.abs(q[:, :, dim - 3]) + 1, "f16")  # what the device gets
        for b, j in ((0, 7), (0, 290), (1, 3), (1, 64), (2, 5)):
            k[k0[b] + j, :, dim - 3] = -np.inf

    for heads, kv, spans in ((4, 2, [(1, 300), (3, 70), (2, 9)]), (6, 2, [(131, 300), (50, 70), (9, 9)]), (7, 1, [(40, 700), (33, 80), (1, 9)])):
        for page in (0, 16):
            got = run_weights(ops, "f16", dim, heads, kv, spans, causal, page, edit=edit)
            assert not np.isnan(got).any()


@pytest.mark.parametrize("dim,heads,kv,spans,causal", [(128, 16, 2, [(600, 900)], False), (64, 4, 4, [(2500, 500)], False),
                                                       (256, 8, 1, [(300, 1300)], True)])
def test_key_weights_of_rows_alike(ops, dim, heads, kv, spans, causal):
    """one sequence most of whose keys all queries see: workgroups alike, two a CU"""
    say(f"[clear] key_weights {dim} dimensions {heads}/{kv} heads, {spans}, causal {causal}")
    run_weights(ops, "bf16", dim, heads, kv, spans, causal, 16, hints=(spans[0][0], spans[0][1]))
    run_weights(ops, "f16", dim, heads, kv, spans, causal, 0, new=True)


def test_key_weights_offsets_past_32_bits(ops):
    """keys past 2^32 bytes and 2^31 values of a pool, in its pages and in one run"""
    say("[clear] key_weights far into a pool of 5.4 GB")
    rows, kv, dim, n, H = 2_600_000, 8, 128, 200, 16
    rng = np.random.default_rng(4)
    k = co.rounded(rng.normal(size=(n, kv, dim)), "bf16")
    first = rows // 16 - 13  # the last 13 pages
    table = np.arange(first + 12, first - 1, -1).astype(np.int32)[None]
    shuffled = np.concatenate([np.arange(16 * p, 16 * p + 16) for p in range(12, -1, -1)])[:n]
    buf = pa.DevBuf(rows * kv * dim // 2)
    pool = pa.Array((rows, kv, dim), "bf16", buf)
    weights = pa.Array((rows, kv), "f32", strides=(1, rows))
    for order, where in ((shuffled, dict(pages=pa.Array.of(table), page_rows=16)),
                         (np.arange(n), dict(k_start=pa.Array.of(np.array([first * 16], np.int64))))):
        tail = np.full((13 * 16, kv, dim), np.nan, np.float32)
        tail[order] = k
        buf.upload(clear.to_bf16(tail).view(np.uint32), offset=first * 16 * kv * dim // 2)
        for queries in (1, 90):
            q = co.rounded(rng.normal(size=(queries, H, dim)), "bf16")
            runs = [(0, queries, 0, n)]
            lse = true_lse(q, k, runs, H // kv, dim ** -0.5, True)
            ops.key_weights(pa.Array.of(q, "bf16"), pool, pa.Array.of(lse), pa.Array.of(np.array([0, queries]), "i32"),
                            pa.Array.of(np.array([n]), "i32"), weights, max_k=n, **where)
            want, bound = co.key_weights(q, k, lse, runs, H // kv, dim ** -0.5, True)
            got = weights.numpy(ops.stream)[first * 16:][order]
            co.check(got, want, bound + 4 * co.E * np.abs(want) + 2.0 ** -140, f"{queries} queries")


def test_calls_of_two_streams_at_once():
    """split weights and the choice of a long cache on two streams, each with a Clear of its own: what each gives alone"""
    say("[clear] key_weights and evict on two streams at once")
    H, KV, D, n, m = 8, 2, 64, 700, 20000
    sides = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        c = pa.Clear(pa.Stream())
        args = [pa.Array.of(rng.normal(size=(n, H, D)), "bf16"), pa.Array.of(rng.normal(size=(n, KV, D)), "bf16"),
                pa.Array.of((rng.random((n, H)) + 6).astype(np.float32)), pa.Array.of(np.array([0, n]), "i32"),
                pa.Array.of(np.array([n]), "i32"), pa.Array((n, KV), "f32")]
        long = [pa.Array.of(rng.random((m, KV)).astype(np.float32)), pa.Array.of(np.array([m]), "i32"), 5000,
                pa.Array.of(np.zeros((1, KV, 5000, 2), np.int32)), pa.Array.of(np.zeros((1, KV), np.int32))]
        k0 = pa.Array.of(np.zeros(1, np.int64))
        sides.append((c, args, long, k0))

    def call(side):
        c, args, long, k0 = side
        c.key_weights(*args, k_start=k0)
        c.evict(*long, k_start=k0)

    def answers(side):
        c, args, long, _ = side
        return [x.numpy(c.stream) for x in (args[-1], *long[3:])]

    alone = []
    for side in sides:
        call(side)
        alone.append(answers(side))
    for _ in range(20):
        for side in sides:
            call(side)
    for side, want in zip(sides, alone):
        assert all(np.array_equal(x, y) for x, y in zip(answers(side), want))
