"""Eviction from a cache on the GPU against its definition (tests/clear_oracle.py): whole numbers and moved words, equal to the last
one. Each test prints its case before the GPU runs."""
import sys

import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import clear
from tests import clear_oracle as co
from tests.test_gpu_clear_paged import paged

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ops():
    assert pa.device_count() >= 1, "no GPU visible"
    return pa.Clear(pa.Stream())


def per_key(a, kind, order):
    """host values [rows][kv heads] on the device: a row after the other ("rows"), a head after the other ("heads"), or either
    with gaps ("padded")"""
    rows, kv = a.shape
    st = {"rows": (kv, 1), "heads": (1, rows), "padded": (2 * kv + 3, 2)}[order]
    x = pa.Array((rows, kv), kind, strides=st)
    flat = np.zeros(x.buf.words, {"f32": np.float32, "i32": np.int32}[kind])
    np.lib.stride_tricks.as_strided(flat, (rows, kv), [4 * s for s in st])[...] = a
    x.buf.upload(flat.view(np.uint32))
    return x


def run_evict(ops, lens, kv, keep, recent, first, page_rows, weigh, places=True, next_place=True, order="heads", most=None, max_k=None,
              dim=16, kind="bf16", seed=0):
    """weigh(rng, n): the weights of n keys"""
    rng = np.random.default_rng(seed + sum(lens) + keep)
    if page_rows:
        table, rows, pool = paged(rng, lens, page_rows)
        where = dict(pages=pa.Array.of(table), page_rows=page_rows)
    else:
        starts = np.concatenate([[0], np.cumsum([n + 2 for n in lens])])
        rows, pool = [np.arange(s, s + n) for s, n in zip(starts, lens)], int(starts[-1]) + 1
        where = dict(k_start=pa.Array.of(starts[:-1].astype(np.int64)))
    w = np.full((pool, kv), 7e30, np.float32)
    p = np.full((pool, kv), -5, np.int32)
    nxt = np.array([n + int(rng.integers(0, 50)) for n in lens])
    for b, r in enumerate(rows):
        for g in range(kv):
            w[r, g] = weigh(rng, len(r))
            p[r, g] = rng.permutation(nxt[b])[:len(r)] if places else np.arange(len(r))
    k = co.rounded(rng.normal(size=(pool, kv, dim)), kind)
    most = max(1, min(keep, max(lens) - keep)) if most is None else most
    moves = pa.Array.of(np.full((len(lens), kv, most, 2), -9, np.int32))
    count, kept_len = pa.Array.of(np.full((len(lens), kv), -9, np.int32)), pa.Array.of(np.full(len(lens), -9, np.int32))
    dw, dp, dk = per_key(w, "f32", order), per_key(p, "i32", order), pa.Array.of(k, kind)
    dn = pa.Array.of(np.array(lens, np.int32))
    ops.evict(dw, dn, keep, moves, count, places=dp if places else None,
              next_place=pa.Array.of(nxt.astype(np.int32)) if next_place else None, recent=recent, first=first, kept_len=kept_len,
              max_k=max_k, **where)
    want = np.full((len(lens), kv, most, 2), -9)
    number = np.zeros((len(lens), kv), int)
    for b, r in enumerate(rows):
        for g in range(kv):
            _, mv = co.kept(w[r, g], p[r, g], nxt[b] if next_place else len(r), keep, recent, first)
            number[b, g] = len(mv)
            for i, (x, y) in enumerate(mv[:most]):
                want[b, g, i] = x, y
                k[r[y], g], w[r[y], g], p[r[y], g] = k[r[x], g], w[r[x], g], p[r[x], g]
    assert (count.numpy(ops.stream) == number).all()
    got = moves.numpy(ops.stream)
    assert (got == want).all(), f"{int((got != want).any(-1).sum())} moves differ"
    assert (kept_len.numpy(ops.stream) == np.minimum(lens, keep)).all()
    ops.move_rows(moves, count, (dk, dw, dp), **where)
    for x, y in ((dk, k), (dw, w), (dp, p)):
        assert np.array_equal(x.numpy(ops.stream), y, equal_nan=True)
    return number


def spread(rng, n):
    return np.exp(2.5 * rng.normal(size=n) - 3) * (rng.random(n) > 0.1)


CASES = [
    # lengths, kv heads, keep, recent, first, rows of a page
    ([528], 12, 512, 32, 4, 0), ([1], 1, 1, 0, 0, 16), ([2], 3, 1, 0, 0, 16), ([17, 0, 3, 40], 2, 9, 2, 1, 16),
    ([64, 65, 63, 128], 1, 64, 0, 0, 0), ([700, 30, 1025], 5, 333, 40, 4, 32), ([1000], 2, 999, 0, 0, 64), ([1000], 2, 1, 0, 0, 16),
    ([5000, 4097, 4100], 4, 4096, 256, 4, 16), ([16384], 1, 4000, 100, 0, 0), ([16385, 20000], 2, 10000, 0, 8, 128),
    ([40], 2, 0, 0, 0, 16), ([40, 12], 2, 12, 12, 0, 16), ([300], 1, 100, 90, 10, 0),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("order", ["heads", "rows", "padded"])
def test_evict(ops, case, order):
    lens, kv, keep, recent, first, page = CASES[case]
    say(f"[clear] evict lengths {lens} kv {kv} keep {keep} recent {recent} first {first} pages of {page} {order}")
    run_evict(ops, lens, kv, keep, recent, first, page, spread, order=order)


@pytest.mark.parametrize("page", [0, 16])
@pytest.mark.parametrize("lens", [[70000], [65536, 66000], [66000, 100]])
def test_evict_of_long_caches(ops, lens, page):
    """chunks in registers, and more keys than they hold; a longest run that was not expected"""
    say(f"[clear] evict lengths {lens} pages of {page}")
    run_evict(ops, lens, 2, 17000, 500, 4, page, spread)
    run_evict(ops, lens, 2, 60000, 500, 4, page, spread, max_k=100)


@pytest.mark.parametrize("page", [0, 16])
def test_evict_of_short_runs_beside_long_ones(ops, page):
    """slices of no key, of one key, and sequences that keep all, where the longest is shared out to many workgroups"""
    say(f"[clear] evict of lengths from 0 to 20000 together, pages of {page}")
    for keep in (1, 2, 3, 15, 16, 17, 100):
        run_evict(ops, [20000, keep + 1, keep, 0, keep + 2, 2 * keep + 31, 2000], 3, keep, 0, 0, page, spread)
    run_evict(ops, [16385, 5000], 2, 4999, 40, 4, page, spread)


@pytest.mark.parametrize("what", ["alike", "few", "zeros", "signs", "bits"])
@pytest.mark.parametrize("n,keep", [(900, 300), (20000, 15000), (130, 65)])
def test_evict_of_ties_and_strange_weights(ops, what, n, keep):
    """weights alike go by their number; infinities, NaN, zeros of both signs, subnormal and neighbouring values"""
    say(f"[clear] evict {what}: {n} keys, {keep} kept")

    def weigh(rng, m):
        if what == "alike":
            return np.full(m, 0.25)
        if what == "few":
            return rng.integers(0, 4, m) * 0.5
        if what == "zeros":
            return np.where(rng.random(m) < 0.8, 0.0, rng.random(m)) * np.where(rng.random(m) < 0.5, 1, -1)
        if what == "signs":
            x = rng.normal(size=m)
            x[rng.random(m) < 0.3] = np.nan
            x[rng.random(m) < 0.2] = -np.inf
            x[rng.random(m) < 0.2] = np.inf
            return x
        return (np.float32(1e-42) * rng.integers(-3, 4, m) if m % 2 else
                np.nextafter(np.float32(1), np.float32(2)) * (1 + np.float32(2.0 ** -23) * rng.integers(0, 3, m)))

    run_evict(ops, [n, n - 7], 3, keep, 0, 0, 16, weigh)
    run_evict(ops, [n], 2, keep, 20, 3, 0, weigh)


def test_evict_without_places(ops):
    """a key's number is its place, the length the next one; either given alone"""
    say("[clear] evict without places")
    run_evict(ops, [400, 350], 2, 300, 50, 4, 16, spread, places=False, next_place=False)
    run_evict(ops, [400, 350], 2, 300, 50, 4, 0, spread, places=False, next_place=True)
    run_evict(ops, [400, 350], 2, 300, 50, 4, 0, spread, places=True, next_place=False)


def test_evict_with_room_for_few_moves(ops):
    """the number that there are is told, those that fit are written and moved"""
    say("[clear] evict with room for 5 moves")
    assert (run_evict(ops, [900, 700], 2, 500, 0, 0, 16, spread, most=5) > 5).all()


def test_evict_many_sequences(ops):
    say("[clear] evict of 200 sequences")
    rng = np.random.default_rng(3)
    run_evict(ops, [int(n) for n in rng.integers(0, 90, 200)], 3, 40, 7, 2, 16, spread)


@pytest.mark.parametrize("page", [0, 16])
def test_evict_cuts_lengths_and_bad_pages(ops, page):
    """lengths past the buffers end with them; keys on a page that the pool does not have leave first and no row of theirs moves"""
    say(f"[clear] evict with lengths past the cache, pages of {page}")
    rng = np.random.default_rng(8)
    kv, pool, keep = 2, 96, 40
    w = rng.random((pool, kv)).astype(np.float32)
    dw = per_key(w, "f32", "heads")
    if page:
        table = np.array([[3, 9, 0, -1, 4], [-2 ** 31, 2 ** 31 - 1, 5, 2, 1]])
        where, runs = dict(pages=pa.Array.of(table, "i32"), page_rows=16), table
        lens = [2 ** 31 - 1, 70]
    else:
        where, runs, lens = dict(k_start=pa.Array.of(np.array([10, -1, 96, 50], np.int64))), [10, -1, 96, 50], [2 ** 31 - 1, 60, 60, -3]
    seqs = len(lens)
    moves, count = pa.Array.of(np.full((seqs, kv, 60, 2), -9, np.int32)), pa.Array.of(np.zeros((seqs, kv), np.int32))
    kept_len = pa.Array.of(np.zeros(seqs, np.int32))
    ops.evict(dw, pa.Array.of(np.array(lens), "i32"), keep, moves, count, kept_len=kept_len, **where)
    x = np.arange(pool * kv, dtype=np.float32).reshape(pool, kv)
    dx = per_key(x, "f32", "rows")
    for b in range(seqs):
        if page:
            j = np.arange(min(lens[b], 80))
            p = runs[b][j // 16].astype(np.int64)
            rows = np.where((p >= 0) & (p < 6), p * 16 + j % 16, -1)
        else:
            at = runs[b]
            rows = np.arange(at, min(at + max(lens[b], 0), pool)) if 0 <= at < pool else np.zeros(0, int)
        assert kept_len.numpy(ops.stream)[b] == min(len(rows), keep)
        for g in range(kv):
            # below every weight, NaN too, and never protected: the lowest of all
            mine = np.where(rows < 0, np.nan, w[rows, g]) if len(rows) else np.zeros(0)
            _, mv = co.kept(mine, np.arange(len(rows)), len(rows), keep, 0, 0)
            assert count.numpy(ops.stream)[b, g] == len(mv)
            assert (moves.numpy(ops.stream)[b, g, :len(mv)] == np.array(mv).reshape(-1, 2)).all()
            for s, d in mv:
                if rows[s] >= 0 and rows[d] >= 0:
                    x[rows[d], g] = x[rows[s], g]
    ops.move_rows(moves, count, (dx,), **where)
    assert (dx.numpy(ops.stream) == x).all()


@pytest.mark.parametrize("kind,dim,order", [("bf16", 64, "rows"), ("bf16", 128, "heads"), ("f16", 256, "rows"), ("f32", 80, "padded"),
                                            ("bf16", 7, "rows"), ("f16", 1, "rows"), ("f32", 3, "padded"), ("i64", 5, "rows"),
                                            ("bf16", 514, "rows"), ("i32", 700, "heads")])
def test_move_rows_of_all_types_and_layouts(ops, kind, dim, order):
    """words move as they are (NaN with their bits), gaps of the tensors stay, moves outside the cache or the lists are skipped"""
    say(f"[clear] move_rows {kind} dim {dim} {order}")
    rng = np.random.default_rng(dim)
    rows, kv, seqs, most = 70, 3, 2, 9
    size = clear.SIZES[kind]
    st = {"rows": (kv * dim, dim, 1), "heads": (dim, rows * dim, 1), "padded": (kv * (dim + 5) + 2, dim + 5, 1)}[order]
    x = pa.Array((rows, kv, dim), kind, strides=st)
    word = {2: np.uint16, 4: np.uint32, 8: np.uint64}[size]
    flat = rng.integers(0, 256, 4 * x.buf.words, np.uint8).view(word)
    x.buf.upload(flat.view(np.uint32))
    table = np.array([[3, 0], [1, 2]])
    moves = np.full((seqs, kv, most, 2), -1, np.int32)
    count = np.array([[4, 0, most + 5], [-3, 1, 2]], np.int32)
    for b in range(seqs):
        for g in range(kv):
            moves[b, g, :, 0] = 16 + rng.permutation(16)[:most]
            moves[b, g, :, 1] = rng.permutation(16)[:most]
    moves[0, 2, 3] = 40, 2      # past the table
    moves[0, 2, 4] = -1, 3
    moves[0, 2, 5] = 20, -2 ** 31
    moves[0, 2, 6] = 2 ** 31 - 1, 5
    ops.move_rows(pa.Array.of(moves), pa.Array.of(count), (x,), pages=pa.Array.of(table, "i32"), page_rows=16)
    view = np.lib.stride_tricks.as_strided(flat, x.shape, [s * size for s in st])
    for b in range(seqs):
        for g in range(kv):
            for s, d in moves[b, g, :max(0, min(count[b, g], most))]:
                if 0 <= s < 32 and 0 <= d < 32:
                    view[table[b, d // 16] * 16 + d % 16, g] = view[table[b, s // 16] * 16 + s % 16, g].copy()
    assert (x.buf.download(stream=ops.stream).view(word) == flat).all()


def test_evict_and_moves_far_into_a_pool(ops):
    """rows past 2^32 bytes"""
    say("[clear] evict and move_rows far into a pool of 5.4 GB")
    rows, kv, dim, n, keep = 1_300_000, 8, 128, 96, 64
    first = rows - n
    rng = np.random.default_rng(6)
    k = co.rounded(rng.normal(size=(n, kv, dim)), "bf16")
    buf = pa.DevBuf(rows * kv * dim // 2)
    buf.upload(clear.to_bf16(k).view(np.uint32), offset=first * kv * dim // 2)
    cache = pa.Array((rows, kv, dim), "bf16", buf)
    w = np.zeros((rows, kv), np.float32)
    w[first:] = spread(rng, n * kv).reshape(n, kv)
    moves, count = pa.Array.of(np.zeros((1, kv, 32, 2), np.int32)), pa.Array.of(np.zeros((1, kv), np.int32))
    table = np.arange(first // 16, rows // 16)[None]
    where = dict(pages=pa.Array.of(table, "i32"), page_rows=16)
    ops.evict(per_key(w, "f32", "heads"), pa.Array.of(np.array([n]), "i32"), keep, moves, count, **where)
    ops.move_rows(moves, count, (cache,), **where)
    for g in range(kv):
        for s, d in co.kept(w[first:, g], np.arange(n), n, keep, 0, 0)[1]:
            k[d, g] = k[s, g]
    got = buf.download(stream=ops.stream, offset=first * kv * dim // 2).view(np.uint16)
    assert (clear.from_bf16(got).reshape(k.shape) == k).all()


def test_evict_of_long_caches_replays_as_a_graph(ops):
    """the launches of a long cache's choice captured once: replays with eager calls between them equal the eager lists"""
    say("[clear] evict of 30000 keys as a graph, 3 replays")
    st, n, kv, keep = ops.stream, 30000, 2, 9000
    rng = np.random.default_rng(7)
    w = [spread(rng, n * kv).reshape(kv, n).astype(np.float32) for _ in range(3)]
    dw, k0, dn = pa.Array((n, kv), "f32", strides=(1, n)), pa.Array.of(np.zeros(1, np.int64)), pa.Array((1,), "i32")
    moves, count = pa.Array((1, kv, keep, 2), "i32"), pa.Array((1, kv), "i32")

    def load(i):
        dw.buf.upload(w[i].reshape(-1).view(np.uint32), st)
        dn.buf.upload(np.array([n - 37 * i], np.uint32), st)
        moves.buf.upload(np.zeros(moves.buf.words, np.uint32), st)

    def step():
        ops.evict(dw, dn, keep, moves, count, k_start=k0, recent=50, first=4)

    eager = []
    for i in range(3):
        load(i)
        step()
        eager.append((moves.numpy(st), count.numpy(st)))
        for g in range(kv):
            mv = co.kept(w[i][g, :n - 37 * i], np.arange(n - 37 * i), n - 37 * i, keep, 50, 4)[1]
            assert (eager[i][0][0, g, :len(mv)] == np.array(mv)).all() and eager[i][1][0, g] == len(mv)
    load(0)
    graph = pa.Graph(st, step)
    for i in range(3):
        load((i + 1) % 3)
        step()
        st.sync()
        load(i)
        graph.launch(st)
        assert (moves.numpy(st) == eager[i][0]).all() and (count.numpy(st) == eager[i][1]).all()


@pytest.mark.parametrize("seqs", [6, 9, 20, 42, 43])
def test_evict_of_long_caches_by_fewer_workgroups(ops, seqs):
    """3 heads of 6 to 42 sequences: from 14 slices of a cache down to 2; of 43, none"""
    say(f"[clear] evict of {seqs} sequences, one of 17000 keys")
    rng = np.random.default_rng(seqs)
    lens = [17000] + [int(n) for n in rng.integers(0, 600, seqs - 1)]
    run_evict(ops, lens, 3, 200, 20, 4, 16, spread)
    run_evict(ops, lens[1:], 3, 200, 20, 4, 0, spread, max_k=16385)


@pytest.mark.parametrize("n", [127, 128, 129, 130, 300, 17000])
def test_evict_of_weights_within_a_quarter_of_an_octave(ops, n):
    """one first digit for all: as many to be ranked as there is room for, one fewer and more"""
    say(f"[clear] evict of {n} weights of one first digit")
    for keep in (1, n // 2, n - 1):
        run_evict(ops, [n], 2, keep, 0, 0, 16, lambda rng, m: 1 + 0.249 * rng.random(m))
