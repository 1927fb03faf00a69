"""attention.PagedBlock as a program runs it: sequences of different lengths append prompts, chunks and tokens over a shared pool, gather
their keys' weights and are cut to what a scoring holds, against a cache kept on the host in 64 bits from the definitions. Each step
prints its case before the GPU runs."""
import sys

import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import attention, clear
from tests import clear_oracle as co

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


class Host:
    """a sequence's cache on the host: keys and values as stored, weights in 64 bits with their bounds, places by key head"""

    def __init__(self, kv, dim):
        self.k = self.v = np.zeros((0, kv, dim))
        self.w = self.bound = np.zeros((0, kv))
        self.p, self.next = np.zeros((0, kv), int), 0

    def grow(self, n, kv):
        self.w, self.bound = (np.concatenate([x, np.zeros((n, kv))]) for x in (self.w, self.bound))
        self.p = np.concatenate([self.p, np.repeat(np.arange(self.next, self.next + n)[:, None], kv, 1)])
        self.next += n

    def move(self, moves, keep):
        for g, pairs in enumerate(moves):
            for s, d in pairs:
                for x in (self.k, self.v, self.w, self.bound, self.p):
                    x[d, g] = x[s, g]
        self.k, self.v, self.w, self.bound, self.p = (x[:keep] for x in (self.k, self.v, self.w, self.bound, self.p))


def drive(kind, H, KV, D, keep, recent, first, steps, page_rows, layout="half", decay=1.0, scaling=None, seed=0):
    rng = np.random.default_rng(seed)
    seqs = len(steps[0])
    st = pa.Stream()
    ops = pa.Clear(st)
    table = clear.rotary_table(1000, D, scaling=scaling)
    w = (1 + 0.1 * rng.normal(size=(2, D))).astype(np.float32)
    blk = attention.PagedBlock(ops, H, KV, D, seqs, 120 // page_rows * seqs + 30, page_rows, keep, recent, first, tokens=400, dtype=kind,
                               table=pa.Array.of(table), layout=layout, q_weight=pa.Array.of(w[0]), k_weight=pa.Array.of(w[1]), decay=decay)
    host = [Host(KV, D) for _ in range(seqs)]
    group, scale = H // KV, D ** -0.5
    free = len(blk._free)
    for counts in steps:
        say(f"[paged block] {kind} lengths {blk.lengths} + {list(counts)}")
        rows = co.rounded(rng.normal(size=(sum(counts), H + 2 * KV, D)) * 2, kind)
        q, out, lse = (x.numpy(st) for x in blk.append(pa.Array.of(rows, kind), counts))
        at = 0
        for b, n in enumerate(counts):
            if not n:
                continue
            x, h = rows[at:at + n], host[b]
            places = np.arange(h.next, h.next + n)
            y, mag = co.rotary(co.norm(x[:, :H], w[0], 1e-6), places, table, layout)
            co.check(q[at:at + n], y, co.norm_rotary_bound(y, mag, kind, D), "queries")
            mine = blk._rows(b, np.arange(blk.lengths[b]))
            k, v = blk.k.numpy(st)[mine], blk.v.numpy(st)[mine]
            y, mag = co.rotary(co.norm(x[:, H:H + KV], w[1], 1e-6), places, table, layout)
            co.check(k[-n:], y, co.norm_rotary_bound(y, mag, kind, D), "keys")
            assert (k[:-n] == h.k).all() and (v[:-n] == h.v).all() and (v[-n:] == x[:, H + KV:]).all()
            h.k, h.v = k.astype(np.float64), v.astype(np.float64)
            span = [(0, n, 0, len(k))]
            want, wl, spread, dlse = co.attention(q[at:at + n], k, v, span, group, scale, True)
            co.check(out[at:at + n], want, co.attention_bound(want, spread, dlse, kind, 12.0), "attention")
            co.check(lse[at:at + n], wl, dlse, "lse")
            h.grow(n, KV)
            add, bound = co.key_weights(q[at:at + n], k, lse[at:at + n], span, group, scale, True)
            h.w = decay * h.w + add
            h.bound = decay * h.bound + bound + 8 * co.E * h.w
            co.check(blk.weights.numpy(st)[mine], h.w, h.bound + 2.0 ** -140, "weights")
            assert (blk.places.numpy(st)[mine] == h.p).all()
            at += n
        longer = max(blk.lengths) > keep
        device = blk.weights.numpy(st)
        before = [device[blk.rows_of(b)] for b in range(seqs)]
        moves, count = blk.evict()
        assert (moves is not None) == longer
        if longer:
            moves, count = moves.numpy(st), count.numpy(st)
            for b, h in enumerate(host):
                want = [co.kept(before[b][:, g], h.p[:, g], h.next, keep, recent, first)[1] for g in range(KV)]
                for g in range(KV):
                    assert [tuple(m) for m in moves[b, g, :count[b, g]]] == [tuple(int(y) for y in m) for m in want[g]]
                h.move(want, keep)
                mine = blk.rows_of(b)
                assert len(mine) == len(h.k) <= keep
                assert (blk.keys(b) == h.k.reshape(len(mine), KV * D)).all() and (blk.v.numpy(st)[mine] == h.v).all()
                assert (blk.places.numpy(st)[mine] == h.p).all()
        used = [p for x in blk._pages for p in x]
        assert len(set(used)) == len(used) and sorted(used + blk._free) == list(range(free))
    return blk, host


def test_a_pool_of_sequences_that_are_cut():
    """prompts, chunks and tokens together; some sequences idle; every one past its keep more than once"""
    steps = [(70, 5, 0), (1, 60, 33), (20, 0, 40), (1, 1, 1), (0, 17, 1), (33, 1, 64), (1, 1, 1)]
    drive("bf16", 8, 2, 64, 64, 16, 4, steps, 16)
    drive("f16", 6, 6, 80, 50, 10, 0, steps, 32, layout="interleaved", decay=0.75, scaling=("by_turns", 4, 64, 1, 4))


def test_the_scoring_s_512_keys():
    """a prompt longer than the encrypted scoring holds, cut to its 512 keys, then a token: the scoring's own sizes; the keys that are
    left pack into its slots, and their scores and the token's log-sum-exp give the token's probabilities"""
    H, D, T = attention.HEADS, attention.HEAD_DIM, attention.TOKENS
    blk, host = drive("bf16", H, H, D, T, 32, 4, [(400,), (170,), (1,)], 16, seed=3)
    st = blk.ops.stream
    assert blk.lengths == [T] and blk.next_places == [571]
    K = blk.keys(0)
    assert K.shape == (T, H * D)
    slots = attention.key_slots(K, 2 ** 16)
    q = blk.q.numpy(st)[0]
    sums = [np.repeat((z * p).reshape(-1, D).sum(1), D) for z, p in zip(slots, attention.query_slots(q, 2 ** 16))]
    scores = attention.scores_from_slots(sums)
    want = np.einsum("hd,thd->ht", q.astype(np.float64), K.reshape(T, H, D))
    assert np.abs(scores - want).max() < 1e-9 * np.abs(want).max()
    assert (np.sort(host[0].p[:, 0])[:4] == np.arange(4)).all() and (np.sort(host[0].p[:, 0])[-32:] == np.arange(539, 571)).all()


def test_a_sequence_that_ended_leaves_its_pages():
    say("[paged block] a pool that fills up, a sequence dropped")
    ops = pa.Clear(pa.Stream())
    rng = np.random.default_rng(1)
    blk = attention.PagedBlock(ops, 2, 1, 64, 2, 4, keep=100, recent=0, first=0, tokens=64)
    rows = lambda n: pa.Array.of(rng.normal(size=(n, 4, 64)), "bf16")  # noqa: E731
    blk.append(rows(60), (30, 30))
    with pytest.raises(ValueError):
        blk.append(rows(5), (5, 0))
    assert blk.lengths == [30, 30]
    blk.append(rows(2), (2, 0))
    blk.drop(0)
    q, out, lse = blk.append(rows(30), (28, 2))
    assert blk.lengths == [28, 32] and blk.next_places == [28, 32]
    assert np.isfinite(out.numpy(ops.stream)).all() and (blk.places.numpy(ops.stream)[blk.rows_of(0), 0] == np.arange(28)).all()


def test_a_cut_replays_as_a_graph():
    """a token's attention, its weights, the choice and the moves captured once: three replays over lengths and caches that change between
    them equal the eager calls, words and lists"""
    say("[paged block] attention_paged, key_weights, evict and move_rows as a graph, 3 replays")
    st = pa.Stream()
    ops = pa.Clear(st)
    rng = np.random.default_rng(4)
    B, H, KV, D, P, keep, width = 3, 8, 2, 64, 16, 40, 6
    pool = B * width * P
    table = pa.Array.of(rng.permutation(B * width).reshape(B, width), "i32")
    cases = []
    for i in range(3):
        cases.append(dict(q=co.rounded(rng.normal(size=(B, H, D)), "bf16"), k=co.rounded(rng.normal(size=(pool, KV, D)), "bf16"),
                          v=co.rounded(rng.normal(size=(pool, KV, D)), "bf16"), w=rng.random((KV, pool)).astype(np.float32),
                          p=rng.integers(0, 200, (KV, pool)).astype(np.int32), n=rng.integers(20, 96, B).astype(np.int32),
                          x=rng.integers(90, 210, B).astype(np.int32)))
    q, k, v, out = (pa.Array(s, "bf16") for s in ((B, H, D), (pool, KV, D), (pool, KV, D), (B, H, D)))
    w, p = (pa.Array((pool, KV), t, strides=(1, pool)) for t in ("f32", "i32"))
    n, x, lse, q0 = pa.Array((B,), "i32"), pa.Array((B,), "i32"), pa.Array((B, H), "f32"), pa.Array.of(np.arange(B + 1), "i32")
    moves, count, kept = pa.Array((B, KV, keep, 2), "i32"), pa.Array((B, KV), "i32"), pa.Array((B,), "i32")
    where = dict(pages=table, page_rows=P)

    def load(c):
        for a, b in ((q, c["q"]), (k, c["k"]), (v, c["v"])):
            a.buf.upload(clear.to_bf16(b).view(np.uint32), st)
        for a, b in ((w, c["w"]), (p, c["p"]), (n, c["n"]), (x, c["x"])):
            a.buf.upload(b.reshape(-1).view(np.uint32), st)
        moves.buf.upload(np.zeros(moves.buf.words, np.uint32), st)

    def step():
        ops.attention_paged(q, k, v, q0, table, P, n, out, lse, max_q=1, max_k=width * P)
        ops.key_weights(q, k, lse, q0, n, w, before=w, places=p, next_place=x, max_q=1, max_k=width * P, **where)
        ops.evict(w, n, keep, moves, count, places=p, next_place=x, recent=6, first=2, kept_len=kept, max_k=width * P, **where)
        ops.move_rows(moves, count, (k, v, w, p), **where)

    def results():
        return [a.numpy(st) for a in (out, lse, k, v, w, p, moves, count, kept)]

    eager = []
    for c in cases:
        load(c)
        step()
        eager.append(results())
    load(cases[0])
    graph = pa.Graph(st, step)
    for i, c in enumerate(cases):
        load(cases[(i + 1) % 3])
        step()  # eager work between the replays
        st.sync()
        load(c)
        graph.launch(st)
        for a, b in zip(results(), eager[i]):
            assert (a == b).all(), i


def test_refusals():
    ops = pa.Clear(pa.Stream())
    good = dict(ops=ops, heads=4, kv_heads=2, dim=64, seqs=2, pages=8)
    for bad in (dict(kv_heads=3), dict(dim=60), dict(seqs=0), dict(pages=0), dict(page_rows=24), dict(page_rows=8), dict(keep=0),
                dict(keep=20, recent=20, first=1), dict(recent=-1), dict(tokens=0), dict(dtype="f32"), dict(decay=-1.0),
                dict(table=pa.Array((10, 40, 2), "f32"))):
        with pytest.raises(ValueError):
            attention.PagedBlock(**{**good, **bad})
    blk = attention.PagedBlock(**good, tokens=20, table=pa.Array.of(clear.rotary_table(12, 64)))
    rows = pa.Array((10, 8, 64), "bf16")
    for x, counts in ((rows, (5, 4)), (rows, (10,)), (rows, (11, -1)), (pa.Array((10, 7, 64), "bf16"), (5, 5)), (pa.Array((10, 8, 32), "bf16"), (5, 5)),
                      (pa.Array((30, 8, 64), "bf16"), (15, 15)), (pa.Array((13, 8, 64), "bf16"), (13, 0))):
        with pytest.raises(ValueError):
            blk.append(x, counts)
    assert blk.lengths == [0, 0] and len(blk._free) == 8
