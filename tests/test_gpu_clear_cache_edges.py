"""The cache's operators at the edges of what their header allows: sequences without queries beside keys that hold infinities and NaN,
runs of as many keys as there are numbers, weights and places past 32 bits of offset, calls of two streams. Each test prints its case before the GPU runs."""
import sys

import numpy as np
import pytest

import perseus_amd as pa
from tests import clear_oracle as co
from tests.test_gpu_clear_evict import spread
from tests.test_gpu_clear_weights import run_weights

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ops():
    assert pa.device_count() >= 1, "no GPU visible"
    return pa.Clear(pa.Stream())


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("page_rows", [0, 16])
@pytest.mark.parametrize("dim,heads,kv", [(64, 4, 2), (80, 6, 2), (128, 2, 2), (256, 4, 1)])
def test_key_weights_of_sequences_without_queries(ops, kind, page_rows, dim, heads, kv):
    """keys that no query of the call sees weigh decay times what they did, whatever they hold, by either kernel"""
    say(f"[clear] key_weights, sequences without queries, {kind} dim {dim} heads {heads}/{kv} pages of {page_rows}")

    for spans in ([(0, 40)], [(1, 70), (0, 40), (2, 90), (0, 300)], [(0, 40), (50, 60), (0, 1)]):
        def edit(q, k, k0):
            for b, (n, m) in enumerate(spans):
                if not n:
                    for j, x in ((0, np.inf), (m // 2, -np.inf), (m - 1, np.nan)):
                        k[k0[b] + j, 0, dim // 2] = x

        for hints in (None, (1, 300), (4096, 300)):  # tokens' kernel, a prompt's
            for causal in (True, False):
                got = run_weights(ops, kind, dim, heads, kv, spans, causal, page_rows, hints=hints, edit=edit)
                assert np.isfinite(got).all()
                run_weights(ops, kind, dim, heads, kv, spans, causal, page_rows, hints=hints, edit=edit, inplace=True, new=True)


@pytest.mark.parametrize("sliced", [True, False])
def test_evict_of_as_many_keys_as_there_are_numbers(sliced):
    """2^31 - 1 keys, the most of a run: pages of one pool again and again, weights above all others in two of them, the last key's
    among them; in slices, and by one workgroup that expects few keys"""
    say(f"[clear] evict of 2^31 - 1 keys, in slices: {sliced}")
    ops = pa.Clear(pa.Stream(), workspace=64 << 20 if sliced else 0)
    page, pool, n, keep, high = 1 << 20, 8, 2 ** 31 - 1, 1500, 1000
    rng = np.random.default_rng(3)
    w = rng.random((pool, page), np.float32)
    w[-1, -high:] = 10 + rng.permutation(high) / np.float32(high)  # on the pool's last page: no two alike
    table = (np.arange(2048) % (pool - 1)).astype(np.int32)
    table[[5, 2047]] = pool - 1
    moves, count, kept = pa.Array.of(np.full((1, 1, keep, 2), -9, np.int32)), pa.Array.of(np.zeros((1, 1), np.int32)), pa.Array.of(np.zeros(1, np.int32))
    ops.evict(pa.Array.of(w.reshape(-1, 1)), pa.Array.of(np.array([n]), "i32"), keep, moves, count, pages=pa.Array.of(table[None]),
              page_rows=page, kept_len=kept, max_k=n if sliced else 5000)
    j = np.concatenate([e * page + np.arange(page - high, page) for e in (5, 2047)])[:-1]  # the last row has no key
    stay = np.sort(j[np.lexsort((j, -w[-1, j % page]))[:keep]])
    got = moves.numpy(ops.stream)[0, 0]
    assert count.numpy(ops.stream)[0, 0] == keep == kept.numpy(ops.stream)[0]
    assert (got[:, 0] == stay).all() and (got[:, 1] == np.arange(keep)).all()


@pytest.mark.parametrize("page_rows", [0, 16])
@pytest.mark.parametrize("n,keep", [(900, 700), (5000, 3100), (6000, 1000), (17000, 5000)])
def test_evict_of_weights_and_places_past_32_bits_of_offset(ops, n, keep, page_rows):
    """rows of weights and places 1024 words apart, the keys in the last of 1.3 million: a word a lane, 5, 16, and in slices"""
    say(f"[clear] evict of {n} keys far into 5.3 GB of weights and places, pages of {page_rows}")
    rows, kv, apart, recent, first = 1_300_000, 2, 1024, 50, 3
    rng = np.random.default_rng(n)
    begin = (rows - n) // 16 * 16
    buf = pa.DevBuf(rows * apart)
    w, p = pa.Array((rows, kv), "f32", buf, 0, (apart, 1)), pa.Array((rows, kv), "i32", buf, 500, (apart, 2))
    if page_rows:
        pages = begin // 16 + rng.permutation(-(-n // 16))
        at = (pages[np.arange(n) // 16] * 16 + np.arange(n) % 16) - begin
        where = dict(pages=pa.Array.of(pages[None].astype(np.int32)), page_rows=16)
    else:
        at, where = np.arange(n), dict(k_start=pa.Array.of(np.array([begin], np.int64)))
    weights, places = spread(rng, n * kv).reshape(n, kv).astype(np.float32), np.stack([rng.permutation(n) for _ in range(kv)], 1)
    tail = np.zeros((rows - begin, apart), np.uint32)
    tail[at, :kv] = weights.view(np.uint32)
    tail[at, 500:500 + 2 * kv:2] = places
    buf.upload(tail, ops.stream, begin * apart)
    most = min(keep, n - keep)
    moves, count = pa.Array.of(np.full((1, kv, most, 2), -9, np.int32)), pa.Array.of(np.full((1, kv), -9, np.int32))
    ops.evict(w, pa.Array.of(np.array([n]), "i32"), keep, moves, count, places=p, recent=recent, first=first, max_k=n, **where)
    got, number = moves.numpy(ops.stream)[0], count.numpy(ops.stream)[0]
    for g in range(kv):
        want = np.array(co.kept(weights[:, g], places[:, g], n, keep, recent, first)[1])
        assert number[g] == len(want) and (got[g, :len(want)] == want).all() and (got[g, len(want):] == -9).all()


def test_calls_of_two_streams_leave_out_no_write():
    """split weights and the choice of a long cache on two streams at once, over weights and lists that hold another value before each
    round: what each stream's calls write alone, and nothing past it"""
    say("[clear] key_weights and evict on two streams at once, over cleared outputs")
    H, KV, D, n, m, keep = 8, 2, 64, 700, 20000, 5000
    sides = []
    for seed in (1, 2):
        rng = np.random.default_rng(seed)
        k0 = pa.Array.of(np.zeros(1, np.int64))
        outs = [pa.Array((n, KV), "f32"), pa.Array((1, KV, keep, 2), "i32"), pa.Array((1, KV), "i32")]
        first = (pa.Array.of(rng.normal(size=(n, H, D)), "bf16"), pa.Array.of(rng.normal(size=(n, KV, D)), "bf16"),
                 pa.Array.of((rng.random((n, H)) + 6).astype(np.float32)), pa.Array.of(np.array([0, n]), "i32"),
                 pa.Array.of(np.array([n]), "i32"), outs[0])
        second = (pa.Array.of(rng.random((m, KV)).astype(np.float32)), pa.Array.of(np.array([m]), "i32"), keep, *outs[1:])
        sides.append((pa.Clear(pa.Stream()), first, second, k0, outs))

    def clear_outputs(side):
        for x in side[-1]:
            x.buf.upload(np.full(x.buf.words, np.uint32(0xC2C8C2C8), np.uint32), side[0].stream)  # -100.4 as f32

    def call(side):
        ops, first, second, k0, _ = side
        ops.key_weights(*first, k_start=k0)
        ops.evict(*second, k_start=k0)

    def answers(side):
        return [x.numpy(side[0].stream) for x in side[-1]]

    alone = []
    for side in sides:
        clear_outputs(side)
        call(side)
        alone.append(answers(side))
        weights, moves, count = alone[-1]
        assert (weights >= 0).all() and ((count > 0) & (count <= keep)).all()
        for g in range(KV):
            assert (moves[0, g, :count[0, g]] >= 0).all() and (moves[0, g, count[0, g]:] < 0).all()
    for _ in range(20):
        for side in sides:
            clear_outputs(side)
        for side in sides:
            call(side)
        for side, want in zip(sides, alone):
            assert all(np.array_equal(x, y) for x, y in zip(answers(side), want))
