"""The cache's operators at the edges of what their header allows: sequences without queries beside keys that hold infinities and NaN,
runs of as many keys as there are numbers. Each test prints its case before the GPU runs."""
import sys

import numpy as np
import pytest

import perseus_amd as pa
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
