"""The cache's operators at the edges of what their header allows: sequences without queries beside keys that hold infinities and NaN.
Each test prints its case before the GPU runs."""
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
