"""The clear side's attention and rotary positions on the GPU at the ends of their ranges, against their definitions in 64 bits
(tests/clear_oracle.py). Each test prints its case before the GPU runs."""
import numpy as np
import pytest

import perseus_amd as pa
from tests import clear_oracle as co
from tests.test_gpu_clear import say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert pa.device_count() >= 1, "no GPU visible"
    return pa.Clear(pa.Stream())


@pytest.mark.parametrize("dim,queries,causal", [(8, 1, True), (8, 1, False), (72, 200, True), (72, 200, False), (136, 200, True)])
@pytest.mark.parametrize("short", [0, 30, 62])
def test_attention_of_key_runs_up_to_31_bits(ops, dim, queries, causal, short):
    """2^31 - 1 keys and a few less, all one row in memory (a token stride of 0): one query, and tiles of many. Scores of zero give
    every key the weight 1, whose sums are whole numbers and whose products with powers of two are exact up to the join of 256
    parts: the output is the row itself, the log-sum-exp the log of the keys seen."""
    keys = 2 ** 31 - 1 - short
    say(f"[clear] attention of {queries} queries over {keys} keys, dim {dim} causal {causal}")
    row = np.resize(np.float32([1, 2, -1, 0, 4, -8, 0.5]), dim)
    x = pa.Array.of(row, "f16")
    cache = pa.Array((2 ** 31 - 1, 1, dim), "f16", x.buf, strides=(0, dim, 1))
    q, out = pa.Array.of(np.zeros((queries, 1, dim)), "f16"), pa.Array.of(np.full((queries, 1, dim), 9.0), "f16")
    lse = pa.Array((queries, 1), "f32")
    ops.attention(q, cache, cache, pa.Array.of(np.array([0, queries]), "i32"), pa.Array.of(np.zeros(1), "i64"),
                  pa.Array.of(np.array([keys]), "i32"), out, lse, causal=causal)
    seen = keys - (queries - 1 - np.arange(queries)) if causal else np.full(queries, keys)
    want = np.broadcast_to(row.astype(np.float64), (queries, 1, dim))
    # 256 parts of either sum joined in f32, a division and the store's rounding; the logarithm's own error
    co.check(out.numpy(ops.stream), want, (co.UNIT["f16"] + 600 * co.E) * np.abs(want), "out")
    co.check(lse.numpy(ops.stream), np.log(seen)[:, None], 600 * co.E + 4 * co.E * 22, "lse")
