"""The clear side's attention and rotary positions on the GPU at the ends of their ranges, against their definitions in 64 bits
(tests/clear_oracle.py). Each test prints its case before the GPU runs."""
import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import clear
from tests import clear_oracle as co
from tests.test_gpu_clear import placed, say

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


def attend(ops, kind, q, k, v, causal=True, scale=1.0, order="rows"):
    """one sequence: (out, lse, and the oracle's out, lse, bounds' parts)"""
    T, H, D = q.shape
    dq, dk, dv = (placed(a, kind, order) for a in (q, k, v))
    out, lse = placed(np.full((T, H, D), 9.0), kind, order), pa.Array((T, H), "f32")
    ops.attention(dq, dk, dv, pa.Array.of(np.array([0, T]), "i32"), pa.Array.of(np.zeros(1), "i64"),
                  pa.Array.of(np.array([len(k)]), "i32"), out, lse, scale=scale, causal=causal)
    return (out.numpy(ops.stream), lse.numpy(ops.stream)) + co.attention(q, k, v, [(0, T, 0, len(k))], H // k.shape[1], scale,
                                                                         causal)


def small_weights_bound(out, spread, dlse, lost, twice):
    """f16: the store's rounding; each weight's, relative, or (twice: what it leaves is a second product) its square; what falls
    below half a subnormal step; the scores' errors and the f32 sums"""
    u = co.UNIT["f16"]
    n = 2 * dlse[..., None]
    return u * np.abs(out) + co.TINY["f16"] + spread * ((u * u if twice else u) + n + 4 * co.E) + lost


@pytest.mark.parametrize("queries,dim,keys,above", [
    (1, 64, 131072, 17.5), (1, 128, 131072, 17.5), (2, 256, 60000, 17.0), (1, 64, 2000, 16.5), (200, 128, 100000, 17.5),
    (150, 192, 40000, 17.0), (300, 64, 3000, 17.5), (1100, 32, 1100, 17.5)])
def test_f16_attention_of_many_small_weights(ops, queries, dim, keys, above):
    """one key in 32 far above the others, with a value of 0: the output is made of the others' weights, and none may be lost,
    though each is below what f16 holds beside 1. A row's largest weight is 2^7 or more, so that half a subnormal step is 2^-32 of
    it, for each key, over the sum of the weights."""
    say(f"[clear] attention f16, {keys} keys, one in 32 {above} nats above the others, {queries} queries, dim {dim}")
    rng = np.random.default_rng(keys + dim)
    heads = 12 if dim == 32 else 1
    q = np.zeros((queries, heads, dim), np.float32)
    q[..., 0] = 4
    k = np.zeros((keys, heads, dim), np.float32)
    v = co.rounded(1000 * (1 + 0.25 * rng.random((keys, heads, dim))), "f16")
    k[31::32, :, 0] = co.rounded(above / 4, "f16")
    v[31::32] = 0
    got, gl, want, wl, spread, dlse = attend(ops, "f16", q, k, v, causal=False)
    lost = keys * 2.0 ** -32 * 1250 / (keys // 32)
    co.check(got, want, small_weights_bound(want, spread, dlse, lost, queries <= 32), "out")
    co.check(gl, wl, dlse, "lse")


@pytest.mark.parametrize("queries,dim", [(1, 64), (3, 128), (200, 128), (300, 64), (150, 256)])
@pytest.mark.parametrize("step", [7.9, 8.1, 15.0])
def test_f16_attention_where_the_maximum_grows_late(ops, queries, dim, step):
    """the last keys, which are taken first, lie `step` powers of two below the first ones: weights beyond 1 while the running
    maximum lags behind must not leave f16"""
    say(f"[clear] attention f16, maxima that grow by 2^{step}, {queries} queries, dim {dim}")
    keys, rng = 700, np.random.default_rng(dim)
    q = np.zeros((queries, 1, dim), np.float32)
    q[..., 0] = 4
    k = np.zeros((keys, 1, dim), np.float32)
    k[:64, 0, 0] = co.rounded(step * np.log(2) / 4, "f16")
    v = co.rounded(rng.normal(size=(keys, 1, dim)) * 1000, "f16")
    got, gl, want, wl, spread, dlse = attend(ops, "f16", q, k, v)
    co.check(got, want, small_weights_bound(want, spread, dlse, keys * 2.0 ** -32 * 4e3, queries <= 32), "out")
    co.check(gl, wl, dlse, "lse")


def test_rotary_of_more_tokens_than_one_grid_takes(ops):
    """67 million tokens of one short head: 2^24 workgroups of 256 threads and more, which no launch takes"""
    dim, period, times = 8, 50021, 1342
    say(f"[clear] rotary of {period * times} tokens of one head of {dim}")
    rng = np.random.default_rng(8)
    x = co.rounded(rng.normal(size=(period, 1, dim)), "bf16")
    pos = rng.integers(0, 100, period).astype(np.int32)
    table = clear.rotary_table(100, dim)
    words = clear.to_bf16(x).reshape(-1).view(np.uint32)
    d = pa.Array((period * times, 1, dim), "bf16")
    d.buf.upload(np.tile(words, times))
    ops.rotary(d, pa.Array.of(np.tile(pos, times), "i32"), pa.Array.of(table), d, layout="interleaved")
    got = d.buf.download(stream=ops.stream).reshape(times, -1)
    assert (got == got[0]).all(), "the same rows at the same places turned differently"
    y, mag = co.rotary(x, pos, table, "interleaved")
    co.check(clear.from_bf16(got[0].view(np.uint16)).reshape(x.shape), y, co.rotary_bound(y, mag, "bf16"))


def cut(a, kind, token, head, base=0):
    """host values [T][H][D] on the device with the strides that are given, NaN around them"""
    x = pa.Array(a.shape, kind, strides=(token, head, 1))
    flat = np.full(2 * x.buf.words, np.nan, np.float32)
    np.lib.stride_tricks.as_strided(flat, a.shape, [4 * token, 4 * head, 4])[...] = a
    raw = clear.to_bf16(flat) if kind == "bf16" else flat.astype(np.float16)
    x.buf.upload(raw.view(np.uint32))
    return x


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [64, 80])
def test_strides_of_single_tokens_and_heads_do_not_matter(ops, kind, dim):
    """one token, one head, one key row, as views out of tensors with strides of any kind leave them"""
    say(f"[clear] strides of dimensions of size 1, {kind} dim {dim}")
    rng = np.random.default_rng(dim)
    for T, H, KV, R, qt, qh, kt, kh in ((1, 4, 2, 9, 4 * dim + 3, dim, 2 * dim, dim), (3, 1, 1, 40, dim, 5, 2 * dim + 8, 7),
                                        (1, 1, 1, 1, 1, 3, 2 ** 22 + 1, 1), (1, 1, 1, 1, 2 ** 40 + 1, 2 ** 41, 2 ** 40, 2 ** 50),
                                        (1, 6, 1, 33, 3, dim + 8, dim, 1), (150, 1, 1, 150, dim, 9, dim, 9)):
        q, k, v = (co.rounded(rng.normal(size=s), kind) for s in ((T, H, dim), (R, KV, dim), (R, KV, dim)))
        dq, dk, dv, out = cut(q, kind, qt, qh), cut(k, kind, kt, kh), cut(v, kind, kt, kh), cut(0 * q, kind, qt, qh)
        lse = pa.Array((T, H), "f32")
        ops.attention(dq, dk, dv, pa.Array.of(np.array([0, T]), "i32"), pa.Array.of(np.zeros(1), "i64"),
                      pa.Array.of(np.array([R]), "i32"), out, lse)
        want, wl, spread, dlse = co.attention(q, k, v, [(0, T, 0, R)], H // KV, dim ** -0.5, True)
        co.check(out.numpy(ops.stream), want, co.attention_bound(want, spread, dlse, kind, 5.0), f"out {T} {H} {R}")
        co.check(lse.numpy(ops.stream), wl, dlse, "lse")
    table, pos = clear.rotary_table(40, dim), np.array([33])
    for H, token, head in ((3, 5, dim), (1, 2 ** 40 + 3, 7)):
        x = co.rounded(rng.normal(size=(1, H, dim)), kind)
        d = cut(x, kind, token, head)
        ops.rotary(d, pa.Array.of(pos, "i32"), pa.Array.of(table), d)
        y, mag = co.rotary(x, pos, table, "half")
        co.check(d.numpy(ops.stream), y, co.rotary_bound(y, mag, kind), f"rotary {H}")


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim,queries,keys,step", [(128, 200, 70, 0), (128, 200, 600, 8), (64, 100, 45, 0), (64, 1, 45, 0), (256, 150, 33, 16), (64, 130, 97, 0)])
def test_attention_over_values_that_share_memory(ops, kind, dim, queries, keys, step):
    """one row of values for every key (a token stride of 0), or rows a few values apart: what is read past the last key of a
    tile are the seen values again, an infinite one among them, and they must count nothing"""
    say(f"[clear] attention {kind} over values {step} apart, {queries} queries, {keys} keys, dim {dim}")
    rng = np.random.default_rng(dim + keys)
    q, k = (co.rounded(rng.normal(size=(n, 1, dim)), kind) for n in (queries, keys))
    flat = co.rounded(rng.normal(size=dim + step * (keys - 1) + 2), kind)
    flat[3], flat[dim - 1] = np.inf, -np.inf
    buf = pa.Array.of(flat, kind).buf
    dv = pa.Array((keys, 1, dim), kind, buf, strides=(step, dim, 1))
    v = np.lib.stride_tricks.as_strided(flat, (keys, 1, dim), (4 * step, 4 * dim, 4))
    for causal in (False, True):
        out, lse = pa.Array((queries, 1, dim), kind), pa.Array((queries, 1), "f32")
        ops.attention(pa.Array.of(q, kind), pa.Array.of(k, kind), dv, pa.Array.of(np.array([0, queries]), "i32"),
                      pa.Array.of(np.zeros(1), "i64"), pa.Array.of(np.array([keys]), "i32"), out, lse, causal=causal)
        want, wl, spread, dlse = co.attention(q, k, v, [(0, queries, 0, keys)], 1, dim ** -0.5, causal)
        co.check(out.numpy(ops.stream), want, co.attention_bound(want, spread, dlse, kind, 5.0), f"out, causal {causal}")
        co.check(lse.numpy(ops.stream), wl, dlse, "lse")
