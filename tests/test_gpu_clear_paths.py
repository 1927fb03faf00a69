"""Each kernel of the clear side's attention that a call can reach, at sizes that choose it, against the definition in 64 bits
(tests/clear_oracle.py): prompts of 64 dimensions and less by the number of their tiles, keys split at every width, among more
than 64 sequences and over tens of thousands of keys, widths between the tiles'; and the second product of token rows. Each test
prints its case before the GPU runs."""
import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import clear
from tests import clear_oracle as co
from tests.test_gpu_clear import placed, run_attention, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    assert pa.device_count() >= 1, "no GPU visible"
    return pa.Clear(pa.Stream())


def unseen(spans):
    """NaN and infinities at the last keys, which in a causal order only the last queries see"""
    def edit(q, k, v, k0):
        for s, (n, m) in zip(k0, spans):
            if m > 3:
                v[s + m - 1, 0, 3] = np.nan
                v[s + m - 2, -1, 0] = np.inf
                k[s + m - 3, 0, 1] = np.nan
    return edit


def longest(spans):
    """what a caller expects of these lengths"""
    return max(n for n, _ in spans), max(m for _, m in spans)


# dim, heads, kv heads, [(queries, keys)]
MANY_64 = [
    (64, 32, 32, [(40, 300)] * 8),                   # tiles in plenty, one in part and several whole for each
    (64, 16, 16, [(33, 64), (64, 128), (65, 191), (34, 192), (40, 193), (7, 700), (50, 449), (1, 63)] * 2),
    (48, 64, 32, [(200, 200), (129, 320), (90, 500)]),
    (32, 24, 12, [(700, 700), (650, 1000)]),
]


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("shape", range(len(MANY_64)))
def test_many_tiles_of_64_dimensions(ops, kind, causal, shape):
    """128 rows a tile, odd and even numbers of tiles of keys, whole ones and ones in part"""
    dim, heads, kv, spans = MANY_64[shape]
    say(f"[clear paths] many tiles {kind} causal {causal} dim {dim} heads {heads}/{kv} {spans}")
    run_attention(ops, kind, dim, heads, kv, spans, causal, gap=3)
    if causal:
        run_attention(ops, kind, dim, heads, kv, spans, causal, edit=unseen(spans), hints=longest(spans))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("queries,keys", [(700, 700), (705, 1111), (1000, 1000)])
def test_a_prompt_of_64_dimensions_in_tiles_of_32(ops, kind, queries, keys):
    """12 heads of 64: more tiles of 32 rows than CUs, fewer of 128"""
    say(f"[clear paths] {queries} queries over {keys} keys x 12 heads of 64, {kind}")
    for causal in (True, False):
        run_attention(ops, kind, 64, 12, 12, [(queries, keys)], causal)
    run_attention(ops, kind, 64, 12, 12, [(queries, keys)], True, edit=unseen([(queries, keys)]))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim,heads,kv,spans", [
    (64, 16, 16, [(40, 1100)] * 16), (192, 2, 2, [(200, 1500)]), (256, 4, 2, [(150, 2100), (80, 100)]), (160, 3, 1, [(70, 1030)]),
    (96, 6, 2, [(90, 1700)]), (128, 4, 4, [(129, 20000)])])
def test_many_rows_with_their_keys_split(ops, kind, dim, heads, kv, spans):
    say(f"[clear paths] split keys {kind} dim {dim} heads {heads}/{kv} {spans}")
    for causal in (True, False):
        run_attention(ops, kind, dim, heads, kv, spans, causal, hints=longest(spans))
    run_attention(ops, kind, dim, heads, kv, spans, True, edit=unseen(spans), hints=longest(spans))


@pytest.mark.parametrize("dim,heads,kv,spans", [
    (64, 4, 1, [(1, 900)] * 70), (128, 4, 1, [(1, 900), (2, 1), (0, 50), (1, 0), (1, 800)] * 15), (72, 4, 1, [(40, 1100)] * 70),
    (72, 4, 1, [(40, 1100), (3, 9), (41, 512), (0, 0), (33, 1025)] * 14)])
def test_split_keys_of_more_than_64_sequences(ops, dim, heads, kv, spans):
    say(f"[clear paths] {len(spans)} sequences with their keys split, dim {dim} heads {heads}/{kv} {spans[:5]}")
    run_attention(ops, "bf16", dim, heads, kv, spans, True, hints=longest(spans))
    run_attention(ops, "f16", dim, heads, kv, spans, False, gap=2, hints=longest(spans))


@pytest.mark.parametrize("dim,heads,kv,spans", [
    (128, 8, 1, [(1, 20001)]), (64, 6, 2, [(9, 30000)]), (256, 2, 1, [(2, 17000), (1, 9)]), (80, 32, 2, [(2, 12345)])])
def test_few_rows_over_tens_of_thousands_of_keys(ops, dim, heads, kv, spans):
    say(f"[clear paths] few rows dim {dim} heads {heads}/{kv} {spans}")
    run_attention(ops, "bf16", dim, heads, kv, spans, True, hints=longest(spans))
    run_attention(ops, "f16", dim, heads, kv, spans, True, hints=longest(spans))


@pytest.mark.parametrize("kind", ["bf16", "f16"])
@pytest.mark.parametrize("dim", [24, 56, 88, 104, 112, 120, 144, 184, 232, 248])
def test_widths_between_the_tiles(ops, kind, dim):
    say(f"[clear paths] dim {dim} {kind}")
    for spans, heads, kv in (([(1, 130), (2, 33), (1, 1)], 6, 3), ([(150, 150), (64, 300)], 3, 3)):
        for order in ("rows", "padded"):
            run_attention(ops, kind, dim, heads, kv, spans, True, order=order)


# ---------------------------------------------------------------------------------------------------- the second product


def once(x, kind):
    """weights as the type holds them, from 64 bits"""
    return co.rounded(x, kind).astype(np.float64)


@pytest.mark.parametrize("kind,keys", [("bf16", 2), ("bf16", 300), ("bf16", 2500), ("f16", 2), ("f16", 300), ("f16", 800)])
@pytest.mark.parametrize("dim,heads,kv,queries", [(64, 4, 4, 1), (64, 32, 1, 1), (80, 8, 2, 3), (128, 8, 1, 2), (192, 2, 2, 1), (256, 4, 2, 1)])
def test_the_rows_of_tokens_take_their_weights_whole(ops, kind, keys, dim, heads, kv, queries):
    """Half the keys have the weight 1, half one in the middle between two that the type holds, with values that cancel but for a
    thousandth: a weight rounded once would leave more of its rounding than of the answer. The product of what the rounding leaves
    takes the error to the rounding of that, the square of the type's unit; f16 ends at 2^-32 of the largest weight."""
    say(f"[clear paths] weights of tokens {kind}, {keys} keys, {queries} queries x {heads}/{kv} heads of {dim}")
    rng = np.random.default_rng(keys + dim)
    unit = co.UNIT[kind]
    w = 0.75 + unit / 2
    scale = -np.log(w)
    q, k = np.zeros((queries, heads, dim), np.float32), np.zeros((keys, kv, dim), np.float32)
    q[..., 0] = 1
    second = np.arange(keys) % 2 == 1
    k[second, :, 0] = -1
    sign = np.float32(2.0) ** rng.integers(-2, 3, (kv, dim)) * rng.choice([-1, 1], (kv, dim))
    v = np.where(second[:, None, None], -1.0, 0.75) * sign
    dq, dk, dv = (placed(a.astype(np.float32), kind) for a in (q, k, v))
    out, lse = pa.Array((queries, heads, dim), kind), pa.Array((queries, heads), "f32")
    # every query sees every key: the cancellation is the same for all
    ops.attention(dq, dk, dv, pa.Array.of(np.array([0, queries]), "i32"), pa.Array.of(np.zeros(1), "i64"),
                  pa.Array.of(np.array([keys]), "i32"), out, lse, scale=scale, causal=False)
    want, wl, spread, dlse = co.attention(q, k, v, [(0, queries, 0, keys)], heads // kv, np.float32(scale), False)
    bound = (unit * np.abs(want) + co.TINY[kind] + spread * (unit ** 2 + 2 * dlse[..., None] + 4 * co.E) +
             (keys * 2.0 ** -32 * 4 if kind == "f16" else 0))
    # the same on the host with the weights rounded once is past the bound
    p = np.where(second, np.exp(-np.float64(np.float32(scale))), 1.0)
    rough = np.einsum("k,kgd->gd", once(p, kind), v) / p.sum()
    assert (np.abs(rough - want[0, ::heads // kv]) > bound[0, ::heads // kv]).all()
    co.check(out.numpy(ops.stream), want, bound, "out")
    co.check(lse.numpy(ops.stream), wl, dlse, "lse")


# ---------------------------------------------------------------------------------------------------- norms


@pytest.mark.parametrize("kind", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("dim,heads,kv,tokens,order", [(64, 4, 2, 33, "rows"), (128, 3, 3, 5, "padded"), (30, 2, 1, 7, "rows")])
def test_values_copied_without_slots(ops, kind, dim, heads, kv, tokens, order):
    """row t of k and v to row t, v into a tensor of its own"""
    say(f"[clear paths] qk_norm_rotary with values, no slots, {kind} dim {dim} {heads}/{kv} heads {tokens} tokens {order}")
    rng = np.random.default_rng(dim)
    q, k, v = (co.rounded(rng.normal(size=(tokens, h, dim)), kind) for h in (heads, kv, kv))
    rot = dim // 2 // 2 * 2
    table, pos = clear.rotary_table(60, rot), rng.integers(0, 60, tokens)
    dq, dk, dv = (placed(a, kind, order) for a in (q, k, v))
    ko, vo = (placed(np.full_like(k, 3), kind, order) for _ in range(2))
    ops.qk_norm_rotary(dq, dk, None, None, pa.Array.of(pos, "i32"), pa.Array.of(table), dq, ko, eps=1e-5, v=dv, v_out=vo)
    for got, x in ((dq, q), (ko, k)):
        y, mag = co.rotary(co.norm(x, None, 1e-5), pos, table, "half")
        co.check(got.numpy(ops.stream), y, co.norm_rotary_bound(y, mag, kind, dim))
    assert (vo.numpy(ops.stream) == v).all()
