"""The clear side and the encrypted scoring together, as a program uses them (12 heads x 64, 512 tokens, N = 2^16): a prompt of 511
tokens and one token through attention.ClearBlock; its cached keys packed, encoded and encrypted, its last query the scoring's
plaintext. The decrypted scores match q . K in 64 bits, and the clear attention's log-sum-exp turns them into the probabilities
whose average of the cached values is the clear attention's output."""
import sys

import numpy as np
import pytest

import perseus_amd as pa
from perseus_amd import attention, clear, encoding
from tests import clear_oracle as co
from tests import twin
from tests.test_oracle_ks import decrypt, encrypt

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


def test_encrypted_scores_of_clear_keys_and_queries():
    say("[clear attention] prompt of 511 tokens, one token, 6 ciphertexts of keys scored")
    assert pa.device_count() >= 1, "no GPU visible"
    H, D, T = attention.HEADS, attention.HEAD_DIM, attention.TOKENS
    st = pa.Stream()
    ops = pa.Clear(st)
    rng = np.random.default_rng(11)
    rows = co.rounded(rng.normal(size=(T, 3 * H, D)), "bf16")
    w = (1 + 0.1 * rng.normal(size=(2, D))).astype(np.float32)
    block = attention.ClearBlock(ops, H, H, D, T, table=pa.Array.of(clear.rotary_table(T, D)), q_weight=pa.Array.of(w[0]),
                                 k_weight=pa.Array.of(w[1]))
    block.append(pa.Array.of(rows[:T - 1], "bf16"))
    q, out, lse = block.append(pa.Array.of(rows[T - 1:], "bf16"))
    q, out, lse = q.numpy(st)[0].astype(np.float64), out.numpy(st)[0], lse.numpy(st)[0]
    K, V = block.keys().astype(np.float64), block.v.numpy(st).astype(np.float64)
    table = clear.rotary_table(T, D)
    for got, x, weight in ((block.q.numpy(st), rows[:, :H], w[0]), (K.reshape(T, H, D), rows[:, H:2 * H], w[1])):
        y, mag = co.rotary(co.norm(x, weight, 1e-6), np.arange(T), table, "half")
        co.check(got, y, co.norm_rotary_bound(y, mag, "bf16", D))
    assert (V == rows[:, 2 * H:]).all()

    ch = pa.preset("c4")
    ctx = pa.Context(ch, k_rot=1)
    oc = twin.Ctx(ch.logn, ch.q, ch.p, ch.dnum)
    n, top = ch.n, len(ch.q) - 1
    g = twin.Prng([77, 1, 2, 3, 4, 5, 6, 7], 0)
    s = g.sparse_ternary(n, 192)
    s_eval = oc.secret_eval(s)
    gals = [twin.rotation_galois(r, n) for r in attention.ladder_steps()]
    seeds = np.stack([g.ksk_seed() for _ in gals])
    errs = np.stack([np.stack([g.gaussian(n) for _ in range(ch.dnum)]) for _ in gals])
    keys = pa.Keys(ctx, gals, seeds=seeds, secret=s, errors=errs)
    delta, ptscale = 2.0 ** 40, float(ch.q[top]) * float(ch.q[top - 1])
    zs, tmp, dst = [], ctx.ct_buf(1), ctx.ct_buf(1)
    for z, qz in zip(attention.key_slots(K, n), attention.query_slots(q, n)):
        ct, _ = encrypt(oc, s_eval, np.rint(encoding.encode(z, n, delta)).astype(np.int64), rng, top)
        pt = np.zeros((ch.rows, n), np.uint32)
        pt[:top + 1] = oc.ntt_fwd(encoding.to_residues(encoding.encode(qz, n, ptscale), ch.primes[:top + 1]),
                                  list(range(top + 1)))
        bct, bpt = pa.DevBuf.from_array(ct), pa.DevBuf.from_array(pt)
        attention.score(ctx, keys, bct, bpt, top, dst, tmp, st)
        st.sync()
        coef = encoding.from_residues(decrypt(oc, s_eval, dst.download((2, ch.rows, n)), top - 2), ch.primes[:top - 1])
        zs.append(encoding.decode(coef, n, delta))
    scores = attention.scores_from_slots(zs)
    want = np.einsum("hd,thd->ht", q, K.reshape(T, H, D))
    err = np.abs(scores - want).max()
    say(f"[clear attention] max |score error| = {err:.3g} (scores up to {np.abs(want).max():.1f})")
    assert err < 1e-3
    p = np.exp(scores / np.sqrt(D) - lse[:, None])
    # a score off by 1e-3 moves a probability by 1e-3 / 8 of itself; the log-sum-exp's own error is far below
    assert np.abs(p.sum(1) - 1).max() < 2.5e-4
    mean, spread = np.einsum("ht,thd->hd", p, V), np.einsum("ht,thd->hd", p, np.abs(V))
    co.check(out, mean, co.UNIT["bf16"] * np.abs(mean) + (co.UNIT["bf16"] + 2.5e-4) * spread)


def test_clear_block_in_chunks_is_the_block_at_once():
    """tokens in chunks of any size give the queries and keys of one call to the bit, and attention within its rounding"""
    say("[clear attention] 200 tokens at once and in chunks, grouped heads")
    st = pa.Stream()
    ops = pa.Clear(st)
    rng = np.random.default_rng(3)
    H, KV, D, T = 6, 2, 80, 200
    rows = co.rounded(rng.normal(size=(T, H + 2 * KV, D)), "f16")
    table = pa.Array.of(clear.rotary_table(T, 48, scaling=("by_turns", 4, 64, 1, 4)))
    a, b = (attention.ClearBlock(ops, H, KV, D, T, "f16", table, "interleaved") for _ in range(2))
    a.append(pa.Array.of(rows, "f16"))
    at = 0
    for n in (1, 37, 1, 100, 60, 1):
        q, out, lse = b.append(pa.Array.of(rows[at:at + n], "f16"))
        assert q.shape == (n, H, D) and lse.shape == (n, H)
        at += n
    for x, y in ((a.q, b.q), (a.k, b.k), (a.v, b.v)):
        assert (x.numpy(st) == y.numpy(st)).all()
    want, wl, spread, dlse = co.attention(a.q.numpy(st), a.k.numpy(st), a.v.numpy(st), [(0, T, 0, T)], H // KV, D ** -0.5, True)
    for blk in (a, b):
        co.check(blk.out.numpy(st), want, co.attention_bound(want, spread, dlse, "f16", 5.0))
        co.check(blk.lse.numpy(st), wl, dlse)
    with pytest.raises(ValueError):
        b.append(pa.Array.of(rows[:1], "f16"))
    with pytest.raises(ValueError):
        attention.ClearBlock(ops, H, KV, D, T, "f16", table).append(pa.Array.of(rows[:1, :9], "f16"))
