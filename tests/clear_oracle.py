"""The clear side's operators in 64 bits from their definitions, for the tests, with a bound on what f32 arithmetic and one
rounding to the stored type may differ from them."""
import numpy as np

# half a unit in the last place, relative, and half the smallest subnormal step
UNIT = {"bf16": 2.0 ** -8, "f16": 2.0 ** -11, "f32": 2.0 ** -24}
TINY = {"bf16": 2.0 ** -134, "f16": 2.0 ** -25, "f32": 2.0 ** -150}
E = 2.0 ** -24


def rounded(a, kind):
    """host values as the type holds them, float32"""
    from perseus_amd import clear

    a = np.asarray(a, np.float32)
    if kind == "bf16":
        return clear.from_bf16(clear.to_bf16(a))
    return a.astype(np.float16).astype(np.float32) if kind == "f16" else a


def rotary(x, positions, table, layout, inverse=False):
    """(y, magnitude): the turned heads and |a c| + |b s| (|x| where not turned); x [T][H][D]"""
    x, table = np.asarray(x, np.float64), np.asarray(table, np.float64)
    y, mag = x.copy(), np.abs(x)
    half = table.shape[1]
    rot = 2 * half
    if not half:
        return y, mag
    a, b = (slice(0, half), slice(half, rot)) if layout == "half" else (slice(0, rot, 2), slice(1, rot, 2))
    for t, p in enumerate(positions):
        if not 0 <= p < len(table):
            y[t, :, :rot] = np.nan
            continue
        c, s = table[p, :, 0], table[p, :, 1] * (-1 if inverse else 1)
        xa, xb = x[t, :, a], x[t, :, b]
        y[t, :, a], y[t, :, b] = xa * c - xb * s, xb * c + xa * s
        mag[t, :, a], mag[t, :, b] = np.abs(xa * c) + np.abs(xb * s), np.abs(xb * c) + np.abs(xa * s)
    return y, mag


def norm(x, w, eps):
    x = np.asarray(x, np.float64)
    return x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * (1 if w is None else np.asarray(w, np.float64))


def check(got, want, bound, what=""):
    """got within bound of want, NaN and infinities in the same places"""
    got, want, bound = (np.broadcast_to(np.asarray(v, np.float64), np.shape(want)) for v in (got, want, bound))
    assert (np.isnan(got) == np.isnan(want)).all(), f"{what}: NaN in other places"
    fine = np.isfinite(want)
    assert (got[~fine & ~np.isnan(want)] == want[~fine & ~np.isnan(want)]).all(), f"{what}: infinities"
    off = np.abs(got - want, where=fine, out=np.zeros(want.shape)) - np.where(fine, bound, 0)
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum())} of {off.size} past the bound, worst by {off.max():.3g}"


def rotary_bound(y, mag, kind):
    """two products, a sum (three roundings of f32) and the store's"""
    return UNIT[kind] * np.abs(y) + TINY[kind] + 4 * E * mag


def norm_rotary_bound(y, mag, kind, dim):
    """besides: the sum of dim squares (relative dim E at most, halved by the root), the mean, the root, its inverse, the
    two factors"""
    return UNIT[kind] * np.abs(y) + TINY[kind] + (dim / 2 + 16) * E * mag


def attention(q, k, v, spans, group, scale, causal):
    """spans: per sequence (query row, queries, key row, keys). (out, lse, bound of out per unit, bound of lse): out [T][H][D]
    and lse [T][H] with NaN at rows of no sequence."""
    T, H, D = q.shape
    out, lse = np.full((T, H, D), np.nan), np.full((T, H), np.nan)
    spread, dlse = np.zeros((T, H, D)), np.zeros((T, H))
    for q0, n, k0, m in spans:
        for h in range(H):
            Q = np.asarray(q[q0:q0 + n, h], np.float64)
            K, V = np.asarray(k[k0:k0 + m, h // group], np.float64), np.asarray(v[k0:k0 + m, h // group], np.float64)
            for i in range(n):
                seen = max(0, min(m, m - n + i + 1)) if causal else m
                if not seen:
                    out[q0 + i, h], lse[q0 + i, h] = 0, -np.inf
                    continue
                with np.errstate(invalid="ignore", over="ignore"):
                    z = scale * (K[:seen] @ Q[i])
                    dz = scale * (np.abs(K[:seen]) @ np.abs(Q[i]))
                    top = z.max()
                    p = np.exp(z - top)
                    total = p.sum()
                    out[q0 + i, h] = p @ V[:seen] / total
                    lse[q0 + i, h] = top + np.log(total)
                    # a score: D products summed in f32, scaled, less the maximum; an exponential of 2 units
                    d = (D + 4) * E * dz.max() + 8 * E * np.abs(z).max()
                    spread[q0 + i, h] = p @ np.abs(V[:seen]) / total
                    dlse[q0 + i, h] = d + (seen + 16) * E + 4 * E * abs(lse[q0 + i, h])
    return out, lse, spread, dlse


def attention_bound(out, spread, dlse, kind, vmax):
    """the store's rounding, each weight's rounding to the type before its product with v (relative, or half a subnormal step
    of a weight whose row's largest is 1 or more: that over a sum of 1 or more, for every key), the sums of weights and of
    products in f32 and the scores' errors (dlse, in numerator and denominator)"""
    n = 2 * dlse[..., None]
    return UNIT[kind] * np.abs(out) + TINY[kind] + spread * (UNIT[kind] + n + 4 * E) + TINY[kind] * 2.0 ** 12 * vmax


def kept(w, place, nxt, keep, recent, first):
    """the keys that stay of one (sequence, key head), and the moves (from, to) that close the gaps: weights w, places"""
    n = len(w)
    if n <= keep:
        return np.arange(n), []
    place = np.asarray(place, np.int64)
    w = np.asarray(w, np.float64)
    held = (place >= int(nxt) - recent) | (place < first)
    worth = np.where(held | np.isnan(w), -np.inf, w)  # protected keys are alike
    order = np.lexsort((np.arange(n), -worth, np.isnan(w) & ~held, ~held))
    stay = np.sort(order[:keep])
    gone = np.ones(n, bool)
    gone[stay] = False
    return stay, list(zip(stay[stay >= keep], np.flatnonzero(gone[:keep])))


def key_weights(q, k, lse, spans, group, scale, causal):
    """spans: per sequence (query row, queries, key row, keys). (sums, bound): what each key of [rows][kv heads] gathers, 0 at rows
    of no sequence, and how far f32 may be off: an exponent's D products and their sum, its scaling and the log-sum-exp's
    (each a few roundings of their sizes), an exponential of 2 units, sums of 32 at a time that are added one after the other"""
    R, KV, D = k.shape
    out, bound = np.zeros((R, KV)), np.zeros((R, KV))
    for q0, n, k0, m in spans:
        for h in range(KV * group if n and m else 0):
            g = h // group
            Q, K = np.asarray(q[q0:q0 + n, h], np.float64), np.asarray(k[k0:k0 + m, g], np.float64)
            L = np.asarray(lse[q0:q0 + n, h], np.float64)[:, None]
            with np.errstate(invalid="ignore", over="ignore"):
                z = scale * (Q @ K.T)
                dz = scale * (np.abs(Q) @ np.abs(K).T)
                sees = np.arange(m) <= m - n + np.arange(n)[:, None] if causal else np.ones((n, m), bool)
                p = np.where(sees & (L > -np.inf) | sees & np.isnan(L), np.exp(z - L), 0)
                d = (D + 4) * E * dz + 8 * E * (np.abs(z) + np.where(np.isfinite(L), np.abs(L), 0)) + 8 * E
                out[k0:k0 + m, g] += p.sum(0)
                d = np.where(p == 0, 0, d)  # at scores of -infinity d is infinite, the weight 0
                bound[k0:k0 + m, g] += (p * d).sum(0) + (n * group / 16 + 32) * E * p.sum(0)
    return out, bound
