"""Encrypted attention scoring for a GPT-2-small-shaped decode step (12 heads of 64 dimensions, d_model 768, a KV cache
of 512 tokens): the keys K live encrypted in HBM, the query q is a plaintext, and the scores s[h][t] = sum_d q[h][d]
K[t][64 h + d] come out encrypted, one per slot. The operation sequence is the reference's scoring recipe
(crates/pc-gpu/src/ops.rs:927-951 mult_pt, crates/pc-gpu/src/rescale.rs:230-264, crates/pc-gpu/src/rotate.rs:924-992
rotate_and_sum): per ciphertext a plaintext product, a two-prime rescale back to the ciphertext's scale, and the
log-step rotate-and-sum over each 64-slot head block.

Packing (complex, two real vectors per ciphertext): N/2 = 2^15 slots hold 512 blocks of 64; ciphertext c carries heads
2c and 2c + 1, block (hl, t) = 256 hl + t for t < 256, its real part token t and its imaginary part token t + 256, slot
64 block + d the key's dimension d. The query plaintext repeats q[h] over its head's blocks (a real multiplier, so it
scales both parts alike). After the sums, slot 64 block holds s[h][t] + i s[h][t + 256]."""
import numpy as np

HEADS, HEAD_DIM, TOKENS = 12, 64, 512
BLOCK = HEAD_DIM
HEADS_PER_CT = 2
TOK_PER_PART = TOKENS // 2


def n_cts():
    return HEADS // HEADS_PER_CT


def key_slots(K, n):
    """The ciphertexts' slot vectors (N/2 complex each) of the key matrix K [TOKENS][HEADS * HEAD_DIM]."""
    assert n // 2 == HEADS_PER_CT * TOK_PER_PART * BLOCK, "the packing fills N/2 slots at N = 2^16"
    out = []
    for c in range(n_cts()):
        z = np.zeros(n // 2, np.complex128)
        for hl in range(HEADS_PER_CT):
            h = HEADS_PER_CT * c + hl
            blk = K[:, h * HEAD_DIM:(h + 1) * HEAD_DIM]  # [TOKENS][64]
            part = blk[:TOK_PER_PART] + 1j * blk[TOK_PER_PART:]
            z[hl * TOK_PER_PART * BLOCK:(hl + 1) * TOK_PER_PART * BLOCK] = part.reshape(-1)
        out.append(z)
    return out


def query_slots(q, n):
    """The plaintexts' slot vectors (real) of the query q [HEADS][HEAD_DIM], one per ciphertext."""
    out = []
    for c in range(n_cts()):
        z = np.zeros(n // 2, np.float64)
        for hl in range(HEADS_PER_CT):
            h = HEADS_PER_CT * c + hl
            z[hl * TOK_PER_PART * BLOCK:(hl + 1) * TOK_PER_PART * BLOCK] = np.tile(q[h], TOK_PER_PART)
        out.append(z)
    return out


def scores_from_slots(zs):
    """s [HEADS][TOKENS] from the decrypted, decoded slot vectors of the ciphertexts."""
    s = np.zeros((HEADS, TOKENS))
    for c, z in enumerate(zs):
        for hl in range(HEADS_PER_CT):
            h = HEADS_PER_CT * c + hl
            v = z[hl * TOK_PER_PART * BLOCK:(hl + 1) * TOK_PER_PART * BLOCK:BLOCK]
            s[h, :TOK_PER_PART] = v.real
            s[h, TOK_PER_PART:] = v.imag
    return s


# the ladder's radix 2^3: two rungs of seven rotations, each rung one ModUp shared by its seven key dots (measured on
# MI355X: 0.95 ms per scoring against 1.6 ms for the six-rung log ladder and 1.9 ms for one rung of 63)
RADIX_BITS = 3


def ladder_steps(radix_bits=RADIX_BITS):
    """The rotation steps the ladder over a 64-slot block takes: 1, 2, 4, ..., 32 rung by rung; with radix_bits r,
    rungs of 2^r - 1 summed rotations by j g (j < 2^r, g = 1, 2^r, 4^r, ...)."""
    if radix_bits <= 1:
        return [1 << k for k in range(6)]
    out, g = [], 1
    while g < BLOCK:
        n = min(radix_bits, (BLOCK // g).bit_length() - 1)
        out += [j * g for j in range(1, 1 << n)]
        g <<= n
    return out


def score(ctx, keys, ct, pt, top, out, tmp, stream, radix_bits=RADIX_BITS):
    """One ciphertext's scores: out = rotate_and_sum(rescale(ct pt)) over the head blocks at limb top - 2; keys holds
    the rotations of ladder_steps(radix_bits). ct is left untouched; out and tmp are single ciphertexts (tmp: the
    ladder's scratch)."""
    ctx.mul_plain(ct, pt, top, out, stream)
    ctx.rescale(out, top, 2, out, stream)
    ctx.rotate_and_sum(keys, out, top - 2, 1, BLOCK, out, tmp, stream, radix_bits=radix_bits)


def score_batch(ctx, keys, cts, pts, top, outs, tmp, stream, radix_bits=RADIX_BITS):
    """Every ciphertext's scores at once: cts, outs and tmp each K consecutive ciphertexts of one buffer (the ctx's
    k_max and k_rot at least K), pts the K plaintexts; the plaintext products (each ciphertext by its own plaintext),
    the two-prime rescale and the ladder as K-ciphertext launches (pcx_mul_plain_k, pcx_rescale_k,
    pcx_rotate_and_sum_k). The words of score() on each ciphertext."""
    K = len(pts)
    ctx.mul_plain_k(cts, pts, top, outs, stream)
    ctx.rescale(outs, top, 2, outs, stream, K=K)
    ctx.rotate_and_sum(keys, outs, top - 2, 1, BLOCK, outs, tmp, stream, radix_bits=radix_bits, K=K)


def score_streams(lanes, cts, pts, top, outs, main, radix_bits=RADIX_BITS):
    """The scorings of independent ciphertexts side by side: lane i = (context, keys, stream, tmp) takes ciphertexts
    i, i + len(lanes), ...; each lane has its own context (its own workspace), so the lanes' small kernels overlap on
    the chip. Ordered after the work already on `main`, and `main` waits for every lane."""
    from .engine import Event

    start = Event()
    start.record(main)
    ends = []
    for i, (ctx, keys, st, tmp) in enumerate(lanes):
        st.wait(start)
        for c in range(i, len(cts), len(lanes)):
            score(ctx, keys, cts[c], pts[c], top, outs[c], tmp, st, radix_bits)
        e = Event()
        e.record(st)
        ends.append(e)
    for e in ends:
        main.wait(e)


class ClearBlock:
    """One attention block's clear side for a program that scores against encrypted keys: it makes the queries and keys of a
    public prompt and of the tokens after it (norms, rotation, the cache), and the attention in the clear that decrypted
    scores are held against. `rows` are the block's projected rows, an Array (or another library's device tensor) [tokens]
    [heads + 2 kv_heads][dim]: queries, then keys, then values. One sequence of up to `capacity` tokens; nothing is
    synchronised or allocated after the constructor."""

    def __init__(self, ops, heads, kv_heads, dim, capacity, dtype="bf16", table=None, layout="half", q_weight=None,
                 k_weight=None, eps=1e-6):
        from .clear import Array, block_checked

        block_checked(heads, kv_heads, dim, capacity, dtype, table, layout, q_weight, k_weight)
        self.ops, self.heads, self.kv_heads, self.dim, self.capacity = ops, heads, kv_heads, dim, capacity
        self.table, self.layout, self.q_weight, self.k_weight, self.eps = table, layout, q_weight, k_weight, eps
        self.k, self.v = (Array((capacity, kv_heads, dim), dtype) for _ in range(2))
        self.q, self.out = (Array((capacity, heads, dim), dtype) for _ in range(2))
        self.lse = Array((capacity, heads), "f32")
        places = np.arange(capacity, dtype=np.int64)
        # every length the cache takes: a step points at its own, so that no call uploads anything
        self._places, self._slots = Array.of(places, "i32"), Array.of(places, "i64")
        self._runs = Array.of(np.stack([np.zeros(capacity + 1), np.arange(capacity + 1)], 1), "i32")
        self._first = Array.of(np.zeros(1), "i64")
        self.length = 0

    def _rows(self, x, first, count):
        from .clear import Array, SIZES

        step = x._strides[0] * SIZES[x.dtype]
        return Array((count,) + x.shape[1:], x.dtype, x.buf, x.offset + first * step // 4, x._strides)

    def append(self, rows, causal=True):
        """The next tokens' rows into the cache, and their attention over all of it: (q, out, lse) of these tokens, views of
        the block's buffers. A whole prompt, a chunk of one, or one token."""
        from .clear import Array

        n, at = rows.shape[0], self.length
        if n < 1 or at + n > self.capacity:
            raise ValueError(f"{n} tokens after {at}: the block holds {self.capacity}")
        H, KV = self.heads, self.kv_heads
        if rows.shape[1] != H + 2 * KV or rows.shape[2] != self.dim:
            raise ValueError("rows: [tokens][heads + 2 kv_heads][dim]")
        part = rows.heads if isinstance(rows, Array) else lambda a, c: rows[:, a:a + c]
        q, out = self._rows(self.q, at, n), self._rows(self.out, at, n)
        lse = Array((n, H), "f32", self.lse.buf, at * H)
        self.ops.qk_norm_rotary(part(0, H), part(H, KV), self.q_weight, self.k_weight,
                                None if self.table is None else Array((n,), "i32", self._places.buf, at), self.table, q,
                                self.k, eps=self.eps, layout=self.layout, v=part(H + KV, KV), v_out=self.v,
                                slots=Array((n,), "i64", self._slots.buf, 2 * at))
        runs = self._runs.buf  # (0, n) for every n: a run's start and end, or its second alone as a length
        self.ops.attention(q, self.k, self.v, Array((2,), "i32", runs, 2 * n), self._first,
                           Array((1,), "i32", runs, 2 * (at + n) + 1), out, lse, causal=causal, max_q=n, max_k=at + n)
        self.length = at + n  # only now: tokens that failed are appended again at the same places
        return q, out, lse

    def keys(self):
        """The cached keys on the host, float32 [length][kv_heads dim]: what key_slots packs for encryption."""
        return self.k.numpy(self.ops.stream)[:self.length].reshape(self.length, -1)


class PagedBlock:
    """One attention block's clear side for several sequences that share a pool of pages, and for sequences longer than an encrypted
    scoring holds: each key's attention weight is gathered as queries see it, and `evict` cuts a sequence to its `keep` keys of
    largest weight (per key head), its last `recent` places and its first `first` among them. A key's place is its token's number
    in the sequence, which it is rotated by and keeps.

    `rows` are the block's projected rows of several sequences one after the other, an Array (or another library's device tensor)
    [tokens][heads + 2 kv_heads][dim]: queries, then keys, then values. A call uploads where its tokens go, a plan of seqs x pages
    words whatever it uses of them, and waits for that (so for the stream's work before it); nothing is allocated after the
    constructor. tokens: the most of one call."""

    def __init__(self, ops, heads, kv_heads, dim, seqs, pages, page_rows=16, keep=TOKENS, recent=32, first=4, tokens=TOKENS,
                 dtype="bf16", table=None, layout="half", q_weight=None, k_weight=None, eps=1e-6, decay=1.0):
        from .clear import Array, block_checked
        from .engine import DevBuf

        block_checked(heads, kv_heads, dim, 1, dtype, table, layout, q_weight, k_weight)
        if min(seqs, pages, tokens, keep) < 1 or min(recent, first) < 0 or first + recent > keep or not decay >= 0:
            raise ValueError("sequences, pages, tokens and keep: one or more; recent and first at most keep together; decay 0 or more")
        if page_rows < 16 or page_rows & (page_rows - 1):
            raise ValueError(f"page_rows {page_rows}: a power of two, 16 or more")
        if decay > 3.4e38 or max(seqs, kv_heads) > 65535 or kv_heads * dim > 1 << 22 or page_rows * kv_heads * dim >= 1 << 31:
            raise ValueError("decay: finite in 32 bits; up to 65535 sequences and key heads, 2^22 values a row of keys, below 2^31 a page")
        self.ops, self.heads, self.kv_heads, self.dim, self.page_rows = ops, heads, kv_heads, dim, page_rows
        self.keep, self.recent, self.first, self.decay, self.tokens = keep, recent, first, decay, tokens
        self.table, self.layout, self.q_weight, self.k_weight, self.eps = table, layout, q_weight, k_weight, eps
        rows = pages * page_rows
        self.k, self.v = (Array((rows, kv_heads, dim), dtype) for _ in range(2))
        self.q, self.out = (Array((tokens, heads, dim), dtype) for _ in range(2))
        self.lse = Array((tokens, heads), "f32")
        # a head's rows one after the other, as both of their operators read them
        self.weights, self.places = (Array((rows, kv_heads), kind, strides=(1, rows)) for kind in ("f32", "i32"))
        self.moves = Array((seqs, kv_heads, keep, 2), "i32")
        self.count = Array((seqs, kv_heads), "i32")
        self._free = list(range(pages))
        self._pages = [[] for _ in range(seqs)]
        self.lengths, self.next_places = [0] * seqs, [0] * seqs
        # what a call uploads, in one buffer: [slots i64][positions][q_start][k_len][next_place][tables]
        self._words = [2 * tokens, tokens, seqs + 1, seqs, seqs, seqs * pages]
        self._at = [sum(self._words[:i]) for i in range(len(self._words) + 1)]
        self._host = np.zeros(self._at[-1], np.int32)
        self._plan = DevBuf(self._at[-1])

    def _put(self, i, values, kind=np.int32):
        values = np.ascontiguousarray(values, kind).reshape(-1).view(np.int32)
        self._host[self._at[i]:self._at[i] + values.size] = values

    def _array(self, i, shape, kind="i32", strides=None):
        from .clear import Array

        return Array(shape, kind, self._plan, self._at[i], strides)

    def _upload(self, lengths, next_places, longest):
        """the sequences' lengths, places and pages as the next calls find them"""
        n, width = len(lengths), -(-longest // self.page_rows)
        table = np.full((n, width), -1, np.int32)
        for b, p in enumerate(self._pages):
            table[b, :len(p[:width])] = p[:width]
        self._put(3, lengths)
        self._put(4, next_places)
        self._put(5, table)
        self._plan.upload(self._host.view(np.uint32), self.ops.stream)
        return dict(pages=self._array(5, (n, width)), page_rows=self.page_rows)

    def append(self, rows, counts, causal=True):
        """The next counts[b] tokens of each sequence b (0: none) into its cache, and their attention over all of it: (q, out, lse) of
        these tokens, views of the block's buffers until the next call. Their weights are gathered by the keys that they see."""
        from .clear import Array

        counts = [int(c) for c in counts]
        T, H, KV, P = rows.shape[0], self.heads, self.kv_heads, self.page_rows
        if len(counts) != len(self.lengths) or min(counts) < 0 or sum(counts) != T or not 1 <= T <= self.tokens:
            raise ValueError(f"{T} rows, {counts} tokens: 1 to {self.tokens} in all, a number for each of {len(self.lengths)} sequences")
        if rows.shape[1] != H + 2 * KV or rows.shape[2] != self.dim:
            raise ValueError("rows: [tokens][heads + 2 kv_heads][dim]")
        if self.table is not None and any(c and at + c > self.table.shape[0] for at, c in zip(self.next_places, counts)):
            raise ValueError(f"the rotation's table has {self.table.shape[0]} places")
        lengths = [n + c for n, c in zip(self.lengths, counts)]
        need = [max(0, -(-n // P) - len(p)) for n, p in zip(lengths, self._pages)]
        if sum(need) > len(self._free):
            raise ValueError(f"{sum(need)} more pages wanted, {len(self._free)} are free: evict, or a larger pool")
        for p, n in zip(self._pages, need):
            p += [self._free.pop() for _ in range(n)]
        at = [np.arange(n, m) for n, m in zip(self.lengths, lengths)]
        self._put(0, np.concatenate([self._rows(b, j) for b, j in enumerate(at)]), np.int64)
        self._put(1, np.concatenate([np.arange(n, n + c) for n, c in zip(self.next_places, counts)]))
        self._put(2, np.concatenate([[0], np.cumsum(counts)]))
        next_places = [n + c for n, c in zip(self.next_places, counts)]
        seqs, longest = len(counts), max(n for n, c in zip(lengths, counts) if c)
        # sequences without new tokens are of length 0 to this call: their weights stay
        where = self._upload([n if c else 0 for n, c in zip(lengths, counts)], next_places, longest)
        q, out, lse = (Array((T,) + x.shape[1:], x.dtype, x.buf, 0, x.stride()) for x in (self.q, self.out, self.lse))
        part = rows.heads if isinstance(rows, Array) else lambda a, c: rows[:, a:a + c]
        q_start, k_len = self._array(2, (seqs + 1,)), self._array(3, (seqs,))
        expect = dict(max_q=max(counts), max_k=longest)
        self.ops.qk_norm_rotary(part(0, H), part(H, KV), self.q_weight, self.k_weight,
                                None if self.table is None else self._array(1, (T,)), self.table, q, self.k, eps=self.eps,
                                layout=self.layout, v=part(H + KV, KV), v_out=self.v, slots=self._array(0, (T,), "i64"))
        self.ops.attention_paged(q, self.k, self.v, q_start, where["pages"], P, k_len, out, lse, causal=causal, **expect)
        self.ops.key_weights(q, self.k, lse, q_start, k_len, self.weights, before=self.weights, decay=self.decay, places=self.places,
                             next_place=self._array(4, (seqs,)), causal=causal, **expect, **where)
        self.lengths, self.next_places = lengths, next_places  # only now: tokens that failed are appended again at the same places
        return q, out, lse

    def evict(self):
        """Cuts each sequence longer than `keep` to that many keys; their pages go back to the pool. Returns the (moves, count) of
        move_rows, for a copy of the cache elsewhere (on the host, say) that is to be kept alike: row moves[b][g][i][0] of
        sequence b and key head g went to row [i][1], i < count[b][g]; (None, None) where no sequence is longer. Nothing here
        moves the slots of an encrypted copy: that is made anew from keys()."""
        P, longest = self.page_rows, max(self.lengths)
        if longest <= self.keep:
            return None, None
        where = self._upload(self.lengths, self.next_places, longest)
        seqs = len(self.lengths)
        self.ops.evict(self.weights, self._array(3, (seqs,)), self.keep, self.moves, self.count, places=self.places,
                       next_place=self._array(4, (seqs,)), recent=self.recent, first=self.first, max_k=longest, **where)
        self.ops.move_rows(self.moves, self.count, (self.k, self.v, self.weights, self.places), **where)
        self.lengths = [min(n, self.keep) for n in self.lengths]
        for n, p in zip(self.lengths, self._pages):
            while len(p) > -(-n // P):
                self._free.append(p.pop())
        return self.moves, self.count

    def drop(self, seq):
        """Ends a sequence: its pages go back to the pool, its number is free for another."""
        self._free += self._pages[seq]
        self._pages[seq], self.lengths[seq], self.next_places[seq] = [], 0, 0

    def _rows(self, seq, j):
        return np.array(self._pages[seq] or [0], np.int64)[j // self.page_rows] * self.page_rows + j % self.page_rows

    def rows_of(self, seq):
        """The pool's rows of a sequence's keys, in the order of its cache (of k, v, weights and places)."""
        return self._rows(seq, np.arange(self.lengths[seq]))

    def keys(self, seq):
        """A sequence's cached keys on the host, float32 [length][kv_heads dim]: what key_slots packs for encryption."""
        from .clear import Array, SIZES

        n, step = self.lengths[seq], self.page_rows * self.kv_heads * self.dim * SIZES[self.k.dtype] // 4
        pages = [Array((self.page_rows, self.kv_heads * self.dim), self.k.dtype, self.k.buf, p * step).numpy(self.ops.stream)
                 for p in self._pages[seq]]
        return np.concatenate(pages)[:n] if n else np.zeros((0, self.kv_heads * self.dim), np.float32)
