"""The operators of a cache in pages: attention of chunks and tokens over it, the attention weight that its keys gather, and the
eviction of the keys that gathered least.

An encrypted scoring holds a fixed number of keys. These operators keep the clear side's cache at such a size: sequences share a
pool of pages, each key's weight is summed over the queries that saw it, and rows that are kept close the gaps of those that are
not, as few moves as there are gaps.

`run` takes the plain form (elementary torch operations in 32 bits, rounded once) or, with `own`, the package's entry points
(`perseus_amd.Clear`). Lengths of a ragged case come from its own `mix`, so that a case's work is known without its inputs.
"""
import functools
import math
import random

import numpy as np
import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


# ---------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # one token over the 512 keys of the encrypted scoring (12 heads of 64): the smallest call, latency only
        dict(name="paged_token", op="attention_paged", type="bf16", heads=12, kv_heads=12, dim=64, seqs=1, new=1, past=511,
             mix=0, causal=True, page=16),
        # one token each of 48 sequences over caches of different lengths, small pages
        dict(name="paged_tokens", op="attention_paged", type="bf16", heads=32, kv_heads=8, dim=128, seqs=48, new=1,
             past=8000, mix=11, causal=True, page=16),
        # one token over a long cache
        dict(name="paged_token_long", op="attention_paged", type="f16", heads=64, kv_heads=8, dim=128, seqs=1, new=1,
             past=131071, mix=0, causal=True, page=64),
        # chunks of prompts of different lengths, each after what of its sequence is there already
        dict(name="paged_chunks", op="attention_paged", type="bf16", heads=32, kv_heads=8, dim=128, seqs=6, new=512,
             past=6000, mix=5, causal=True, page=16),
        # a chunk of a long prompt, large pages
        dict(name="paged_chunk_long", op="attention_paged", type="f16", heads=16, kv_heads=4, dim=128, seqs=1, new=2048,
             past=30000, mix=0, causal=True, page=128),
        # chunks that see every key (a retrieved block), a head width that fills no power of two, pages within a tile of keys
        dict(name="paged_chunk_full", op="attention_paged", type="f16", heads=20, kv_heads=4, dim=80, seqs=5, new=200,
             past=5000, mix=7, causal=False, page=32),
        # what one token adds to the weights of 512 keys
        dict(name="weights_token", op="key_weights", type="bf16", heads=12, kv_heads=12, dim=64, seqs=1, new=1, past=511,
             mix=0, causal=True, page=0),
        # one token each of 48 sequences
        dict(name="weights_tokens", op="key_weights", type="bf16", heads=32, kv_heads=8, dim=128, seqs=48, new=1, past=8000,
             mix=11, causal=True, page=16),
        # a whole prompt's weights, before its keys are cut to what the scoring holds
        dict(name="weights_prompt", op="key_weights", type="f16", heads=32, kv_heads=8, dim=128, seqs=1, new=8192, past=0,
             mix=0, causal=True, page=0),
        # 16 tokens past the 512 that the encrypted scoring holds
        dict(name="evict_scoring", op="evict", type="bf16", kv_heads=12, dim=64, seqs=1, past=528, mix=0, keep=512, recent=32,
             first=4, page=0),
        # 48 sequences that have grown by up to 64 tokens since their last eviction
        dict(name="evict_steps", op="evict", type="bf16", kv_heads=8, dim=128, seqs=48, past=4160, mix=9, keep=4096,
             recent=256, first=4, page=16),
        # a long prompt's keys, cut to a quarter
        dict(name="evict_prompt", op="evict", type="f16", kv_heads=8, dim=128, seqs=1, past=65536, mix=0, keep=16384,
             recent=1024, first=4, page=64),
    ]


def _spread(rng, lo, hi):
    """a whole number of lo..hi, even over its logarithm"""
    return round(math.exp(rng.uniform(math.log(lo), math.log(hi))))


def draw(rng):
    op = rng.choice(["attention_paged", "attention_paged", "key_weights", "evict"])
    kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    dim = rng.choice([32, 40, 64, 64, 72, 80, 96, 112, 128, 128, 128, 192, 256])
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if op != "attention_paged" and rng.random() < 0.4:
        page = 0
    mix = rng.randint(1, 1000) if rng.random() < 0.7 else 0
    case = dict(op=op, type=rng.choice(["bf16", "f16"]), kv_heads=kv, dim=dim, mix=mix, page=page)
    if op == "evict":
        seqs = _spread(rng, 1, 48)
        past = _spread(rng, 16, min(65536, (400 << 20) // (2 * dim * kv * seqs)))
        keep = max(2, round(past * rng.choice([0.25, 0.5, 0.9, 0.98])))
        return dict(case, seqs=seqs, past=past, keep=keep, recent=rng.randint(0, keep // 2), first=rng.randint(0, min(8, keep // 2)))
    case.update(heads=kv * group, causal=rng.random() < 0.75)
    kind = rng.choice(["token", "token", "chunk", "prompt"])
    if kind == "token":
        seqs = _spread(rng, 1, 64)
        past = _spread(rng, 1, min(131072, (800 << 20) // (4 * dim * kv * seqs)))
        return dict(case, seqs=seqs, new=1, past=past)
    cells = 1.0e9 * 128 / max(dim, 64)
    if kind == "chunk":
        seqs, past = rng.randint(1, 6), _spread(rng, 16, 30000)
        return dict(case, seqs=seqs, new=_spread(rng, 2, max(2, min(2048, int(cells / (seqs * past * kv * group))))), past=past)
    seqs = rng.randint(1, 12)
    return dict(case, seqs=seqs, new=min(8192, _spread(rng, 17, int(math.sqrt(cells / (seqs * kv * group))))), past=0)


@functools.lru_cache(maxsize=None)
def _lengths(seqs, new, past, mix):
    """(new tokens, cached tokens) of each sequence; mix 0: all the longest"""
    rng = random.Random(mix)
    if not mix:
        return ((new, past),) * seqs
    got = [(rng.randint(1, new) if new else 0, rng.randint(0, past)) for _ in range(seqs)]
    got[rng.randrange(seqs)] = (new, past)
    return tuple(got)


def lengths(case):
    if case["op"] == "evict" and case["mix"]:  # sequences that were cut to `keep` before and have grown since
        rng = random.Random(case["mix"])
        low = min(case["keep"], case["past"])
        got = [(0, rng.randint(low, case["past"])) for _ in range(case["seqs"])]
        got[rng.randrange(case["seqs"])] = (0, case["past"])
        return tuple(got)
    return _lengths(case["seqs"], case.get("new", 0), case["past"], case["mix"])


def pairs(case):
    """the (query, key) pairs that a head computes"""
    return sum(n * p + (n * (n + 1) // 2 if case["causal"] else n * n) for n, p in lengths(case))


def work(case):
    n, m = sum(a for a, _ in lengths(case)), sum(a + b for a, b in lengths(case))
    kv, dim = case["kv_heads"], case["dim"]
    if case["op"] == "evict":
        # a move for each evicted row among the first `keep`: as many as there are on average, weights being in no order
        moved = 0.0
        for _, past in lengths(case):
            loose = past - min(past, case["recent"] + case["first"])
            if past > case["keep"] and loose:
                moved += (past - case["keep"]) * min(1.0, (case["keep"] - case["first"]) / loose)
        return {"bytes": 8 * m * kv + moved * kv * (8 + 2 * (2 * 2 * dim + 4 + 4)), "flops": 0}
    q, k = 2 * dim * n * case["heads"], 2 * dim * m * kv
    if case["op"] == "key_weights":  # queries, keys, log-sum-exps, the weights read and written
        return {"bytes": q + k + 4 * n * case["heads"] + 8 * m * kv, "flops": 2 * dim * case["heads"] * pairs(case)}
    return {"bytes": 2 * (q + k) + 4 * n * case["heads"], "flops": 4 * dim * case["heads"] * pairs(case)}


# ---------------------------------------------------------------------------------------------------- inputs


def _normal(gen, kind, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(TYPES[kind])


def _cache(case, gen, keys):
    """where the sequences' rows lie: state's k_start (one run each) or pages (shuffled over a pool), and the pool's rows"""
    page = case["page"]
    if not page:
        starts = [sum(keys[:b]) for b in range(len(keys))]
        return dict(k_start=torch.tensor(starts, device="cuda", dtype=torch.int64)), max(1, sum(keys))
    counts = [-(-n // page) for n in keys]
    pool = sum(counts) + 3
    order = torch.randperm(pool, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(keys), max(1, max(counts))), -1, device="cuda", dtype=torch.int32)
    at = 0
    for b, n in enumerate(counts):
        table[b, :n] = order[at:at + n]
        at += n
    return dict(pages=table, page=page), pool * page


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind, kv, dim, spans = case["type"], case["kv_heads"], case["dim"], lengths(case)
    new, keys = [a for a, _ in spans], [a + b for a, b in spans]
    state, rows = _cache(case, gen, keys)
    state.update(case=case, k=_normal(gen, kind, rows, kv, dim), max_k=max(keys),
                 k_len=torch.tensor(keys, device="cuda", dtype=torch.int32))
    if case["op"] == "evict":
        return _prepare_evict(state, gen, rows)
    state.update(q=_normal(gen, kind, sum(new), case["heads"], dim) * 1.5, max_q=max(new), scale=1 / math.sqrt(dim),
                 q_start=torch.tensor([sum(new[:b]) for b in range(len(new) + 1)], device="cuda", dtype=torch.int32))
    if case["op"] == "attention_paged":
        state["v"] = _normal(gen, kind, rows, kv, dim)
        state.update(out=torch.empty_like(state["q"]), lse=torch.empty(state["q"].shape[:2], device="cuda"))
        return state
    # the log-sum-exps that the attention of the same queries left, and the weights of the steps before, a row for each head
    state["lse"] = torch.empty(state["q"].shape[:2], device="cuda")
    at = _rows(state)
    for b, (n, past) in enumerate(spans):
        first = sum(new[:b])
        k = state["k"][at[b, :n + past]].float()
        for h in range(case["heads"]):
            z = (state["q"][first:first + n, h].float() * state["scale"]) @ k[:, h // (case["heads"] // kv)].T
            if case["causal"]:
                z.masked_fill_(torch.ones_like(z, dtype=torch.bool).triu_(past + 1), -math.inf)
            state["lse"][first:first + n, h] = z.logsumexp(-1)
    state["before"] = torch.rand(kv, rows, generator=gen, device="cuda").t()
    state["weights"] = torch.zeros(kv, rows, device="cuda").t()
    return state


def _prepare_evict(state, gen, rows):
    case = state["case"]
    kv, dim = case["kv_heads"], case["dim"]
    # gathered weights spread over orders of magnitude; what far keys got may have vanished, so that zeros tie
    w = torch.exp(2.5 * torch.randn(kv, rows, generator=gen, device="cuda") - 3)
    w *= torch.rand(kv, rows, generator=gen, device="cuda") > 0.02
    # after earlier evictions rows are in no order of their tokens' places: here any order of them, another for each head
    places = torch.empty(kv, rows, device="cuda", dtype=torch.int32)
    at = _rows(state)
    for b, (_, n) in enumerate(lengths(case)):
        places[:, at[b, :n]] = torch.rand(kv, n, generator=gen, device="cuda").argsort(-1).to(torch.int32)
    most = max(1, min(case["keep"], max(0, state["max_k"] - case["keep"])))
    # the rows' weights and places move too, in copies of their own here, so that a pass can be run again
    state.update(v=_normal(gen, case["type"], rows, kv, dim), weights=w.t(), places=places.t(), moved_weights=w.clone().t(),
                 moved_places=places.clone().t(), next_place=state["k_len"].clone(),
                 moves=torch.full((case["seqs"], kv, most, 2), -1, device="cuda", dtype=torch.int32),
                 count=torch.zeros(case["seqs"], kv, device="cuda", dtype=torch.int32))
    return state


# ---------------------------------------------------------------------------------------------------- the package's operators


@functools.lru_cache(maxsize=None)
def _clear(stream):
    """what a program keeps: the operators on its stream, with their workspace"""
    import perseus_amd as pa

    return pa.Clear(pa.Stream.of(stream))


def _run_own(s):
    case = s["case"]
    ops = _clear(torch.cuda.current_stream().cuda_stream)
    where = dict(pages=s["pages"], page_rows=s["page"]) if "pages" in s else dict(k_start=s["k_start"])
    if case["op"] == "attention_paged":
        ops.attention_paged(s["q"], s["k"], s["v"], s["q_start"], s["pages"], s["page"], s["k_len"], s["out"], s["lse"],
                            scale=s["scale"], causal=case["causal"], max_q=s["max_q"], max_k=s["max_k"])
        return {"out": s["out"], "lse": s["lse"]}
    if case["op"] == "key_weights":
        ops.key_weights(s["q"], s["k"], s["lse"], s["q_start"], s["k_len"], s["weights"], before=s["before"], decay=0.97,
                        scale=s["scale"], causal=case["causal"], max_q=s["max_q"], max_k=s["max_k"], **where)
        return s["weights"]
    ops.evict(s["weights"], s["k_len"], case["keep"], s["moves"], s["count"], places=s["places"], next_place=s["next_place"],
              recent=case["recent"], first=case["first"], max_k=s["max_k"], **where)
    ops.move_rows(s["moves"], s["count"], (s["k"], s["v"], s["moved_weights"], s["moved_places"]), **where)
    return _evicted(s)


def _evicted(s):
    return {"moves": s["moves"], "count": s["count"], "k": s["k"], "v": s["v"], "weights": s["moved_weights"],
            "places": s["moved_places"]}


# ---------------------------------------------------------------------------------------------------- the plain forms


def _rows(s):
    """the pool's row of each sequence's key, [sequence][key up to the longest] (any row past a sequence's own)"""
    j = torch.arange(s["max_k"], device="cuda")
    if "k_start" in s:
        return (s["k_start"][:, None] + j).clamp_max(s["k"].shape[0] - 1)
    return s["pages"].long().clamp_min(0)[:, j // s["page"]] * s["page"] + j % s["page"]


def _scores(s):
    """scores [sequence][kv head][group][query][key], -infinity where a query does not see, every sequence padded to the
    longest; the queries' rows and whether there is one"""
    case = s["case"]
    group, kv, dim = case["heads"] // case["kv_heads"], case["kv_heads"], case["dim"]
    q_start, q_len = s["q_start"][:-1].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    k_len, n, m = s["k_len"].long(), s["max_q"], s["max_k"]
    i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    at = (q_start[:, None] + i).clamp_max(s["q"].shape[0] - 1)
    q = s["q"][at].float().view(-1, n, kv, group, dim).permute(0, 2, 3, 1, 4)
    k = s["k"][_rows(s)].float().permute(0, 2, 3, 1).contiguous()
    seen = (j < k_len[:, None])[:, None, :]
    if case["causal"]:
        seen = seen & (j <= (k_len - q_len)[:, None, None] + i[:, None])
    live = i < q_len[:, None]
    z = torch.matmul((q * s["scale"]).reshape(-1, kv, group * n, dim), k).view(-1, kv, group, n, m)
    return z.masked_fill_(~(seen & live[:, :, None])[:, None, None], -math.inf), at, live


def _attend(s):
    case = s["case"]
    kv, dim = case["kv_heads"], case["dim"]
    p, _, live = _scores(s)
    _, _, group, n, m = p.shape
    v = s["v"][_rows(s)].float().permute(0, 2, 1, 3).contiguous()
    top = p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(-1, kv, group * n, m), v).view(-1, kv, group, n, dim) / total.clamp_min(1e-30)
    lse = (top + total.log()).squeeze(-1)
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, n, case["heads"], dim)[live]
    return {"out": o.to(TYPES[case["type"]]), "lse": lse.permute(0, 3, 1, 2).reshape(-1, n, case["heads"])[live]}


def _weigh(s):
    p, at, _ = _scores(s)
    lse = s["lse"][at].view(*at.shape, s["case"]["kv_heads"], -1).permute(0, 2, 3, 1)[..., None]
    p.sub_(lse).exp_()
    got = p.sum(-2).sum(2).permute(0, 2, 1)  # [sequence][key][kv head]
    there = torch.arange(s["max_k"], device="cuda") < s["k_len"][:, None]
    rows = _rows(s)[there]
    out = torch.zeros(s["k"].shape[1], s["k"].shape[0], device="cuda").t()
    out[rows] = 0.97 * s["before"][rows] + got[there]
    return out


def _evict(s):
    case = s["case"]
    rows, k_len, keep = _rows(s), s["k_len"].long()[:, None, None], case["keep"]
    j = torch.arange(s["max_k"], device="cuda")
    w = s["weights"][rows].permute(0, 2, 1)  # [sequence][kv head][key]
    place = s["places"][rows].permute(0, 2, 1)
    held = (place >= s["next_place"][:, None, None] - case["recent"]) | (place < case["first"])
    w = torch.where(held, math.inf, w).masked_fill(j >= k_len, -math.inf)
    rank = torch.empty_like(w, dtype=torch.int64)
    rank.scatter_(-1, w.argsort(dim=-1, descending=True, stable=True), j.expand_as(w))
    kept = rank < k_len.clamp_max(keep)
    hole, mover = ~kept & (j < keep) & (j < k_len), kept & (j >= keep)
    moves, count = torch.full_like(s["moves"], -1), mover.sum(-1)
    for side, which in ((0, mover), (1, hole)):
        b, g, at = which.nonzero(as_tuple=True)
        moves[b, g, (which.cumsum(-1) - 1)[which], side] = at.to(torch.int32)
    b, g, i = (torch.arange(moves.shape[2], device="cuda") < count[..., None]).nonzero(as_tuple=True)
    source, to = (rows[b, moves[b, g, i, x].long()] for x in (0, 1))
    for x in (s["k"], s["v"], s["moved_weights"], s["moved_places"]):
        x[to, g] = x[source, g]
    s["moves"].copy_(moves)
    s["count"].copy_(count)
    return _evicted(s)


def run(state):
    if own:
        return _run_own(state)
    return {"attention_paged": _attend, "key_weights": _weigh, "evict": _evict}[state["case"]["op"]](state)


# ---------------------------------------------------------------------------------------------------- in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    spans, page = lengths(case), case["page"]
    table = s["pages"].tolist() if page else s["k_start"].tolist()

    def run_of(b, n):  # the rows of sequence b's keys, in their order
        if not page:
            return torch.arange(table[b], table[b] + n, device="cuda")
        return torch.tensor([table[b][j // page] * page + j % page for j in range(n)], device="cuda", dtype=torch.int64)

    if case["op"] == "evict":
        return _exact_evict(s, run_of)
    group = case["heads"] // case["kv_heads"]
    out, lse = torch.zeros_like(s["q"], dtype=torch.float64), torch.full(s["q"].shape[:2], -math.inf, device="cuda", dtype=torch.float64)
    weights = torch.zeros(s["k"].shape[:2], device="cuda", dtype=torch.float64)
    first = 0
    for b, (n, past) in enumerate(spans):
        rows = run_of(b, n + past)
        if case["op"] == "key_weights":
            weights[rows] = 0.97 * s["before"][rows].double()
        for h in range(case["heads"]):
            g = h // group
            z = s["q"][first:first + n, h].double() @ s["k"][rows, g].double().T * s["scale"]
            if case["causal"]:
                z += torch.full_like(z, -math.inf).triu(past + 1)
            if case["op"] == "key_weights":
                weights[rows, g] += (z - s["lse"][first:first + n, h, None].double()).exp().sum(0)
            else:
                lse[first:first + n, h] = z.logsumexp(-1)
                out[first:first + n, h] = torch.softmax(z, -1) @ s["v"][rows, g].double()
        first += n
    return weights if case["op"] == "key_weights" else {"out": out, "lse": lse}


def _exact_evict(s, run_of):
    case = s["case"]
    got = {n: s[m].clone() for n, m in (("k", "k"), ("v", "v"), ("weights", "moved_weights"), ("places", "moved_places"))}
    moves, count = torch.full_like(s["moves"], -1), torch.zeros_like(s["count"])
    for b, (_, n) in enumerate(lengths(case)):
        rows = run_of(b, n)
        for g in range(case["kv_heads"] if n > case["keep"] else 0):
            place, w = (s[x][rows, g].cpu().numpy() for x in ("places", "weights"))
            loose = (place < n - case["recent"]) & (place >= case["first"])
            kept = np.sort(np.lexsort((np.arange(n), -w.astype(np.float64), loose))[:case["keep"]])
            at = np.stack([kept[kept >= case["keep"]], np.setdiff1d(np.arange(case["keep"]), kept)], 1)
            count[b, g] = len(at)
            if len(at):
                at = torch.from_numpy(at).cuda()
                moves[b, g, :len(at)] = at.to(torch.int32)
                for x in got.values():
                    x[rows[at[:, 1]], g] = x[rows[at[:, 0]], g]
    return {"moves": moves, "count": count, "k": got["k"].double(), "v": got["v"].double(), "weights": got["weights"].double(),
            "places": got["places"]}
