"""The operators of the clear side of an encrypted transformer block: rotary positions, the norms of queries and keys with the
rotation in the same pass, and attention (a prompt's, packed sequences', a chunk's or one token's over a cache of keys).

The engine scores plaintext queries against encrypted keys. These operators make what it starts from (queries and keys, normed
and rotated) and what its answers are held against (the attention in the clear, with its log-sum-exp).

`run` takes the plain form (elementary torch operations in 32 bits, rounded once) or, with `own`, the package's entry points
(`perseus_amd.clear`). Lengths of a ragged case come from its own `mix`, so that a case's work is known without its inputs.
"""
import functools
import math
import random

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}


# ---------------------------------------------------------------------------------------------------- the cases


def listed():
    return [
        # one token's queries and keys (12 + 12 heads of 64): the smallest call, latency only
        dict(name="rotary_token", op="rotary", type="bf16", tokens=1, heads=24, dim=64, rot=64, layout="half",
             inverse=False, places=512, scaled=False),
        # a prompt's queries and keys, a quarter of each head rotated in neighbouring pairs, the table scaled for 128k places
        dict(name="rotary_prompt", op="rotary", type="f16", tokens=8191, heads=40, dim=128, rot=32,
             layout="interleaved", inverse=False, places=131072, scaled=True),
        # cached keys taken back to place 0 in 32 bits, before they are rotated to other places
        dict(name="rotary_undo", op="rotary", type="f32", tokens=16384, heads=8, dim=128, rot=128, layout="half",
             inverse=True, places=32768, scaled=False),
        # a step of 48 sequences: norms and rotation of one token each
        dict(name="qk_norm_tokens", op="qk_norm_rotary", type="bf16", tokens=48, heads=32, kv_heads=8, dim=128, rot=128,
             layout="half", places=32768, scaled=False),
        # a long prompt's queries and keys
        dict(name="qk_norm_prompt", op="qk_norm_rotary", type="bf16", tokens=16384, heads=32, kv_heads=8, dim=128,
             rot=128, layout="half", places=32768, scaled=False),
        # the attention-scoring shape (12 heads of 64, 512 tokens) as a prompt
        dict(name="prompt_512", op="attention", type="bf16", heads=12, kv_heads=12, dim=64, seqs=1, new=512, past=0,
             mix=0, causal=True),
        # nine packed prompts of different lengths, grouped heads
        dict(name="prompt_packed", op="attention", type="bf16", heads=32, kv_heads=8, dim=128, seqs=9, new=2048, past=0,
             mix=3, causal=True),
        # one long prompt
        dict(name="prompt_long", op="attention", type="f16", heads=16, kv_heads=4, dim=128, seqs=1, new=16384, past=0,
             mix=0, causal=True),
        # chunks of up to 200 tokens appended to caches, a head width that fills no power of two, every key seen (no causal
        # order: an encoder's or a retrieved block)
        dict(name="chunk_full", op="attention", type="f16", heads=20, kv_heads=4, dim=80, seqs=5, new=200, past=5000, mix=7,
             causal=False),
        # one token over 512 cached keys: the plain answer beside the encrypted scoring's
        dict(name="token_512", op="attention", type="bf16", heads=12, kv_heads=12, dim=64, seqs=1, new=1, past=511,
             mix=0, causal=True),
        # one token each of 48 sequences over caches of different lengths
        dict(name="token_batch", op="attention", type="bf16", heads=32, kv_heads=8, dim=128, seqs=48, new=1, past=8000,
             mix=11, causal=True),
        # one token over a long cache
        dict(name="token_long", op="attention", type="f16", heads=64, kv_heads=8, dim=128, seqs=1, new=1, past=131071,
             mix=0, causal=True),
    ]


def _spread(rng, lo, hi):
    """a whole number of lo..hi, even over its logarithm"""
    n = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
    return n + 1 if n == 3072 else n


def draw(rng):
    op = rng.choice(["rotary", "qk_norm_rotary", "attention", "attention", "attention"])
    kv = rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    group = rng.choice([1, 1, 2, 3, 4, 5, 7, 8])
    dim = rng.choice([32, 40, 64, 64, 72, 80, 96, 112, 128, 128, 128, 192, 256])
    if op != "attention":
        rot = dim if rng.random() < 0.6 else rng.choice([r for r in (8, 16, 24, 32, 64, 96, 128) if r <= dim])
        case = dict(op=op, type=rng.choice(["bf16", "f16", "f32"]), dim=dim, rot=rot,
                    layout=rng.choice(["half", "interleaved"]), places=rng.choice([2048, 32768, 131072]),
                    scaled=rng.random() < 0.4)
        tokens = _spread(rng, 1, max(2, min(20000, (100 << 20) // (dim * kv * (group + 1) * BYTES[case["type"]]))))
        if op == "rotary":
            return dict(case, tokens=tokens, heads=kv * (group + 1), inverse=rng.random() < 0.3)
        return dict(case, tokens=tokens, heads=kv * group, kv_heads=kv)
    case = dict(op=op, type=rng.choice(["bf16", "f16"]), heads=kv * group, kv_heads=kv, dim=dim,
                causal=rng.random() < 0.75)
    kind = rng.choice(["token", "token", "chunk", "prompt"])
    mix = rng.randint(1, 1000) if rng.random() < 0.7 else 0
    if kind == "token":
        seqs = _spread(rng, 1, 64)
        past = _spread(rng, 1, min(131072, (800 << 20) // (4 * dim * kv * seqs)))
        return dict(case, seqs=seqs, new=1, past=past, mix=mix)
    if kind == "chunk":
        seqs, past = rng.randint(1, 6), _spread(rng, 16, 8000)
        new = _spread(rng, 2, max(2, min(300, int(2e9 / (seqs * past * kv * group * dim / 128)))))
        return dict(case, seqs=seqs, new=new, past=past, mix=mix)
    seqs = rng.randint(1, 12)
    cells = (4.2e9 if case["causal"] else 2.1e9) * 128 / max(dim, 64)
    new = _spread(rng, 17, int(math.sqrt(cells / (seqs * kv * group))))
    return dict(case, seqs=seqs, new=min(new, 16384), past=0, mix=mix)


@functools.lru_cache(maxsize=None)
def _lengths(seqs, new, past, mix):
    """(new tokens, cached tokens) of each sequence; mix 0: all the longest"""
    rng = random.Random(mix)
    if not mix:
        return ((new, past),) * seqs
    got = [(rng.randint(1, new), rng.randint(0, past)) for _ in range(seqs)]
    got[rng.randrange(seqs)] = (new, past)
    return tuple(got)


def lengths(case):
    return _lengths(case["seqs"], case["new"], case["past"], case["mix"])


def pairs(case):
    """the (query, key) pairs that a head computes"""
    return sum(n * p + (n * (n + 1) // 2 if case["causal"] else n * n) for n, p in lengths(case))


def work(case):
    es = BYTES[case["type"]]
    if case["op"] == "attention":
        n, k = sum(a for a, _ in lengths(case)), sum(a + b for a, b in lengths(case))
        return {"bytes": 2 * es * case["dim"] * (n * case["heads"] + k * case["kv_heads"]) + 4 * n * case["heads"],
                "flops": 4 * case["dim"] * case["heads"] * pairs(case)}
    heads = case["heads"] + case.get("kv_heads", 0)
    values, turned = case["tokens"] * heads * case["dim"], case["tokens"] * heads * case["rot"]
    return {"bytes": 2 * es * values + 4 * case["tokens"] + 4 * case["rot"] * min(case["tokens"], case["places"]),
            "flops": 3 * turned + (4 * values if "kv_heads" in case else 0)}


# ---------------------------------------------------------------------------------------------------- inputs


def _rotation_table(places, rot, scaled):
    """cos and sin of every place and pair, f32 [places][rot / 2][2], from angles in 64 bits; scaled: pairs that turn less
    than once in 2048 places go eight times slower, those that turn more than four times keep their pace, a ramp between"""
    rate = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    if scaled:
        turns = 2048 * rate / (2 * math.pi)
        keep = ((turns - 1) / 3).clamp(0, 1)
        rate = rate * (keep + (1 - keep) / 8)
    angle = torch.arange(places, device="cuda", dtype=torch.float64)[:, None] * rate
    return torch.stack([angle.cos(), angle.sin()], -1).float()


def _normal(gen, kind, *shape):
    return torch.randn(*shape, generator=gen, device="cuda", dtype=torch.float32).to(TYPES[kind])


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = case["type"]
    state = dict(case=case)
    if case["op"] == "attention":
        spans = lengths(case)
        new, keys = [a for a, _ in spans], [a + b for a, b in spans]
        # caches of one size per sequence where there is a past; prompts lie packed
        room = [case["new"] + case["past"]] * len(spans) if case["past"] else keys
        q_start = [sum(new[:i]) for i in range(len(new) + 1)]
        k_start = [sum(room[:i]) for i in range(len(room))]
        state.update(
            q=_normal(gen, kind, q_start[-1], case["heads"], case["dim"]) * 1.5,
            k=_normal(gen, kind, sum(room), case["kv_heads"], case["dim"]),
            v=_normal(gen, kind, sum(room), case["kv_heads"], case["dim"]),
            q_start=torch.tensor(q_start, device="cuda", dtype=torch.int32),
            k_start=torch.tensor(k_start, device="cuda", dtype=torch.int64),
            k_len=torch.tensor(keys, device="cuda", dtype=torch.int32),
            max_q=max(new), max_k=max(keys), scale=1 / math.sqrt(case["dim"]))
        state.update(out=torch.empty_like(state["q"]), lse=torch.empty(state["q"].shape[:2], device="cuda"))
        return state
    tokens, dim = case["tokens"], case["dim"]
    state["table"] = _rotation_table(case["places"], case["rot"], case["scaled"])
    if tokens <= 64:  # a step of sequences that stand at different places
        at = torch.randint(0, case["places"], (tokens,), generator=gen, device="cuda")
    else:  # one run of a prompt
        at = torch.arange(tokens, device="cuda") + torch.randint(0, max(1, case["places"] - tokens), (1,), generator=gen,
                                                                  device="cuda")
    state["positions"] = (at % case["places"]).to(torch.int32)
    if case["op"] == "rotary":
        state["x"] = _normal(gen, kind, tokens, case["heads"], dim)
        state["out"] = torch.empty_like(state["x"])
        return state
    # queries and keys as a joint projection leaves them: columns of one row [queries | keys | values]
    heads, kv = case["heads"], case["kv_heads"]
    rows = _normal(gen, kind, tokens, heads + 2 * kv, dim)
    rows[:, :heads] *= 3
    state.update(q=rows[:, :heads], k=rows[:, heads:heads + kv], eps=1e-6,
                 q_weight=1 + 0.2 * torch.randn(dim, generator=gen, device="cuda"),
                 k_weight=1 + 0.2 * torch.randn(dim, generator=gen, device="cuda"),
                 q_out=torch.empty(tokens, heads, dim, device="cuda", dtype=TYPES[kind]),
                 k_out=torch.empty(tokens, kv, dim, device="cuda", dtype=TYPES[kind]))
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
    if case["op"] == "rotary":
        ops.rotary(s["x"], s["positions"], s["table"], s["out"], layout=case["layout"], inverse=case["inverse"])
        return s["out"]
    if case["op"] == "qk_norm_rotary":
        ops.qk_norm_rotary(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["table"], s["q_out"],
                           s["k_out"], eps=s["eps"], layout=case["layout"])
        return {"q": s["q_out"], "k": s["k_out"]}
    ops.attention(s["q"], s["k"], s["v"], s["q_start"], s["k_start"], s["k_len"], s["out"], s["lse"], scale=s["scale"],
                  causal=case["causal"], max_q=s["max_q"], max_k=s["max_k"])
    return {"out": s["out"], "lse": s["lse"]}


# ---------------------------------------------------------------------------------------------------- the plain forms


def _turn(x, at, case, inverse=False):
    """x [T][H][D] in 32 bits, its first rot dims turned by at [T][rot / 2][2]"""
    rot = case["rot"]
    cos, sin = at[:, None, :, 0], at[:, None, :, 1]
    sin = -sin if inverse else sin
    head, rest = x[..., :rot], x[..., rot:]
    if case["layout"] == "half":
        a, b = head[..., :rot // 2], head[..., rot // 2:]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, rest], -1)
    a, b = head[..., 0::2], head[..., 1::2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), rest], -1)


def _norm(x, weight, eps):
    return x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps) * weight


def _attend(s):
    case = s["case"]
    group, kv, dim, kind = case["heads"] // case["kv_heads"], case["kv_heads"], case["dim"], TYPES[case["type"]]
    q_start, q_len = s["q_start"][:-1].long(), (s["q_start"][1:] - s["q_start"][:-1]).long()
    k_len, n, m = s["k_len"].long(), s["max_q"], s["max_k"]
    i, j = torch.arange(n, device="cuda"), torch.arange(m, device="cuda")
    # every sequence padded to the longest: [sequence][kv head][group][query][dim]
    q = s["q"][(q_start[:, None] + i).clamp_max(s["q"].shape[0] - 1)].float().view(-1, n, kv, group, dim).permute(0, 2, 3, 1, 4)
    rows = (s["k_start"][:, None] + j).clamp_max(s["k"].shape[0] - 1)
    k, v = s["k"][rows].float().permute(0, 2, 3, 1), s["v"][rows].float().permute(0, 2, 1, 3)
    seen = (j < k_len[:, None])[:, None, :]
    if case["causal"]:
        seen = seen & (j <= (k_len - q_len)[:, None, None] + i[:, None])
    p = torch.matmul((q * s["scale"]).reshape(q.shape[0], kv, group * n, dim), k.contiguous()).view(-1, kv, group, n, m)
    p.masked_fill_(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p.sub_(top).exp_()
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(p.shape[0], kv, group * n, m), v.contiguous()).view(-1, kv, group, n, dim) / total.clamp_min(1e-30)
    lse = (top + total.log()).squeeze(-1)
    live = i < q_len[:, None]
    o = o.permute(0, 3, 1, 2, 4).reshape(-1, n, case["heads"], dim)[live]
    return {"out": o.to(kind), "lse": lse.permute(0, 3, 1, 2).reshape(-1, n, case["heads"])[live]}


def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    if case["op"] == "attention":
        return _attend(state)
    kind, at = TYPES[case["type"]], state["table"][state["positions"].long()]
    if case["op"] == "rotary":
        return _turn(state["x"].float(), at, case, case["inverse"]).to(kind)
    return {"q": _turn(_norm(state["q"].float(), state["q_weight"], state["eps"]), at, case).to(kind),
            "k": _turn(_norm(state["k"].float(), state["k_weight"], state["eps"]), at, case).to(kind)}


# ---------------------------------------------------------------------------------------------------- in 64 bits


def _turned(x, s):
    """the rotation as a product of complex numbers"""
    case = s["case"]
    rot, x = case["rot"], x.double()
    z = torch.view_as_complex(s["table"].double()[s["positions"].long()].contiguous())[:, None]
    z = z.conj() if case.get("inverse") else z
    y = x.clone()
    if case["layout"] == "half":
        w = torch.complex(x[..., :rot // 2], x[..., rot // 2:rot]) * z
        y[..., :rot // 2], y[..., rot // 2:rot] = w.real, w.imag
    else:
        w = torch.complex(x[..., 0:rot:2], x[..., 1:rot:2]) * z
        y[..., 0:rot:2], y[..., 1:rot:2] = w.real, w.imag
    return y


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rotary":
        return _turned(s["x"], s)
    if case["op"] == "qk_norm_rotary":
        def unit(x, w):
            x = x.double()
            return x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + s["eps"]).sqrt() * w.double()
        return {"q": _turned(unit(s["q"], s["q_weight"]), s), "k": _turned(unit(s["k"], s["k_weight"]), s)}
    out, lse = torch.zeros_like(s["out"], dtype=torch.float64), torch.full_like(s["lse"], -math.inf, dtype=torch.float64)
    group, room = case["heads"] // case["kv_heads"], s["k_start"].tolist()
    row = 0
    for (n, past), first in zip(lengths(case), room):
        for h in range(case["heads"]):
            q = s["q"][row:row + n, h].double()
            k, v = (s[x][first:first + n + past, h // group].double() for x in ("k", "v"))
            z = (q @ k.T) * s["scale"]
            if case["causal"]:
                z += torch.full_like(z, -math.inf).triu(past + 1)
            lse[row:row + n, h] = z.logsumexp(-1)
            out[row:row + n, h] = torch.softmax(z, -1) @ v
        row += n
    return {"out": out, "lse": lse}
