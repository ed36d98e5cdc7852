"""The operators of serving many answers to one prompt, as timed cases: appending to an INT8 key/value cache
and reading it back, the attention of a step and of a prompt over that cache, attention of a batch whose
sequences share a prefix, log probabilities.  ``run`` is one call; with ``own`` false the same in elementary
32-bit torch.  ``exact`` is the definition in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False

F32, F64 = torch.float32, torch.float64
THETA = 500000.0


def listed():
    return [
        # a step of a served batch writes one row per sequence; a prompt writes all of its rows
        dict(name="append_step", kind="append", tokens=64, sequences=64, heads=32, kv_heads=8, dim=128, rows=2048),
        dict(name="append_prompt", kind="append", tokens=2048, sequences=1, heads=32, kv_heads=8, dim=128, rows=4096),
        # chat, one user: one query against a 2048-token context
        dict(name="attend_1", kind="attend", batch=1, heads=32, kv_heads=8, dim=128, rows=2048),
        # a served batch, contexts of unequal length
        dict(name="attend_64", kind="attend", batch=64, heads=32, kv_heads=8, dim=128, rows=2048),
        # two users far into long documents
        dict(name="attend_long", kind="attend", batch=2, heads=32, kv_heads=8, dim=128, rows=65536),
        # a prompt from its first position on, and a short last portion of an odd length behind a long one
        dict(name="portion_2048", kind="portion", tokens=2048, first=0, heads=32, kv_heads=8, dim=128),
        dict(name="portion_tail", kind="portion", tokens=37, first=8155, heads=32, kv_heads=8, dim=128),
        # 64 answers to one long prompt, and eight to a shorter one, from a small cache
        dict(name="shared_64", kind="shared", batch=64, prefix=8192, rows=256, heads=32, kv_heads=8, dim=128,
             dtype="bfloat16"),
        dict(name="shared_8_int8", kind="shared", batch=8, prefix=4001, rows=128, heads=32, kv_heads=8, dim=128,
             dtype="int8"),
        # the probability of one token with alternatives, of a batch's tokens, of all tokens of a scored text
        dict(name="log_probs_1", kind="log_probs", tokens=1, vocab=32768, top=5),
        dict(name="log_probs_64", kind="log_probs", tokens=64, vocab=128256, top=20),
        dict(name="log_probs_2048", kind="log_probs", tokens=2048, vocab=32000, top=0),
    ]


def _log(rng, lo: int, hi: int) -> int:
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def _heads(rng) -> dict:
    kv = rng.choice([2, 4, 8])
    return dict(heads=kv * rng.choice([1, 2, 4, 4, 8]), kv_heads=kv, dim=rng.choice([64, 128, 128]))


def draw(rng):
    """A case of the same kinds, odd sizes among them."""
    kind = rng.choice(["append", "attend", "attend", "portion", "shared", "shared", "log_probs"])
    if kind == "append":
        if rng.random() < 0.5:
            tokens = _log(rng, 1, 96)
            return dict(kind=kind, tokens=tokens, sequences=tokens, rows=_log(rng, 16, 2048), **_heads(rng))
        tokens = _log(rng, 16, 2048)
        return dict(kind=kind, tokens=tokens, sequences=1, rows=tokens + rng.randint(0, 2000), **_heads(rng))
    if kind == "attend":
        batch = _log(rng, 1, 64)
        return dict(kind=kind, batch=batch, rows=_log(rng, 1, min(65536, 131072 // batch)), **_heads(rng))
    if kind == "portion":
        tokens = _log(rng, 1, 1536)
        return dict(kind=kind, tokens=tokens, first=rng.choice([0, _log(rng, 1, 8192 if tokens <= 256 else 512)]),
                    **_heads(rng))
    if kind == "shared":
        return dict(kind=kind, batch=_log(rng, 2, 64), prefix=_log(rng, 48, 8192), rows=_log(rng, 1, 256),
                    dtype=rng.choice(["bfloat16", "int8"]), **_heads(rng))
    vocab = _log(rng, 1000, 131072)
    return dict(kind=kind, tokens=_log(rng, 1, min(2048, 65000000 // vocab)), vocab=vocab,
                top=rng.choice([0, 1, 5, 20]))


# ---------------------------------------------------------------------- inputs
def _lengths(batch: int, rows: int) -> list:
    """Filled rows per sequence: from all of them down to half."""
    return [rows - b * rows // (2 * batch) for b in range(batch)]


def _rows(gen, *shape):
    """Rows of keys or values: N(0, 1) with a few channels that are larger, as keys have."""
    x = torch.randn(shape, device="cuda", generator=gen)
    x[..., ::16] *= 3.0
    return x


def _quantised(x):
    peak = x.abs().amax(-1, keepdim=True)
    scale = peak / 127.0
    return torch.round(x / scale).to(torch.int8), scale.squeeze(-1)


def _cache(gen, dtype: str, *shape) -> dict:
    """A filled cache [sequences, kv heads, rows, dim]."""
    k, v = _rows(gen, *shape), _rows(gen, *shape)
    if dtype != "int8":
        return dict(k=k.to(torch.bfloat16), v=v.to(torch.bfloat16), ks=None, vs=None)
    (k, ks), (v, vs) = _quantised(k), _quantised(v)
    return dict(k=k, v=v, ks=ks, vs=vs)


def _cos_sin(positions: int, dim: int):
    inv = THETA ** (-2.0 * torch.arange(dim // 2, device="cuda", dtype=F64) / dim)
    angle = torch.arange(positions, device="cuda", dtype=F64)[:, None] * inv
    return torch.stack([torch.cos(angle), torch.sin(angle)], -1).to(F32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s, kind = dict(case=dict(case)), case["kind"]
    if kind == "log_probs":
        t, v = case["tokens"], case["vocab"]
        s["logits"] = torch.randn(t, v, device="cuda", generator=gen) * 2.5
        # (half of the tokens are likely ones)
        some = torch.randint(0, v, (t,), device="cuda", generator=gen)
        s["targets"] = torch.where(torch.rand(t, device="cuda", generator=gen) < 0.5, s["logits"].argmax(-1), some).to(
            torch.int32)
        if own:
            s["ctx"] = _context()
        return s
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if kind == "append":
        t, n = case["tokens"], case["sequences"]
        s["q"] = torch.randn(t, h, d, device="cuda", generator=gen)
        s["k"], s["v"] = _rows(gen, t, kv, d), _rows(gen, t, kv, d)
        s["cos_sin"] = _cos_sin(case["rows"], d)
        if n == 1:
            first = int(torch.randint(0, case["rows"] - t + 1, (1,), device="cuda", generator=gen))
            s["positions"] = torch.arange(first, first + t, device="cuda", dtype=torch.int32)
            s["sequences"] = torch.zeros(t, device="cuda", dtype=torch.int32)
        else:
            s["positions"] = torch.randint(0, case["rows"], (t,), device="cuda", generator=gen, dtype=torch.int32)
            s["sequences"] = torch.arange(t, device="cuda", dtype=torch.int32)
        shape = (n, kv, case["rows"], d)
        s["cache"] = dict(k=torch.zeros(shape, device="cuda", dtype=torch.int8),
                          v=torch.zeros(shape, device="cuda", dtype=torch.int8),
                          ks=torch.ones(shape[:3], device="cuda"), vs=torch.ones(shape[:3], device="cuda"))
    elif kind == "attend":
        s["q"] = torch.randn(case["batch"], h, d, device="cuda", generator=gen)
        s["cache"] = _cache(gen, "int8", case["batch"], kv, case["rows"], d)
        s["len"] = torch.tensor(_lengths(case["batch"], case["rows"]), device="cuda", dtype=torch.int32)
    elif kind == "portion":
        s["q"] = torch.randn(case["tokens"], h, d, device="cuda", generator=gen)
        s["cache"] = _cache(gen, "int8", 1, kv, case["first"] + case["tokens"], d)
    else:
        s["q"] = torch.randn(case["batch"], h, d, device="cuda", generator=gen)
        s["cache"] = _cache(gen, case["dtype"], case["batch"], kv, case["rows"], d)
        s["prefix"] = _cache(gen, case["dtype"], 1, kv, case["prefix"], d)
        s["len"] = torch.tensor(_lengths(case["batch"], case["rows"]), device="cuda", dtype=torch.int32)
    if own:  # the handles that a program keeps: they name the tensors, no data is touched
        s["ctx"] = _context()
        s["kv"] = _handle(s["ctx"], s["cache"])
        if "prefix" in s:
            s["shared"] = _handle(s["ctx"], s["prefix"])
    return s


_ctx = None


def _context():
    global _ctx
    from quantibbler_b200.gpu import GpuContext
    if _ctx is None:
        _ctx = GpuContext.init()
        _ctx.set_stream(torch.cuda.current_stream().cuda_stream)
    return _ctx


def _handle(ctx, c):
    from quantibbler_b200.cache import KvCache
    return KvCache(ctx, c["k"], c["v"], c["ks"], c["vs"])


# ---------------------------------------------------------------------- one pass
def run(s):
    return _run_own(s) if own else _run_plain(s)


def _run_own(s):
    kind = s["case"]["kind"]
    if kind == "log_probs":
        from quantibbler_b200.scoring import log_probs
        r = log_probs(s["ctx"], s["logits"], s["targets"], top=s["case"]["top"])
        return dict(logprob=r.logprob, entropy=r.entropy, top_logprob=r.top_logprob, top_ids=r.top_ids)
    if kind == "append":
        q = s["kv"].append(s["k"], s["v"], s["cos_sin"], s["positions"], s["sequences"], q=s["q"])
        k, v = s["kv"].read(s["positions"], s["sequences"])
        return dict(q=q, k=k, v=v)
    if kind == "attend":
        return s["kv"].attend(s["q"], s["len"])
    if kind == "portion":
        return s["kv"].portion(s["q"], 0, s["case"]["first"])
    return s["kv"].attend(s["q"], s["len"], prefix=s["shared"], prefix_len=s["case"]["prefix"])


def _values(x, scale):
    return x.to(F32) if scale is None else x.to(F32) * scale[..., None]


def _weighted(scores, visible, values):
    """softmax over the visible entries of the last axis, times values."""
    scores = torch.where(visible, scores, -math.inf)
    w = torch.exp(scores - scores.amax(-1, keepdim=True))
    return (w @ values) / w.sum(-1, keepdim=True)


def _run_plain(s):
    case, kind = s["case"], s["case"]["kind"]
    if kind == "log_probs":
        x = s["logits"]
        x = x - x.amax(-1, keepdim=True)
        e = torch.exp(x)
        z = e.sum(-1, keepdim=True)
        logp = x - torch.log(z)
        # (the lowest index first among equals: a stable sort)
        best = (torch.sort(s["logits"], dim=-1, descending=True, stable=True).indices[:, :case["top"]] if case["top"] else
                s["targets"].new_empty(case["tokens"], 0, dtype=torch.int64))
        return dict(logprob=logp.gather(1, s["targets"].long()[:, None])[:, 0], entropy=-(e * logp).sum(-1) / z[:, 0],
                    top_logprob=logp.gather(1, best), top_ids=best.to(torch.int32))
    q, c = s["q"], s["cache"]
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if kind == "append":
        # (in 64 bits: a code may lie next to a border)
        cs = s["cos_sin"][s["positions"].long()].to(F64)[:, None]
        k, v = _rotated(s["k"], cs), s["v"].to(F64)
        k_codes, k_scale = _codes(k)
        v_codes, v_scale = _codes(v)
        at = (s["sequences"].long(), slice(None), s["positions"].long())
        c["k"][at], c["ks"][at], c["v"][at], c["vs"][at] = k_codes, k_scale, v_codes, v_scale
        return dict(q=_rotated(q, cs).to(F32), k=_values(c["k"][at], c["ks"][at]), v=_values(c["v"][at], c["vs"][at]))
    k, v = _values(c["k"], c["ks"]), _values(c["v"], c["vs"])
    g, scale = h // kv, 1.0 / math.sqrt(d)
    if kind == "portion":
        t, first = case["tokens"], case["first"]
        x = q.reshape(t, kv, g, d).permute(1, 2, 0, 3) * scale
        scores = x @ k[0, :, None].transpose(-1, -2)
        at = torch.arange(first, first + t, device=q.device)
        visible = torch.arange(first + t, device=q.device)[None] <= at[:, None]
        return _weighted(scores, visible, v[0, :, None]).permute(2, 0, 1, 3).reshape(t, h, d)
    b = case["batch"]
    x = q.reshape(b, kv, g, d) * scale
    scores = x @ k.transpose(-1, -2)
    visible = (torch.arange(case["rows"], device=q.device)[None] < s["len"][:, None])[:, None, None]
    if kind == "attend":
        return _weighted(scores, visible, v).reshape(b, h, d)
    p = s["prefix"]
    pk, pv = _values(p["k"], p["ks"])[0], _values(p["v"], p["vs"])[0]
    rows = x.permute(1, 0, 2, 3).reshape(kv, b * g, d)
    shared = (rows @ pk.transpose(-1, -2)).reshape(kv, b, g, -1).permute(1, 0, 2, 3)
    scores = torch.where(visible, scores, -math.inf)
    top = torch.maximum(scores.amax(-1, keepdim=True), shared.amax(-1, keepdim=True))
    mine, all_ = torch.exp(scores - top), torch.exp(shared - top)
    total = mine.sum(-1, keepdim=True) + all_.sum(-1, keepdim=True)
    from_prefix = (all_.permute(1, 0, 2, 3).reshape(kv, b * g, -1) @ pv).reshape(kv, b, g, d).permute(1, 0, 2, 3)
    return ((mine @ v + from_prefix) / total).reshape(b, h, d)


def _rotated(x, cs):
    """x [tokens, heads, dim] in 64 bits, pairs (i, i + dim / 2) turned by cs [tokens, 1, dim / 2, 2]."""
    a, b = x.to(F64).chunk(2, -1)
    return torch.cat([a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]], -1)


def _codes(x):
    scale = (x.abs().amax(-1) / 127.0).to(F32)
    scale = torch.where(scale == 0, 1.0, scale)
    return torch.round(x / scale.to(F64)[..., None]).clamp(-127, 127).to(torch.int8), scale


# ---------------------------------------------------------------------- what a pass cannot do without
def work(case):
    kind = case["kind"]
    if kind == "log_probs":
        t, v, top = case["tokens"], case["vocab"], case["top"]
        return dict(bytes=t * (v * 4 + 12 + 8 * top), flops=6 * t * v)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    if kind == "append":  # q, k, v read, q written, codes and scales written, read back and written as values
        t = case["tokens"]
        return dict(bytes=t * (8 * h * d + 8 * kv * d + 4 * kv * (d + 4) + 8 * kv * d + 4 * d + 8), flops=t * (h + 3 * kv) * d * 3)
    if kind == "portion":
        t, first = case["tokens"], case["first"]
        pairs = t * first + t * (t + 1) // 2
        return dict(bytes=8 * t * h * d + 2 * kv * (first + t) * (d + 4), flops=4 * d * h * pairs)
    per_row = 2 * (d + 4) if case.get("dtype", "int8") == "int8" else 4 * d
    keys = sum(_lengths(case["batch"], case["rows"]))
    prefix = case.get("prefix", 0)
    return dict(bytes=8 * case["batch"] * h * d + per_row * kv * (keys + prefix) + 4 * case["batch"],
                flops=4 * d * h * (keys + case["batch"] * prefix))


# ---------------------------------------------------------------------- the definition, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "log_probs":
        return _exact_log_probs(s, case)
    if kind == "append":
        return _exact_append(s, case)
    h, kv, d = case["heads"], case["kv_heads"], case["dim"]
    g, q = h // kv, s["q"].double()

    def stored(c, seq, head, n):
        k, v = c["k"][seq, head, :n].double(), c["v"][seq, head, :n].double()
        if c["ks"] is not None:
            k, v = k * c["ks"][seq, head, :n].double()[:, None], v * c["vs"][seq, head, :n].double()[:, None]
        return k, v

    out = torch.empty(q.shape, device=q.device, dtype=F64)
    if kind == "portion":
        t, first = case["tokens"], case["first"]
        hidden = torch.ones(t, first + t, device=q.device, dtype=torch.bool).triu(first + 1)
        for head in range(h):
            k, v = stored(s["cache"], 0, head // g, first + t)
            x = (q[:, head] @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf)
            out[:, head] = torch.softmax(x, -1) @ v
        return out
    for b, n in enumerate(_lengths(case["batch"], case["rows"])):
        for head in range(kv):
            k, v = stored(s["cache"], b, head, n)
            if kind == "shared":
                pk, pv = stored(s["prefix"], 0, head, case["prefix"])
                k, v = torch.cat([pk, k]), torch.cat([pv, v])
            mine = slice(head * g, (head + 1) * g)
            out[b, mine] = torch.softmax(q[b, mine] @ k.T / math.sqrt(d), -1) @ v
    return out


def _exact_log_probs(s, case):
    logprob, entropy, best, ids = [], [], [], []
    for x, target in zip(s["logits"].split(64), s["targets"].long().split(64)):
        p = torch.log_softmax(x.double(), -1)
        logprob.append(p[torch.arange(len(p), device=p.device), target])
        entropy.append(-(p.exp() * p).sum(-1))
        order = torch.argsort(-x, dim=-1, stable=True)[:, :case["top"]]
        ids.append(order.to(torch.int32))
        best.append(torch.take_along_dim(p, order, -1))
    return dict(logprob=torch.cat(logprob), entropy=torch.cat(entropy), top_logprob=torch.cat(best), top_ids=torch.cat(ids))


def _exact_append(s, case):
    half = case["dim"] // 2
    turn = s["cos_sin"][s["positions"].long()].double()
    turn = torch.complex(turn[..., 0], turn[..., 1])[:, None]

    def turned(x):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn
        return torch.cat([z.real, z.imag], -1)

    def stored(x):
        step = (x.abs().max(-1, keepdim=True).values / 127).float().double()
        return step * (x / step).round().clamp(-127, 127)

    return dict(q=turned(s["q"]), k=stored(turned(s["k"])), v=stored(s["v"].double()))
