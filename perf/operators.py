"""Measured cases of the long-context cache operators.

Four operators that work on one paged KV cache and are used in this order by a
program that serves long contexts:

  rotary   rotary positions applied to queries and keys (half or interleaved
           pairs, all or part of the head, frequencies scaled for long
           contexts), keys and values appended to the cache; and the rotation
           alone, back and forth
  shared   attention of a batch whose requests share long prefixes: the keys
           of a prefix are read once for all the requests of its group
  weighted single-token attention that adds every key's attention weight,
           summed over the query heads of its KV head, to a weight per cache
           slot
  evict    per request and KV head: the slots that an eviction by those
           weights keeps, and the moves that make the kept ones contiguous

A case is a dict of plain values.  ``run`` computes the operators in their
plain form, or calls the framework's when ``own`` is set.
"""
import math

import numpy as np
import torch

own = False

DEV = "cuda" if torch.cuda.is_available() else "cpu"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
TABLE = 131072      # longest position of the plain form's table of angles


def listed():
    return [
        # decode step of one request: launch latency
        dict(name="rotary 1 token", kind="rotary", tokens=1, nq=32, nkv=8, hd=128, rot=128, pairs="half",
             scaling="llama3", dtype="bf16", block=16, track=False, sequences=1),
        # a full prefill step into a cache that also keeps weights and positions
        dict(name="rotary prompt", kind="rotary", tokens=16384, nq=64, nkv=8, hd=128, rot=64, pairs="interleaved",
             scaling="yarn", dtype="fp16", block=32, track=True, sequences=1),
        # the rotation's gradient (rotation back) on part of small heads, an odd token count
        dict(name="rotary back", kind="rotate", tokens=1111, nq=12, nkv=0, hd=64, rot=48, pairs="half",
             scaling="linear", dtype="bf16", block=16, track=False, sequences=1),
        # two requests behind one short system prompt: launch latency
        dict(name="shared pair", kind="shared", requests=2, groups=1, prefix=517, own_lo=1, own_hi=33, queries=1,
             nq=32, nkv=8, hd=128, dtype="bf16", block=16),
        # a decode batch behind one system prompt
        dict(name="shared system prompt", kind="shared", requests=64, groups=1, prefix=4096, own_lo=16, own_hi=256,
             queries=1, nq=32, nkv=8, hd=128, dtype="bf16", block=16),
        # questions about four long documents
        dict(name="shared documents", kind="shared", requests=128, groups=4, prefix=16384, own_lo=100, own_hi=500,
             queries=1, nq=64, nkv=8, hd=128, dtype="fp16", block=32),
        # chunks of a few query tokens, multi-head attention, several short prefixes
        dict(name="shared chunks", kind="shared", requests=24, groups=5, prefix=1500, own_lo=40, own_hi=90,
             queries=9, nq=40, nkv=40, hd=128, dtype="bf16", block=16),
        # one short request of a small model: launch latency
        dict(name="weighted 1 request", kind="weighted", requests=1, len_lo=129, len_hi=129, nq=4, nkv=2, hd=64,
             dtype="bf16", block=16),
        # a ragged decode batch, multi-head attention
        dict(name="weighted batch", kind="weighted", requests=30, len_lo=300, len_hi=2300, nq=40, nkv=40, hd=128,
             dtype="bf16", block=16),
        # a few very long contexts
        dict(name="weighted long", kind="weighted", requests=4, len_lo=20000, len_hi=65001, nq=32, nkv=8, hd=128,
             dtype="fp16", block=64),
        # steady state of a capped cache: one token over the cap
        dict(name="evict one", kind="evict", requests=48, len_lo=1025, len_hi=1025, keep=1024, sinks=4, recent=64,
             nq=32, nkv=8, hd=128, dtype="bf16", block=16),
        # prompts of many thousands of tokens cut down to the cap at once
        dict(name="evict prompts", kind="evict", requests=8, len_lo=6001, len_hi=20000, keep=4096, sinks=4,
             recent=512, nq=32, nkv=8, hd=128, dtype="bf16", block=16),
    ]


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi]."""
    return min(hi, int(lo * math.exp(rng.random() * math.log((hi + 1) / lo))))


def draw(rng):
    most = {}
    for c in listed():
        w, m = work(c), most.setdefault(c["kind"], {"bytes": 0.0, "flops": 0.0})
        for k in m:
            m[k] = max(m[k], w[k])
    while True:
        kind = rng.choice(["rotary", "rotate", "shared", "shared", "weighted", "weighted", "evict", "evict"])
        hd = rng.choice([64, 128, 128])
        nkv = rng.choice([1, 2, 4, 8, 8, 10, 40])
        group = rng.choice([1, 1, 2, 4, 5, 8]) if nkv <= 10 else 1
        c = dict(kind=kind, nq=nkv * group, nkv=nkv, hd=hd, dtype=rng.choice(["bf16", "bf16", "fp16"]),
                 block=rng.choice([8, 16, 16, 24, 32, 64]))
        if kind in ("rotary", "rotate"):
            c.update(tokens=_log(rng, 1, 16384), rot=rng.choice([hd, hd, hd // 2, 3 * hd // 4]),
                     pairs=rng.choice(["half", "interleaved"]), sequences=rng.choice([1, 1, 9]),
                     scaling=rng.choice(["none", "linear", "llama3", "yarn"]), track=rng.random() < 0.5)
            if kind == "rotate":
                c.update(nkv=0, track=False)
        elif kind == "shared":
            n = _log(rng, 1, 200)
            lo = _log(rng, 1, 300)
            c.update(requests=n, groups=rng.randint(1, min(n, 6)), prefix=_log(rng, 30, 16384), own_lo=lo,
                     own_hi=lo + _log(rng, 1, 300), queries=rng.choice([1, 1, 1, 2, 5, 12]))
        elif kind == "weighted":
            lo = _log(rng, 1, 50000)
            c.update(requests=_log(rng, 1, 100), len_lo=lo, len_hi=min(65001, lo + _log(rng, 1, lo + 8)))
        else:
            lo = _log(rng, 40, 20000)
            hi = min(40000, lo + _log(rng, 1, lo))
            keep = _log(rng, 24, hi)
            c.update(requests=_log(rng, 1, 64), len_lo=lo, len_hi=hi, keep=keep, sinks=rng.choice([0, 4]),
                     recent=rng.randint(0, keep - 8))
        w = work(c)
        if all(w[k] <= most["rotary" if kind == "rotate" else kind][k] for k in w):
            return c


# ------------------------------------------------------------------ lengths
def _spread(n, lo, hi):
    """``n`` whole numbers over [lo, hi] in no order, both ends among them where n allows."""
    return [hi if n == 1 else lo + (i * 7919 % n) * (hi - lo) // (n - 1) for i in range(n)]


def _shared_lengths(c):
    """Group of each request, prefix lengths, own lengths, query counts."""
    n, g = c["requests"], c["groups"]
    group = [i * g // n for i in range(n)]
    prefix = [max(1, c["prefix"] - 37 * i) for i in range(g)]
    queries = [1 + (3 * i + c["queries"] - 1) % c["queries"] for i in range(n)]
    owned = [max(o, q) for o, q in zip(_spread(n, c["own_lo"], c["own_hi"]), queries)]
    return group, prefix, owned, queries


def work(c):
    hd, nq, nkv, el = c["hd"], c["nq"], c["nkv"], 2
    if c["kind"] in ("rotary", "rotate"):
        t, heads = c["tokens"], nq + 2 * nkv
        per = 2 * heads * hd * el + 12 + (8 * nkv if c["track"] else 0)
        return {"bytes": float(t * per), "flops": 3.0 * t * (nq + nkv) * c["rot"]}
    if c["kind"] == "shared":
        group, prefix, owned, queries = _shared_lengths(c)
        t = sum(queries)
        keys = sum(prefix) + sum(owned)
        seen = sum(n * prefix[g] + sum(o - n + j + 1 for j in range(n)) for g, o, n in zip(group, owned, queries))
        return {"bytes": float(2 * keys * nkv * hd * el + 2 * t * nq * hd * el), "flops": 4.0 * seen * nq * hd}
    lens = _spread(c["requests"], c["len_lo"], c["len_hi"])
    if c["kind"] == "weighted":
        return {"bytes": float(sum(lens) * nkv * (2 * hd * el + 8) + 2 * len(lens) * nq * hd * el),
                "flops": 4.0 * sum(lens) * nq * hd}
    moved = sum(c["keep"] * (n - c["keep"]) / n for n in lens if n > c["keep"])   # holes expected below the cap
    return {"bytes": float(nkv * (8 * sum(lens) + moved * (4 * hd * el + 16 + 8))), "flops": 1.0 * nkv * sum(lens)}


# ------------------------------------------------------------------- inputs
def _scaling(c):
    """The scaling entry of a model's configuration."""
    return {"none": None,
            "linear": {"rope_type": "linear", "factor": 4.0},
            "llama3": {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                       "original_max_position_embeddings": 8192},
            "yarn": {"rope_type": "yarn", "factor": 16.0, "beta_fast": 32.0, "beta_slow": 1.0,
                     "original_max_position_embeddings": 4096}}[c["scaling"]]


THETA = 500000.0


def _frequencies(c):
    """Radians per position of each pair (64 bits), and the factor on cos and sin."""
    d, s = c["rot"], _scaling(c)
    f = THETA ** (-torch.arange(0, d, 2, dtype=torch.float64) / d)
    if s is None:
        return f, 1.0
    if s["rope_type"] == "linear":
        return f / s["factor"], 1.0
    old = s["original_max_position_embeddings"]
    if s["rope_type"] == "llama3":
        turns = old * f / (2 * math.pi)     # turns within the original context
        mix = ((turns - s["low_freq_factor"]) / (s["high_freq_factor"] - s["low_freq_factor"])).clamp(0, 1)
        return f * (mix + (1 - mix) / s["factor"]), 1.0
    at = [d * math.log(old / (b * 2 * math.pi)) / (2 * math.log(THETA)) for b in (s["beta_fast"], s["beta_slow"])]
    lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d - 1)
    ramp = ((torch.arange(d // 2, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
    return f * (1 - ramp + ramp / s["factor"]), 0.1 * math.log(s["factor"]) + 1.0


def _rand(g, *shape):
    return torch.randn(*shape, generator=g, device=DEV)


def _cache(c, g, pages_needed):
    """A two-layer pool with a page more than needed (the last one pads the
    tables), its pages in random order, filled with values."""
    pages = pages_needed + 1
    pool = torch.empty(pages, 2, 2, c["block"], c["nkv"], c["hd"], device=DEV, dtype=DTYPES[c["dtype"]])
    for l in range(2):
        for kv in range(2):
            pool[:, l, kv] = _rand(g, *pool[:, l, kv].shape).to(pool.dtype)
    order = torch.randperm(pages_needed, generator=g, device=DEV)
    return pool, order


def _tables(c, lens, order, at=0):
    """Page table [n, widest] of lengths ``lens``, padded with the last page, and the pages used."""
    need = [-(-n // c["block"]) for n in lens]
    table = torch.full((len(lens), max(need)), order.numel(), dtype=torch.int64)
    o = order.cpu()
    for i, n in enumerate(need):
        table[i, :n] = o[at:at + n]
        at += n
    return table, at


def _cover(c, *lens):
    return sum(-(-n // c["block"]) for l in lens for n in l)


def _index(per, counts):
    """Rows of ``per`` items of ``counts`` consecutive numbers, padded with 0; and the (row, column) of each number."""
    most = max(counts)
    idx = torch.zeros(len(counts), most, dtype=torch.int64)
    row, col, at = [], [], 0
    for i, n in enumerate(counts):
        idx[i, :n] = torch.arange(at, at + n)
        row += [i] * n
        col += range(n)
        at += n
    return idx.to(DEV), torch.tensor(row, device=DEV), torch.tensor(col, device=DEV)


def prepare(c, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    dt = DTYPES[c["dtype"]]
    s = dict(c=c)
    if c["kind"] in ("rotary", "rotate"):
        t = c["tokens"]
        f, m = _frequencies(c)
        ang = torch.arange(TABLE, dtype=torch.float64, device=DEV)[:, None] * f.to(DEV)[None]
        s["cos_sin"] = torch.cat([ang.cos() * m, ang.sin() * m], 1).float()
        # one prompt at consecutive positions, or tokens of several sequences
        first = torch.randint(0, TABLE - t, (c["sequences"],), generator=g, device=DEV)
        each = -(-t // c["sequences"])
        at = torch.arange(t, device=DEV)
        s["positions"] = (first[at // each] + at % each).int()
        if c["kind"] == "rotate":
            # the query heads of a wider projection: a strided view
            s["wide"] = _rand(g, t, c["nq"] + 4, c["hd"]).to(dt)
            s["x"] = s["wide"][:, :c["nq"]]
            s["out"] = torch.empty(t, c["nq"], c["hd"], device=DEV, dtype=dt)
        else:
            s["qkv"] = _rand(g, t, c["nq"] + 2 * c["nkv"], c["hd"]).to(dt)
            s["out"] = torch.empty(t, c["nq"], c["hd"], device=DEV, dtype=dt)
            s["pool"], order = _cache(c, g, -(-t // c["block"]))
            s["pages"] = order[at // c["block"]].int()
            s["slots"] = (at % c["block"]).int()
            s["weights"] = _rand(g, s["pool"].shape[0], c["nkv"], c["block"]).abs() if c["track"] else None
            s["slot_positions"] = torch.zeros_like(s["weights"], dtype=torch.int32) if c["track"] else None
    elif c["kind"] == "shared":
        group, prefix, owned, queries = _shared_lengths(c)
        s["pool"], order = _cache(c, g, _cover(c, prefix, owned))
        s["prefix_table"], at = _tables(c, prefix, order)
        s["own_table"], _ = _tables(c, owned, order, at)
        s["prefix_len"] = torch.tensor(prefix, device=DEV)
        s["own_len"] = torch.tensor(owned, device=DEV)
        s["queries"] = torch.tensor(queries, device=DEV)
        s["req_idx"], s["tok_req"], s["tok_at"] = _index(c, queries)
        s["group_idx"], s["tok_group"], s["tok_in_group"] = _index(
            c, [sum(n for n, k in zip(queries, group) if k == i) for i in range(c["groups"])])
        s["q"] = _rand(g, sum(queries), c["nq"], c["hd"]).to(dt)
    else:
        lens = _spread(c["requests"], c["len_lo"], c["len_hi"])
        s["pool"], order = _cache(c, g, _cover(c, lens))
        s["table"], _ = _tables(c, lens, order)
        s["lens"] = torch.tensor(lens, device=DEV)
        # about one earlier pass's worth of weight on every slot
        s["weights"] = _rand(g, s["pool"].shape[0], c["nkv"], c["block"]).square() * (c["nq"] / c["nkv"] / max(lens))
        if c["kind"] == "weighted":
            s["q"] = _rand(g, c["requests"], c["nq"], c["hd"]).to(dt)
        else:
            # earlier evictions have left each head's slots out of order
            n, width = c["requests"], s["table"].shape[1]
            place = torch.rand(n, c["nkv"], width * c["block"], generator=g, device=DEV).argsort(-1).int()
            pos = torch.zeros_like(s["weights"], dtype=torch.int32)
            pos[s["table"].to(DEV)] = place.reshape(n, c["nkv"], width, c["block"]).transpose(1, 2)
            pos[-1] = 0     # the padding page
            s["slot_positions"] = pos
            s["newest"] = width * c["block"] - 1
            # the moves are applied to a second copy, so that every pass finds the weights of the first
            s["moved_weights"], s["moved_positions"] = s["weights"].clone(), pos.clone()
    for k in ("prefix_table", "own_table", "table"):
        if k in s:
            s[k + "_list"] = s[k].tolist()
            s[k] = s[k].to(DEV)
    if own:
        _handles(c, s)
    return s


def _handles(c, s):
    """What a program that calls the operators keeps: the cache's handle, the
    rotation's frequencies, the step's plan."""
    from kunserve_b200 import ops
    from kunserve_b200.kv.layout import KVLayout

    if "pool" in s:
        p = s["pool"]
        s["kv"] = ops.PagedKV(p, KVLayout(p.shape[0], 2, c["block"], c["nkv"], c["hd"], 2))
    if c["kind"] in ("rotary", "rotate"):
        s["rotary"] = ops.Rotary(c["hd"], rotary_dim=c["rot"], theta=THETA, interleaved=c["pairs"] == "interleaved",
                                 scaling=_scaling(c), device=DEV)
    elif c["kind"] == "shared":
        group, prefix, owned, queries = _shared_lengths(c)
        s["plan"] = ops.SharedPrefixPlan(
            [ops.PrefixGroup(s["prefix_table_list"][i][:-(-n // c["block"])], n,
                             [(s["own_table_list"][j][:-(-owned[j] // c["block"])], owned[j], queries[j])
                              for j in range(c["requests"]) if group[j] == i]) for i, n in enumerate(prefix)],
            s["kv"], c["nq"])
    else:
        lens = _spread(c["requests"], c["len_lo"], c["len_hi"])
        s["plan"] = ops.DecodePlan([t[:-(-n // c["block"])] for t, n in zip(s["table_list"], lens)], lens, s["kv"],
                                   c["nq"], newest=[s.get("newest", n - 1) for n in lens])


# ------------------------------------------------------------- plain forms
def _turn(x, cs, c):
    """x [t, h, hd] in 32 bits with its first ``rot`` dims turned by cs [t, rot] (cos, sin)."""
    r = c["rot"]
    cos, sin = cs[:, None, :r // 2], cs[:, None, r // 2:]
    if c["pairs"] == "half":
        a, b = x[..., :r // 2], x[..., r // 2:r]
        return torch.cat([a * cos - b * sin, b * cos + a * sin, x[..., r:]], -1)
    a, b = x[..., 0:r:2], x[..., 1:r:2]
    return torch.cat([torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2), x[..., r:]], -1)


def _gather(pool, table, kv):
    """Keys or values of layer 1 behind a page table: [n, slots, nkv, hd] in 32 bits."""
    return pool[table, 1, kv].flatten(1, 2).float()


def _scores(q, k):
    """q [n, t, nq, d] against k [n, l, nkv, d]: [n, t, nq, l]."""
    n, t, nq, d = q.shape
    a = q.reshape(n, t, k.shape[2], -1, d).transpose(1, 2).flatten(2, 3)
    s = a @ k.permute(0, 2, 3, 1)
    return s.reshape(n, k.shape[2], t, -1, k.shape[1]).transpose(1, 2).flatten(2, 3)


def _mix(p, v):
    """p [n, t, nq, l] times v [n, l, nkv, d]: [n, t, nq, d]."""
    n, t, nq, l = p.shape
    a = p.reshape(n, t, v.shape[2], -1, l).transpose(1, 2).flatten(2, 3)
    o = a @ v.transpose(1, 2)
    return o.reshape(n, v.shape[2], t, -1, v.shape[3]).transpose(1, 2).flatten(2, 3)


def _softmax(s):
    m = s.amax(-1, keepdim=True)
    e = torch.exp(s - torch.where(m == -math.inf, 0.0, m))
    return e / e.sum(-1, keepdim=True).clamp_min(1e-30)


def _rotary(s):
    c = s["c"]
    cs = s["cos_sin"][s["positions"].long()]
    if c["kind"] == "rotate":
        back = torch.cat([cs[:, :c["rot"] // 2], -cs[:, c["rot"] // 2:]], 1)
        s["out"].copy_(_turn(s["x"].float(), back, c))
        return s["out"]
    nq, nkv = c["nq"], c["nkv"]
    x = s["qkv"]
    s["out"].copy_(_turn(x[:, :nq].float(), cs, c))
    pages, slots = s["pages"].long(), s["slots"].long()
    s["pool"][pages, 1, 0, slots] = _turn(x[:, nq:nq + nkv].float(), cs, c).to(x.dtype)
    s["pool"][pages, 1, 1, slots] = x[:, nq + nkv:]
    if not c["track"]:
        return s["out"], s["pool"]
    s["weights"][pages, :, slots] = 0.0
    s["slot_positions"][pages, :, slots] = s["positions"][:, None].expand(-1, nkv)
    return s["out"], s["pool"], s["weights"], s["slot_positions"]


def _shared(s):
    q, c = s["q"].float(), s["c"]
    kp, ko = _gather(s["pool"], s["prefix_table"], 0), _gather(s["pool"], s["own_table"], 0)
    a = _scores(q[s["group_idx"]], kp)[s["tok_group"], s["tok_in_group"]]
    b = _scores(q[s["req_idx"]], ko)[s["tok_req"], s["tok_at"]]
    at = torch.arange(kp.shape[1], device=q.device)
    a = a.masked_fill((at >= s["prefix_len"][s["tok_group"], None])[:, None], -math.inf)
    last = s["own_len"][s["tok_req"]] - s["queries"][s["tok_req"]] + s["tok_at"]   # newest own key a token sees
    at = torch.arange(ko.shape[1], device=q.device)
    b = b.masked_fill((at > last[:, None])[:, None], -math.inf)
    p = _softmax(torch.cat([a, b], -1) / math.sqrt(c["hd"]))
    a, b = p[..., :kp.shape[1]], p[..., kp.shape[1]:]
    o = _mix(a[s["group_idx"]], _gather(s["pool"], s["prefix_table"], 1))[s["tok_group"], s["tok_in_group"]]
    o = o + _mix(b[s["req_idx"]], _gather(s["pool"], s["own_table"], 1))[s["tok_req"], s["tok_at"]]
    return o.to(s["q"].dtype)


def _weighted(s):
    q, c = s["q"].float(), s["c"]
    k = _gather(s["pool"], s["table"], 0)
    a = _scores(q[:, None], k) / math.sqrt(c["hd"])
    at = torch.arange(k.shape[1], device=q.device)
    p = _softmax(a.masked_fill((at >= s["lens"][:, None])[:, None, None], -math.inf))
    o = _mix(p, _gather(s["pool"], s["table"], 1))[:, 0]
    w = p.reshape(q.shape[0], c["nkv"], -1, s["table"].shape[1], c["block"]).sum(2).transpose(1, 2)
    s["weights"][s["table"]] = s["weights"][s["table"]] + w
    return o.to(s["q"].dtype), s["weights"]


def _evict(s):
    c, table, bs = s["c"], s["table"], s["c"]["block"]
    n, width = table.shape
    w = s["weights"][table].transpose(1, 2).flatten(2)
    pos = s["slot_positions"][table].transpose(1, 2).flatten(2)
    at = torch.arange(width * bs, device=w.device)
    valid = at < s["lens"][:, None, None]
    w = torch.where((pos < c["sinks"]) | (pos > s["newest"] - c["recent"]), math.inf, w)
    order = torch.where(valid, w, -math.inf).sort(dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(-1, order, at.expand_as(order))
    left = s["lens"].clamp_max(c["keep"])[:, None, None]
    kept = rank < left
    hole, mover = (at < left) & ~kept, (at >= left) & kept
    cap = max([min(c["keep"], l - c["keep"]) for l in _spread(n, c["len_lo"], c["len_hi"])] + [0])
    moves = torch.full((n, c["nkv"], cap + 1, 2), -1, dtype=torch.int32, device=w.device)
    full = at.int().expand_as(hole)
    for i, m in enumerate((hole, mover)):
        moves[..., i].scatter_(2, torch.where(m, m.cumsum(-1) - 1, cap), full)
    moves = moves[:, :, :cap].contiguous()
    # the moves, the unused ones within the padding page
    real = moves >= 0
    row = torch.arange(n, device=w.device)[:, None, None, None]
    page = torch.where(real, table[row, moves.clamp_min(0).long() // bs], s["pool"].shape[0] - 1)
    slot = torch.where(real, moves.long() % bs, 0)
    head = torch.arange(c["nkv"], device=w.device)[:, None].expand(n, c["nkv"], cap)
    (pd, ps), (sd, ss) = page.unbind(-1), slot.unbind(-1)
    s["pool"][pd, 1, :, sd, head] = s["pool"][ps, 1, :, ss, head]
    for x in (s["moved_weights"], s["moved_positions"]):
        x[pd, head, sd] = x[ps, head, ss]
    return moves, hole.sum(-1).int(), s["pool"], s["moved_weights"], s["moved_positions"]


# ------------------------------------------------------- one pass of a case
def run(s):
    c = s["c"]
    if not own:
        return {"rotary": _rotary, "rotate": _rotary, "shared": _shared, "weighted": _weighted,
                "evict": _evict}[c["kind"]](s)
    from kunserve_b200 import ops

    if c["kind"] == "rotate":
        return ops.rotary_apply(s["x"], s["positions"], s["rotary"], out=s["out"], inverse=True)
    if c["kind"] == "rotary":
        ops.rotary_append(s["qkv"], s["positions"], s["pages"], s["slots"], s["rotary"], s["kv"], 1, out=s["out"],
                          weights=s["weights"], slot_positions=s["slot_positions"])
        return (s["out"], s["pool"], s["weights"], s["slot_positions"]) if c["track"] else (s["out"], s["pool"])
    if c["kind"] == "shared":
        return ops.shared_prefix_attention(s["q"], s["kv"], 1, s["plan"])
    if c["kind"] == "weighted":
        return ops.weighted_decode_attention(s["q"], s["kv"], 1, s["plan"], s["weights"]), s["weights"]
    moves, counts = ops.select_evictions(s["weights"], s["slot_positions"], s["plan"], c["keep"], sinks=c["sinks"],
                                         recent=c["recent"])
    ops.compact_cache(s["kv"], 1, s["plan"], moves, counts, s["moved_weights"], s["moved_positions"])
    return moves, counts, s["pool"], s["moved_weights"], s["moved_positions"]


# ------------------------------------------------------------------ 64 bits
def exact(c, seed):
    s = prepare(c, seed)
    if c["kind"] in ("rotary", "rotate"):
        return _exact_rotary(c, s)
    if c["kind"] == "shared":
        return _exact_shared(c, s)
    if c["kind"] == "weighted":
        return _exact_weighted(c, s)
    return _exact_evict(c, s)


def _exact_rotary(c, s):
    f, m = _frequencies(c)
    z = m * torch.exp(1j * s["positions"].double()[:, None] * f.to(DEV))[:, None]     # a turn as a complex factor
    half = torch.arange(c["rot"] // 2, device=DEV)
    first, second = (half, half + c["rot"] // 2) if c["pairs"] == "half" else (2 * half, 2 * half + 1)

    def turned(x, z):
        y = x.double()
        v = torch.complex(y[..., first], y[..., second]) * z
        y[..., first], y[..., second] = v.real, v.imag
        return y

    if c["kind"] == "rotate":
        return turned(s["x"], z.conj())
    nq, nkv = c["nq"], c["nkv"]
    pool = s["pool"].double()
    pages, slots = s["pages"].long(), s["slots"].long()
    pool[pages, 1, 0, slots] = turned(s["qkv"][:, nq:nq + nkv], z)
    pool[pages, 1, 1, slots] = s["qkv"][:, nq + nkv:].double()
    if not c["track"]:
        return turned(s["qkv"][:, :nq], z), pool
    w = s["weights"].double()
    w[pages, :, slots] = 0
    return turned(s["qkv"][:, :nq], z), pool, w, None


def _attend(q, keys, values, group):
    """Softmax attention of one token's heads q [nq, d] over keys, values [l, nkv, d], all in 64 bits: outputs, weights."""
    k, v = keys.repeat_interleave(group, 1), values.repeat_interleave(group, 1)
    a = torch.einsum("hd,lhd->hl", q, k) / math.sqrt(q.shape[-1])
    p = torch.exp(a - torch.logsumexp(a, -1, keepdim=True))
    return torch.einsum("hl,lhd->hd", p, v), p


def _exact_shared(c, s):
    group, prefix, owned, queries = _shared_lengths(c)
    rows, q, t = [], s["q"].double(), 0
    for i, (o, n) in enumerate(zip(owned, queries)):
        pre = [s["pool"][s["prefix_table"][group[i]], 1, kv].flatten(0, 1)[:prefix[group[i]]] for kv in (0, 1)]
        mine = [s["pool"][s["own_table"][i], 1, kv].flatten(0, 1) for kv in (0, 1)]
        for j in range(n):
            seen = o - n + j + 1
            k, v = (torch.cat([a, b[:seen]]).double() for a, b in zip(pre, mine))
            rows.append(_attend(q[t], k, v, c["nq"] // c["nkv"])[0])
            t += 1
    return torch.stack(rows)


def _exact_weighted(c, s):
    w = s["weights"].double()
    rows = []
    for i, n in enumerate(s["lens"].tolist()):
        k, v = (s["pool"][s["table"][i], 1, kv].flatten(0, 1)[:n].double() for kv in (0, 1))
        o, p = _attend(s["q"][i].double(), k, v, c["nq"] // c["nkv"])
        rows.append(o)
        p = p.reshape(c["nkv"], -1, n).sum(1)
        at = torch.arange(n, device=DEV)
        w[s["table"][i][at // c["block"]], :, at % c["block"]] += p.T
    return torch.stack(rows), w


def _exact_evict(c, s):
    bs, nkv = c["block"], c["nkv"]
    table, w, pos = (s[k].cpu().numpy() for k in ("table", "weights", "slot_positions"))
    lens = s["lens"].tolist()
    cap = max([min(c["keep"], n - c["keep"]) for n in lens] + [0])
    moves = np.full((len(lens), nkv, cap, 2), -1, np.int32)
    counts = np.zeros((len(lens), nkv), np.int32)
    pool = s["pool"].double()
    mw, mp = s["moved_weights"].double(), s["moved_positions"].clone()
    for i, n in enumerate(lens):
        left = min(n, c["keep"])
        at = np.arange(n)
        for h in range(nkv):
            x = w[table[i][at // bs], h, at % bs].astype(np.float64)
            p = pos[table[i][at // bs], h, at % bs]
            x[(p < c["sinks"]) | (p > s["newest"] - c["recent"])] = np.inf
            keep = np.zeros(n, bool)
            keep[np.lexsort((at, -x))[:left]] = True
            dst, src = np.nonzero(~keep[:left])[0], left + np.nonzero(keep[left:])[0]
            counts[i, h] = len(dst)
            moves[i, h, :len(dst), 0], moves[i, h, :len(src), 1] = dst, src
            (pd, sd), (ps, ss) = ((torch.tensor(a, device=DEV) for a in (table[i][m // bs], m % bs))
                                  for m in (dst, src))
            for x in (pool[:, 1, 0], pool[:, 1, 1]):
                x[pd, sd, h] = x[ps, ss, h]
            for x in (mw, mp):
                x[pd, h, sd] = x[ps, h, ss]
    return torch.from_numpy(moves), torch.from_numpy(counts), pool, mw, mp
