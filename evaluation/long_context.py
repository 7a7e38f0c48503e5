"""Decoding long contexts on the cache operators, on one GPU, with a small
decoder of random weights.

    python evaluation/long_context.py shared --requests 64 --prefix 4096 --steps 32
    python evaluation/long_context.py capped --requests 8 --prompt 6000 --cap 1024 --steps 32
    python evaluation/long_context.py shared --check

``shared``: requests behind one system prompt.  The prompt's keys are stored
once; every step appends each request's token with rotary positions scaled
for long contexts (``rotary_append``) and attends with the prompt's keys read
once for the batch (``shared_prefix_attention``).

``capped``: requests that keep at most ``--cap`` tokens (plus ``--slack``
before the next eviction).  Every step accumulates each cached token's
attention weight (``weighted_decode_attention``); a request over the cap keeps
its first and newest tokens and the heaviest of the rest
(``select_evictions``, ``compact_cache``), and the pages behind are free.

``--check`` compares the attention outputs of both ways to store the same
requests, behind a shared prefix and in whole caches whose cap is never
reached, layer by layer and request by request, after the prompts and after a
step on the same tokens.
"""
import argparse
import json
import math
import os
import sys
import time

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from kunserve_b200 import ops  # noqa: E402
from kunserve_b200.kv.layout import KVLayout  # noqa: E402

SCALING = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
           "original_max_position_embeddings": 8192}


class Decoder:
    """Attention layers of random bf16 weights over a paged cache."""

    def __init__(self, pages: int, layers=4, hidden=1024, nq=16, nkv=4, hd=128, vocab=4096, block=16, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(*shape):
            return (torch.randn(*shape, generator=g, device="cuda") / math.sqrt(shape[-1])).bfloat16()

        self.nq, self.nkv, self.hd, self.layers, self.block = nq, nkv, hd, layers, block
        self.embed = weight(vocab, hidden) * math.sqrt(hidden)
        self.w_qkv = [weight((nq + 2 * nkv) * hd, hidden) for _ in range(layers)]
        self.w_o = [weight(hidden, nq * hd) for _ in range(layers)]
        self.layout = KVLayout(pages, layers, block, nkv, hd, 2)
        self.pool = torch.empty(self.layout.base_bytes // 2, dtype=torch.bfloat16, device="cuda")
        self.kv = ops.PagedKV(self.pool, self.layout)
        self.rotary = ops.Rotary(hd, theta=500000.0, scaling=SCALING)
        side = (layers, self.kv.pages_total, nkv, block)
        self.weights = torch.zeros(side, device="cuda")
        self.positions = torch.zeros(side, dtype=torch.int32, device="cuda")
        self.attended = []       # each layer's attention of the last run

    def run(self, tokens, positions, pages, slots, attend):
        """Logits of ``tokens`` appended at the given cache places; ``attend``
        (layer, queries) gives a layer's attention."""
        i32 = [torch.tensor(v, dtype=torch.int32, device="cuda") for v in (positions, pages, slots)]
        h = self.embed[tokens]
        self.attended = []
        for layer in range(self.layers):
            x = torch.nn.functional.rms_norm(h, h.shape[-1:])
            qkv = (x @ self.w_qkv[layer].t()).view(len(positions), -1, self.hd)
            ops.rotary_append(qkv, *i32, self.rotary, self.kv, layer, weights=self.weights[layer],
                              slot_positions=self.positions[layer])
            self.attended.append(attend(layer, qkv[:, :self.nq]).flatten(1))
            h = h + self.attended[-1] @ self.w_o[layer].t()
        return torch.nn.functional.rms_norm(h, h.shape[-1:]) @ self.embed.t()


class Pages:
    """Free pages of the pool, and the places of a sequence's tokens."""

    def __init__(self, total, block):
        self.free, self.block = list(range(total))[::-1], block

    def grow(self, table, tokens):
        while len(table) * self.block < tokens:
            table.append(self.free.pop())
        return table

    def shrink(self, table, tokens):
        while (len(table) - 1) * self.block >= tokens:
            self.free.append(table.pop())

    def places(self, table, start, end):
        return [table[i // self.block] for i in range(start, end)], [i % self.block for i in range(start, end)]


def prefill(model, pool, table, tokens, start=0, prefix=None):
    """Append a prompt (behind ``prefix``, if given: pages and length) as one chunk of queries."""
    n = len(tokens)
    pool.grow(table, n)
    before = prefix or ops.PrefixGroup([], 0, [])
    plan = ops.SharedPrefixPlan([ops.PrefixGroup(before.pages, before.length, [(table, n, n)])], model.kv, model.nq)
    return model.run(tokens, range(start, start + n), *pool.places(table, 0, n),
                     lambda layer, q: ops.shared_prefix_attention(q, model.kv, layer, plan))


def decode_shared(model, pool, prefix_tokens, prompts, steps, first=None):
    """Greedy decoding behind one prefix, from the tokens ``first`` if given;
    returns (tokens, last logits, seconds per step)."""
    shared = []
    prefill(model, pool, shared, prefix_tokens)
    group = ops.PrefixGroup(shared, len(prefix_tokens), [])
    tables, lengths, last = [[] for _ in prompts], [len(p) for p in prompts], []
    for table, p in zip(tables, prompts):
        last.append(prefill(model, pool, table, p, group.length, group)[-1])
    logits = torch.stack(last)
    out = [logits.argmax(-1) if first is None else first]
    torch.cuda.synchronize()
    begin = time.perf_counter()
    for _ in range(steps):
        lengths = [n + 1 for n in lengths]
        for table, n in zip(tables, lengths):
            pool.grow(table, n)
        plan = ops.SharedPrefixPlan([group._replace(requests=[(t, n, 1) for t, n in zip(tables, lengths)])], model.kv,
                                    model.nq)
        at = [pool.places(t, n - 1, n) for t, n in zip(tables, lengths)]
        logits = model.run(out[-1], [group.length + n - 1 for n in lengths], [p[0] for p, _ in at],
                           [s[0] for _, s in at], lambda layer, q: ops.shared_prefix_attention(q, model.kv, layer, plan))
        out.append(logits.argmax(-1))
    torch.cuda.synchronize()
    return torch.stack(out, 1), logits, (time.perf_counter() - begin) / max(steps, 1)


def decode_capped(model, pool, prompts, steps, cap, slack, sinks=4, recent=64, first=None):
    """Greedy decoding with at most ``cap`` cached tokens after each eviction,
    from the tokens ``first`` if given.  A prompt's weights start at zero: the
    first eviction ranks by what the steps before it added."""
    tables, newest, last = [[] for _ in prompts], [len(p) - 1 for p in prompts], []
    for table, p in zip(tables, prompts):
        last.append(prefill(model, pool, table, p)[-1])
    lengths = [len(p) for p in prompts]
    logits = torch.stack(last)
    out = [logits.argmax(-1) if first is None else first]
    torch.cuda.synchronize()
    begin, evictions = time.perf_counter(), 0
    for _ in range(steps):
        lengths, newest = [n + 1 for n in lengths], [n + 1 for n in newest]
        for table, n in zip(tables, lengths):
            pool.grow(table, n)
        plan = ops.DecodePlan(tables, lengths, model.kv, model.nq, newest)
        at = [pool.places(t, n - 1, n) for t, n in zip(tables, lengths)]
        logits = model.run(out[-1], newest, [p[0] for p, _ in at], [s[0] for _, s in at],
                           lambda layer, q: ops.weighted_decode_attention(q, model.kv, layer, plan,
                                                                          model.weights[layer]))
        out.append(logits.argmax(-1))
        if max(lengths) >= cap + slack:
            for layer in range(model.layers):
                moves, counts = ops.select_evictions(model.weights[layer], model.positions[layer], plan, cap, sinks,
                                                     min(recent, cap - sinks))
                ops.compact_cache(model.kv, layer, plan, moves, counts, model.weights[layer], model.positions[layer])
            lengths = [min(n, cap) for n in lengths]
            for table, n in zip(tables, lengths):
                pool.shrink(table, n)
            evictions += 1
    torch.cuda.synchronize()
    return torch.stack(out, 1), logits, (time.perf_counter() - begin) / max(steps, 1), evictions


def random_prompts(n, lo, hi, vocab, seed):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, vocab, (lo + int(torch.randint(0, hi - lo + 1, (1,), generator=g)),), generator=g).cuda()
            for _ in range(n)]


# Two ways to compute an attention output in bf16 differ by roundings of the
# inputs' products, of queries and keys, of probabilities and of outputs, in
# each of two layers: some eight of 2^-9.
CHECK_BOUND = 2.0 ** -6


def check(seed=0):
    """Relative differences of attention outputs, shared prefix against whole
    caches: the largest of any layer and request, of the last prompt token and
    of a step on the same tokens."""
    model, pool = Decoder(600, layers=2, seed=seed), Pages(600, 16)
    prefix = random_prompts(1, 333, 333, 4096, seed)[0]
    prompts = random_prompts(5, 3, 40, 4096, seed + 1)
    whole = [torch.cat([prefix, p]) for p in prompts]
    first = random_prompts(1, 5, 5, 4096, seed + 2)[0]

    def attended(decode, rows):
        decode()
        return torch.stack([x[rows].float() for x in model.attended])     # [layers, rows, q heads * hd]

    def difference(a, b):
        return ((a - b).norm(dim=-1) / b.norm(dim=-1)).max().item()

    last = slice(-1, None)
    prompt = max(difference(attended(lambda: decode_shared(model, pool, prefix, [p], 0), last),
                            attended(lambda: decode_capped(model, pool, [w], 0, 4096, 1), last))
                 for p, w in zip(prompts, whole))
    step = difference(attended(lambda: decode_shared(model, pool, prefix, prompts, 1, first), slice(None)),
                      attended(lambda: decode_capped(model, pool, whole, 1, 4096, 1, first=first), slice(None)))
    ops.check_error()
    return [prompt, step]


def main():
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("mode", choices=("shared", "capped"))
    ap.add_argument("--requests", type=int, default=64)
    ap.add_argument("--prefix", type=int, default=4096, help="tokens of the shared system prompt")
    ap.add_argument("--prompt", type=int, default=64, help="longest own prompt")
    ap.add_argument("--cap", type=int, default=1024)
    ap.add_argument("--slack", type=int, default=16)
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--check", action="store_true")
    args = ap.parse_args()
    if args.check:
        diffs = check()
        print(json.dumps({"relative_difference": diffs, "bound": CHECK_BOUND}))
        return 0 if max(diffs) < CHECK_BOUND else 1
    block = 16
    tokens = args.prefix + args.requests * (args.prompt + args.steps + block)
    model = Decoder(-(-tokens // block) + args.requests + 1)
    pool = Pages(model.kv.pages_total, block)
    prompts = random_prompts(args.requests, max(1, args.prompt // 2), args.prompt, 4096, 1)
    rec = {"mode": args.mode, "requests": args.requests, "steps": args.steps}
    if args.mode == "shared":
        _, _, s = decode_shared(model, pool, random_prompts(1, args.prefix, args.prefix, 4096, 2)[0], prompts,
                                args.steps)
    else:
        _, _, s, rec["evictions"] = decode_capped(model, pool, prompts, args.steps, args.cap, args.slack)
    ops.check_error()
    rec.update(ms_per_step=round(s * 1e3, 3), pages_used=model.kv.pages_total - len(pool.free),
               pages_of_whole_caches=args.requests * -(-(args.prefix * (args.mode == "shared") + args.prompt
                                                         + args.steps) // block))
    print(json.dumps(rec))
    return 0


if __name__ == "__main__":
    sys.exit(main())
