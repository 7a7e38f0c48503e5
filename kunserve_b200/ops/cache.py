"""Operators on a paged KV cache for long contexts: attention of batches that
share prefixes, single-token attention that accumulates each key's weight,
and eviction by those weights.

A step makes one plan from the lengths and page lists the scheduler holds, and
calls the operators with it for every layer.  (Making one takes 0.2 ms for one
or two requests, 0.4 to 0.8 ms for 30 to 130, on the host; its copy to the
device waits for what is queued on the current stream.  A captured graph holds
for the lengths of its plan alone, and needs it alive.)  All of them run on the current
CUDA stream of the cache's device and allocate their scratch from it.  They
serve: their results carry no gradient.
"""
import functools
from typing import List, NamedTuple, Optional, Sequence, Tuple

import numpy as np
import torch

from . import plans
from ._native import native


@functools.lru_cache(maxsize=None)
def _sms(device: int) -> int:
    return torch.cuda.get_device_properties(device).multi_processor_count


def PagedKV(pool: torch.Tensor, layout, fusion_size: int = 1):
    """Handle of a paged pool: the flat (or any contiguous) bf16 or fp16 CUDA
    tensor ``pool``, laid out as ``layout`` (``kv.layout.KVLayout``), addressed
    with the page ids of ``fusion_size``; what the pool holds past the
    layout's pages is extend pages.  Per-slot side tensors of one layer
    (weights, positions) have shape [``pages_total``, kv heads, block_size]."""
    if layout.elem_bytes != 2:
        raise ValueError(f"the cache operators take 16-bit elements, the layout has {layout.elem_bytes} bytes")
    if fusion_size < 1 or layout.num_layers % fusion_size:
        raise ValueError(f"{layout.num_layers} layers do not split into {fusion_size} slices")
    return native().PagedKV(pool, layout.num_pages, fusion_size, layout.num_layers // fusion_size, layout.num_layers,
                            layout.block_size, layout.num_kv_heads, layout.head_dim)


class PrefixGroup(NamedTuple):
    """Requests behind one shared prefix of ``length`` tokens in ``pages``.
    Each request is (pages, tokens, queries): its own tokens, stored from the
    first slot of its own pages on, of which the last ``queries`` are asked
    now (they see the whole prefix and the own tokens up to themselves)."""
    pages: Sequence[int]
    length: int
    requests: Sequence[Tuple[Sequence[int], int, int]]


class SharedPrefixPlan:
    """Plan of ``shared_prefix_attention`` for one step: query rows in the
    order of the groups, their requests and their queries."""

    def __init__(self, groups: Sequence[PrefixGroup], kv, num_q_heads: int):
        bs = kv.block_size
        prefix, own, pages, t = [], [], [], 0
        for i, g in enumerate(groups):
            first, at = t, len(pages)
            pages += plans.take_pages(g.pages, g.length, bs, f"prefix {i}")
            for j, (p, n, q) in enumerate(g.requests):
                if q < 0 or q > n:
                    raise ValueError(f"group {i}, request {j}: {q} queries of {n} own tokens")
                own.append(plans.Span(t, q, n, n - q + 1, len(pages)))
                pages += plans.take_pages(p, n, bs, f"group {i}, request {j}")
                t += q
            prefix.append(plans.Span(first, t - first, g.length, plans.NO_LIMIT, at))
        self.tokens, self.num_q_heads = t, int(num_q_heads)
        blob, table = plans.build(prefix + own, plans.page_array(pages, kv.pages_total), t, self.num_q_heads,
                                  kv.num_kv_heads, _sms(kv.pool.device.index), tiles=kv.tiles)
        blob = plans.append_sections(blob, table, chunks=np.zeros(0), requests=np.zeros(0))
        self._native = native().CachePlan(torch.from_numpy(blob), kv, table)


def shared_prefix_attention(q: torch.Tensor, kv, layer: int, plan: SharedPrefixPlan, scale: Optional[float] = None,
                            out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """softmax(scale q K^T) V of queries ``q`` [tokens, q heads, head_dim] over
    their group's prefix and their request's own tokens in ``layer`` of the
    cache, the keys of a prefix read once for all its requests.  Queries that
    see no key give zeros.  ``scale`` (positive) defaults to head_dim ** -0.5.

    Cache slots past a request's tokens may hold anything; the values of a
    request's asked tokens must be finite, since queries of one call that come
    before a token meet its values with weight zero.  Rows with a NaN score or
    one of +inf give NaN; keys of score -inf count for nothing, and rows of no
    other keys give zeros.

    Sums and statistics are fp32.  Keys that 17 or more query rows (queries
    times heads of a KV head's group) see together, as the requests behind one
    prefix do, meet their values with probabilities rounded to the cache's type:
    outputs are then off by 0.0023 (bf16) or 0.0003 (fp16) of their norm, of
    which 0.0017 and 0.0002 are their own rounding; with fewer rows the rounding
    of the output is all.  In fp16 a weight below 2^-36 of its row's largest may
    count as zero."""
    return native().cached_attention(q, kv, layer, plan._native, scale, out, None)


class DecodePlan:
    """Plan of a decode step with one query per request, for
    ``weighted_decode_attention`` and eviction.

    ``tables``: each request's pages; ``lengths``: its cached tokens, the new
    one included; ``newest``: the position of its newest token (default: its
    length less one; more once tokens were evicted).  Weights (fp32) and slot
    positions (int32) of a layer are [``kv.pages_total``, kv heads,
    block_size]: after evictions every KV head holds other tokens in a
    request's slots.  The pages that hold tokens must be the request's own:
    a page listed twice is refused, since both its weights and its slots would
    change under two requests at once."""

    def __init__(self, tables: Sequence[Sequence[int]], lengths: Sequence[int], kv, num_q_heads: int,
                 newest: Optional[Sequence[int]] = None):
        if len(tables) != len(lengths) or (newest is not None and len(newest) != len(lengths)):
            raise ValueError("tables, lengths and newest must have one entry per request")
        spans, pages, chunks, reqs, cols, col, bs = [], [], [], [], [], 0, kv.block_size
        for i, (table, n) in enumerate(zip(tables, lengths)):
            at = len(pages)
            pages += plans.take_pages(table, n, bs, f"request {i}")
            spans.append(plans.Span(i, 1, n, n, at))
            last = n - 1 if newest is None else int(newest[i])
            reqs.append((n, at, last, 0))
            cols.append(col)
            chunks += [(i, k, min(n, k + plans.CHUNK_KEYS), at, n, col) for k in range(0, n, plans.CHUNK_KEYS)]
            col += -(-n // plans.STAGE_KEYS) * plans.STAGE_KEYS
        if reqs and not -2 ** 31 <= min(r[2] for r in reqs) <= max(r[2] for r in reqs) < 2 ** 31:
            raise ValueError("newest positions must fit 32 bits")
        page_ids = plans.page_array(pages, kv.pages_total)
        plans.check_distinct(page_ids)
        self.lengths: List[int] = list(lengths)
        self.longest = max(self.lengths, default=0)
        self.num_q_heads = int(num_q_heads)
        blob, table = plans.build(spans, page_ids, len(spans), self.num_q_heads, kv.num_kv_heads,
                                  _sms(kv.pool.device.index), score_cols=cols)
        blob = plans.append_sections(blob, table, chunks=np.array(chunks), requests=np.array(reqs))
        table.update(chunks=len(chunks), requests=len(reqs), most_tokens=self.longest, score_cols=col)
        self._native = native().CachePlan(torch.from_numpy(blob), kv, table)
        self._kv = kv


def weighted_decode_attention(q: torch.Tensor, kv, layer: int, plan: DecodePlan, weights: torch.Tensor,
                              scale: Optional[float] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query per request, ``q`` [requests, q heads, head_dim],
    over its cached tokens; ``weights`` gains, at each token's slot and KV
    head, the softmax weight that the head's query group gave it (summed over
    the group, fp32; one writer a slot, so that a repeat gives the same bits).
    Requests without tokens, and rows whose scores are all -inf, give zeros and
    add no weight.  ``scale`` (positive) defaults to head_dim ** -0.5."""
    return native().cached_attention(q, kv, layer, plan._native, scale, out, weights)


def select_evictions(weights: torch.Tensor, slot_positions: torch.Tensor, plan: DecodePlan, keep: int, sinks: int = 0,
                     recent: int = 0) -> Tuple[torch.Tensor, torch.Tensor]:
    """What each (request, KV head) keeps of more than ``keep`` tokens, as the
    moves that bring the kept ones to slots below ``keep``.

    Kept are first the tokens at positions below ``sinks`` and the ``recent``
    newest positions (above ``newest - recent``), then the largest weights;
    among equals the lowest slot, NaN last.  Returns ``moves`` int32
    [requests, kv heads, most, 2] of (to, from) slots in slot order, -1 past
    the ``counts`` int32 [requests, kv heads].  Nothing is changed:
    ``compact_cache`` applies the moves, after which a request holds
    ``min(keep, length)`` tokens."""
    most = max(0, min(keep, plan.longest - keep))      # moves of the longest request, at most
    return native().select_evictions(weights, slot_positions, plan._kv, plan._native, keep, sinks, recent, most)


def compact_cache(kv, layer: int, plan: DecodePlan, moves: torch.Tensor, counts: torch.Tensor,
                  weights: Optional[torch.Tensor] = None, slot_positions: Optional[torch.Tensor] = None) -> None:
    """Move keys and values of ``layer``, and the weights and slot positions
    given, as ``select_evictions`` says; the pages past the kept tokens are
    then free."""
    native().compact_cache(kv, layer, plan._native, moves, counts, weights, slot_positions)
