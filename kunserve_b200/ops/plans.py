"""Work units of the cached-attention kernels for one batch (host side).

A plan is made once per step and serves every layer.  It cuts each set of
query rows (the tokens behind a shared prefix, or one request's tokens) into
row tiles, and the keys they see into ranges, so that the units spread over
the GPU whatever the mix of lengths; and it lists for every (token, head)
which partial rows to join.  ``csrc/kernels/cache_ops.h`` describes the
records; everything the kernels index with is checked here.  The constants up
to ``NO_LIMIT`` are the kernels' (``PLAN_CONSTANTS`` of the extension).
"""
from typing import Dict, List, NamedTuple, Sequence, Tuple

import numpy as np

UNIT_INTS = 8
ROW_UNIT_ROWS = 16
STAGE_KEYS = 32          # keys per stage of the row kernel
TILE_UNIT_ROWS = 128
TILE_KEYS = 128          # keys per block of the tile kernel
CHUNK_KEYS = 512         # keys per block that adds up weights
NO_LIMIT = 1 << 30       # limit of keys that every query sees
# Fewest query rows (tokens x group heads) of a span that the tile kernel takes.
# Prefixes: at 16 rows both take the same (40 heads, 2048 keys: 20.7 us), at 24
# the tile kernel 53 us, row tiles 90 (8 heads, four prefixes of 16384).  Own
# spans of 96 rows (24 requests, 8 heads, us, tile / row kernel): 2048 keys 63 /
# 165, 512 keys 31 / 54, 128 keys 25 / 25, 40 keys 25 / 19; of 20 to 24 rows the
# two meet at 512 keys and the row kernel takes half as long at 40.
TILE_MIN_ROWS = 17
ROW_SLOTS = 6            # warps of the row kernel an SM takes at once
ROW_MIN_STAGES = 2       # shortest range of a row unit, in stages
ROW_START = 1            # what starting and ending a unit takes, in stages
TILE_SLOTS = 1           # CTAs of the tile kernel an SM holds
TILE_MIN_BLOCKS = 2      # shortest range of a tile unit, in blocks
TILE_START = 2           # what starting and ending a unit takes, in blocks


class Span(NamedTuple):
    """Query rows of consecutive tokens over one page list: ``limit`` keys are
    visible to the first token and one more to each further one, never more
    than ``keys``."""
    token: int
    tokens: int
    keys: int
    limit: int
    page: int            # first entry of the page list


def _row_tiles(spans: Sequence[Span], group: int, rows: int) -> np.ndarray:
    """Tiles of at most ``rows`` rows: columns token, tokens, heads, first
    head, visible keys, limit, page list, span."""
    out: List[Tuple[int, ...]] = []
    step = max(1, rows // group)
    for i, s in enumerate(spans):
        for j in range(0, s.tokens, step):
            n = min(step, s.tokens - j)
            keys = min(s.keys, s.limit + j + n - 1)
            if keys <= 0:
                continue
            for g in range(0, group, rows):
                out.append((s.token + j, n, min(rows, group - g), g, keys, min(s.limit + j, NO_LIMIT), s.page, i))
    return np.array(out, dtype=np.int64).reshape(-1, 8)


def _parts(stages: np.ndarray, share: np.ndarray) -> np.ndarray:
    """Equal ranges of at most ``share`` stages per tile (of one stage at least)."""
    parts = -(-stages // share)
    return -(-stages // -(-stages // parts))         # no empty range at the end


def _cut(tiles: np.ndarray, kv_heads: int, slots: int, stage: int, least: int, start: float) -> np.ndarray:
    """Cut the tiles' keys into equal ranges: columns of the tile, then first
    key and end of the range.

    Of a few dozen range lengths the one that takes least is used, in stages:
    units that all start at once take as long as the longest; more of them
    take a slot's share of all, and the longest once more at the end.  A unit
    costs ``start`` stages and an eighth of one per row (its partial sums)
    besides its keys; each part of a row costs the join 1/32."""
    if not len(tiles):
        return np.zeros((0, 10), dtype=np.int64)
    stages = -(-tiles[:, 4] // stage)
    most, total = int(stages.max()), int(stages.sum()) * kv_heads
    extra = start + tiles[:, 1] * tiles[:, 2] / 8.0 * STAGE_KEYS / stage
    tries = {-(-most // k) for k in range(1, 49)} | {-(-total * k // (slots * 8)) for k in range(1, 17)}
    parts = _parts(stages, np.array(sorted({max(least, t) for t in tries}))[:, None])   # [tries, tiles]
    each = -(-stages // parts) + extra
    units = parts.sum(axis=1) * kv_heads
    cost = each.max(axis=1) + parts.max(axis=1) / 32.0 + np.where(
        units > slots, (each * parts).sum(axis=1) * kv_heads / slots, 0.0)
    parts = parts[int(cost.argmin())]
    each = -(-stages // parts)
    idx = np.repeat(np.arange(len(tiles)), parts)
    k = np.arange(len(idx)) - np.repeat(np.cumsum(parts) - parts, parts)
    lo = k * each[idx] * stage
    hi = np.minimum(lo + each[idx] * stage, tiles[idx, 4])
    cut = np.concatenate([tiles[idx], lo[:, None], hi[:, None]], axis=1)
    return cut[np.argsort(lo - hi, kind="stable")]   # the longest start first


def build(spans: Sequence[Span], pages: np.ndarray, tokens: int, num_q_heads: int, kv_heads: int, sms: int,
          tiles: bool = False, score_cols: Sequence[int] = ()) -> Tuple[np.ndarray, Dict[str, int]]:
    """The int32 blob of a plan and its section table.  ``tiles``: spans of
    many rows go to the tile kernel.  ``score_cols``: first score column of
    each span (weighted plans, row kernel only)."""
    if num_q_heads % kv_heads:
        raise ValueError(f"{num_q_heads} query heads are no multiple of {kv_heads} KV heads")
    group = num_q_heads // kv_heads
    if group > 128:
        raise ValueError(f"at most 128 query heads per KV head, got {group}")
    many = [tiles and s.tokens * group >= TILE_MIN_ROWS for s in spans]
    rows = _cut(_row_tiles([s for s, m in zip(spans, many) if not m], group, ROW_UNIT_ROWS), kv_heads,
                sms * ROW_SLOTS, STAGE_KEYS, ROW_MIN_STAGES, ROW_START)
    wide = _cut(_row_tiles([s for s, m in zip(spans, many) if m], group, TILE_UNIT_ROWS), kv_heads, sms * TILE_SLOTS,
                TILE_KEYS, TILE_MIN_BLOCKS, TILE_START)
    head_chunks = -(-group // ROW_UNIT_ROWS)

    units = np.concatenate([rows, wide])
    n_rows = units[:, 1] * units[:, 2]
    part = np.cumsum(n_rows * kv_heads) - n_rows * kv_heads
    rec = np.zeros((len(units), UNIT_INTS), dtype=np.int64)
    rec[:, 0] = units[:, 0]
    rec[:, 1] = units[:, 1] | units[:, 2] << 8 | units[:, 3] << 16
    rec[:, 2:4] = units[:, 8:10]
    rec[:, 4] = units[:, 5]
    rec[:, 5] = units[:, 6]
    rec[:, 6] = part
    if len(score_cols):
        rec[:, 7] = np.asarray(score_cols, dtype=np.int64)[units[:, 7]]
    part_rows = int((n_rows * kv_heads).sum())

    # the partial rows of each (token, chunk of 16 group heads); a tile unit has all chunks of its tokens
    chunks = np.where(np.arange(len(units)) < len(rows), 1, head_chunks)
    per = units[:, 1] * chunks
    idx = np.repeat(np.arange(len(units)), per)
    k = np.arange(len(idx)) - np.repeat(np.cumsum(per) - per, per)
    j = k // chunks[idx]
    key = (units[idx, 0] + j) * head_chunks + units[idx, 3] // ROW_UNIT_ROWS + k % chunks[idx]
    order = np.argsort(key, kind="stable")
    entries = np.stack([part[idx] + j * units[idx, 2] - units[idx, 3], n_rows[idx]], axis=1)[order]
    counts = np.bincount(key, minlength=tokens * head_chunks)
    off = np.concatenate([[0], np.cumsum(counts)])
    if part_rows >= 1 << 31:
        raise ValueError("the batch needs too many partial rows")

    table = dict(tokens=tokens, num_q_heads=num_q_heads, row_units=len(rows), tile_units=len(wide), head_chunks=head_chunks,
                 most_parts=int(counts.max()) if counts.size else 0, part_rows=part_rows,
                 max_page=int(pages.max()) if pages.size else -1, chunks=0, requests=0, most_tokens=0, score_cols=0)
    return _pack(table, row_units=rec[:len(rows)], tile_units=rec[len(rows):], merge=entries, merge_off=off, pages=pages)


def _pack(table: Dict[str, int], **sections: np.ndarray) -> Tuple[np.ndarray, Dict[str, int]]:
    """Lay the sections out on 16-byte boundaries; ``table`` gains ``at_<name>``."""
    at, chunks = 0, []
    for name, a in sections.items():
        a = np.ascontiguousarray(a, dtype=np.int32).reshape(-1)
        table["at_" + name] = at
        chunks += [a, np.zeros(-a.size % 4, dtype=np.int32)]
        at += a.size + (-a.size % 4)
    return np.concatenate(chunks) if chunks else np.zeros(0, np.int32), table


def append_sections(blob: np.ndarray, table: Dict[str, int], **sections: np.ndarray) -> np.ndarray:
    """More sections behind those of ``blob``."""
    more, t = _pack({}, **sections)
    table.update({k: v + blob.size for k, v in t.items()})
    return np.concatenate([blob, more])


def take_pages(pages: Sequence[int], tokens: int, block_size: int, what: str) -> List[int]:
    """The pages that hold ``tokens`` tokens, first of a page list."""
    if not 0 <= tokens < NO_LIMIT:
        raise ValueError(f"{what}: {tokens} tokens")
    need = -(-tokens // block_size)
    pages = list(pages[:need])
    if len(pages) < need:
        raise ValueError(f"{what}: {tokens} tokens need {need} pages of {block_size}, got {len(pages)}")
    return pages


def page_array(pages: Sequence[int], pages_total: int) -> np.ndarray:
    """All page lists of a plan, every id checked against the cache."""
    a = np.array(pages, dtype=np.int64)
    if a.size and not (0 <= int(a.min()) and int(a.max()) < pages_total):
        raise ValueError(f"page ids must lie in [0, {pages_total}), got {int(a.min())} to {int(a.max())}")
    return a


def check_distinct(pages: np.ndarray) -> None:
    """Every page of the plan's lists is listed once."""
    seen = np.zeros(int(pages.max()) + 1 if pages.size else 0, dtype=bool)
    seen[pages] = True
    if np.count_nonzero(seen) < pages.size:
        times = np.bincount(pages)
        raise ValueError(f"page {int(times.argmax())} is listed {int(times.max())} times; slots that gain weight and "
                         "move must belong to one request")
