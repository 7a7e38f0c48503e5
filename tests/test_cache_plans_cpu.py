"""Host side of the long-context cache operators (no GPU): work units of the
cached-attention kernels, page checks, rotary frequencies."""
import math

import numpy as np
import pytest
import torch

from kunserve_b200.ops import plans
from kunserve_b200.ops.rotary import Rotary, rotary_frequencies


def _units(blob, table, name):
    n, at = table[name], table["at_" + name]
    return blob[at:at + n * plans.UNIT_INTS].reshape(n, plans.UNIT_INTS)


def _check(spans, nq, nkv, sms=148, tiles=False):
    """Every (token, head) row meets each key it sees exactly once, and finds
    all of its partial rows in its list."""
    pages = np.arange(10)
    tokens = max((s.token + s.tokens for s in spans), default=0)
    blob, table = plans.build(spans, pages, tokens, nq, nkv, sms, tiles)
    G = nq // nkv
    want, got, parts = {}, {}, {}
    for s in spans:
        for j in range(s.tokens):
            for g in range(G):
                n = min(s.keys, s.limit + j)
                if n > 0:
                    want[(s.token + j, g, s.page)] = n
    used = set()
    for name, most in (("row_units", plans.ROW_UNIT_ROWS), ("tile_units", 128)):
        for u in _units(blob, table, name).tolist():
            tok, packed, lo, hi, lim, page, part, _ = u
            nt, ng, g0 = packed & 255, packed >> 8 & 255, packed >> 16
            assert 0 < nt * ng <= most and lo < hi and g0 + ng <= G
            rows = set(range(part, part + nt * ng * nkv))
            assert not rows & used
            used |= rows
            for j in range(nt):
                for g in range(g0, g0 + ng):
                    k = got.setdefault((tok + j, g, page), [])
                    k += range(lo, min(hi, lim + j))
                    parts.setdefault((tok + j, g), set()).add((part + j * ng + g - g0, nt * ng))
    for row, n in want.items():
        assert sorted(got.get(row, [])) == list(range(n)), row
    assert all(not v for k, v in got.items() if k not in want)
    assert len(used) == table["part_rows"] and used == set(range(table["part_rows"]))
    off = blob[table["at_merge_off"]:][:tokens * table["head_chunks"] + 1]
    merge = blob[table["at_merge"]:][:2 * off[-1]].reshape(-1, 2)
    for t in range(tokens):
        for g in range(G):
            i = t * table["head_chunks"] + g // plans.ROW_UNIT_ROWS
            rows = {(int(a) + g, int(b)) for a, b in merge[off[i]:off[i + 1]]}
            assert len(rows) == off[i + 1] - off[i] <= table["most_parts"]
            assert rows == parts.get((t, g), set())
    assert all(table["at_" + s] % 4 == 0 for s in ("row_units", "tile_units", "merge", "merge_off", "pages"))
    return table


@pytest.mark.parametrize("nq,nkv", [(4, 4), (6, 2), (8, 1), (20, 1), (40, 1), (128, 1), (14, 2)])
@pytest.mark.parametrize("tiles", [False, True])
def test_units_cover_every_key_once(nq, nkv, tiles):
    S = plans.Span
    _check([S(0, 5, 300, plans.NO_LIMIT, 0), S(0, 2, 33, 32, 1), S(2, 3, 3, 1, 2), S(5, 1, 0, 0, 3), S(6, 1, 7, 7, 4)],
           nq, nkv, tiles=tiles)
    _check([S(0, 70, 400, plans.NO_LIMIT, 0), S(0, 70, 90, 21, 1)], nq, nkv, tiles=tiles)
    _check([], nq, nkv, tiles=tiles)
    _check([S(0, 3, 0, plans.NO_LIMIT, 0)], nq, nkv, tiles=tiles)


@pytest.mark.parametrize("seed", range(4))
def test_random_batches(seed):
    rng = np.random.default_rng(seed)
    spans, t = [], 0
    for i in range(int(rng.integers(1, 5))):
        first = t
        own = []
        for _ in range(int(rng.integers(1, 12))):
            q = int(rng.integers(0, 6))
            n = q + int(rng.integers(0, 400))
            own.append(plans.Span(t, q, n, n - q + 1, 100 * i + len(own)))
            t += q
        spans += [plans.Span(first, t - first, int(rng.integers(0, 2000)), plans.NO_LIMIT, 100 * i + 99)] + own
    _check(spans, 8, 2, tiles=seed % 2 == 0)


def test_long_contexts_spread_over_the_gpu():
    """One long context among short ones is cut into about a unit for every
    warp the GPU holds."""
    S = plans.Span
    spans = [S(0, 1, 60000, 60000, 0)] + [S(i, 1, 50, 50, i) for i in range(1, 9)]
    table = _check(spans, 8, 8)
    units = table["row_units"] * 8
    assert 0.6 * 148 * plans.ROW_SLOTS <= units <= 148 * plans.ROW_SLOTS


def test_page_checks():
    assert plans.take_pages([3, 4, 5], 17, 16, "x") == [3, 4]
    assert plans.take_pages([], 0, 16, "x") == []
    for pages, n in (([3], 17), ([0], -1), ([0], 1 << 31)):
        with pytest.raises(ValueError):
            plans.take_pages(pages, n, 16, "x")
    assert plans.page_array([0, 5, 5], 6).tolist() == [0, 5, 5] and plans.page_array([], 6).size == 0
    for pages in ([6], [-1], [0, 7, 2]):
        with pytest.raises(ValueError):
            plans.page_array(pages, 6)
    with pytest.raises(ValueError):
        plans.build([], np.zeros(0), 0, 5, 2, 148)
    with pytest.raises(ValueError):
        plans.build([], np.zeros(0), 0, 129, 1, 148)


# --------------------------------------------------------- rotary frequencies
def test_plain_and_linear_frequencies():
    f, m = rotary_frequencies(8, 10000.0)
    assert m == 1.0 and torch.allclose(f, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14)
    g, _ = rotary_frequencies(8, 10000.0, {"type": "linear", "factor": 4.0})
    assert torch.equal(g * 4, f)


def test_llama3_frequencies():
    s = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
         "original_max_position_embeddings": 8192}
    f, _ = rotary_frequencies(128, 500000.0)
    g, m = rotary_frequencies(128, 500000.0, s)
    wave = 2 * math.pi / f
    assert m == 1.0
    assert torch.allclose(g[wave < 8192 / 4], f[wave < 8192 / 4], rtol=1e-14)
    assert torch.allclose(g[wave > 8192], f[wave > 8192] / 8, rtol=1e-14)
    mid = (wave >= 8192 / 4) & (wave <= 8192)
    smooth = (8192 / wave[mid] - 1.0) / 3.0
    assert mid.any() and torch.allclose(g[mid], (1 - smooth) * f[mid] / 8 + smooth * f[mid], rtol=1e-12)


def test_yarn_and_dynamic_frequencies():
    s = {"rope_type": "yarn", "factor": 16.0, "original_max_position_embeddings": 4096}
    f, _ = rotary_frequencies(64, 10000.0)
    g, m = rotary_frequencies(64, 10000.0, s)
    assert m == pytest.approx(0.1 * math.log(16.0) + 1.0)
    turns = 4096 * f / (2 * math.pi)
    assert torch.allclose(g[turns > 40], f[turns > 40]) and torch.allclose(g[turns < 0.8], f[turns < 0.8] / 16)
    assert (g[1:] < g[:-1]).all()
    assert rotary_frequencies(64, 10000.0, dict(s, attention_factor=1.5))[1] == 1.5
    d = {"rope_type": "dynamic", "factor": 2.0, "original_max_position_embeddings": 4096}
    assert torch.equal(rotary_frequencies(64, 10000.0, d, max_position=4096)[0], f)
    h, _ = rotary_frequencies(64, 10000.0, d, max_position=8192)
    assert torch.allclose(h, (10000.0 * 3.0 ** (64 / 62)) ** (-torch.arange(0, 64, 2, dtype=torch.float64) / 64))


@pytest.mark.parametrize("args", [dict(rotary_dim=7), dict(rotary_dim=0), dict(rotary_dim=8, theta=0.0),
                                  dict(rotary_dim=8, scaling={"rope_type": "other", "factor": 2.0}),
                                  dict(rotary_dim=8, scaling={"rope_type": "linear"}),
                                  dict(rotary_dim=8, scaling={"rope_type": "linear", "factor": 0.5}),
                                  dict(rotary_dim=8, scaling={"rope_type": "linear", "factor": 2.0, "beta_fast": 1}),
                                  dict(rotary_dim=8, scaling={"rope_type": "dynamic", "factor": 2.0,
                                                              "original_max_position_embeddings": 64})])
def test_frequency_refusals(args):
    with pytest.raises(ValueError):
        rotary_frequencies(**args)


def test_rotary_steps_are_turn_fractions():
    r = Rotary(64, rotary_dim=32, theta=10000.0, device="cpu")
    steps = [int(s) % 2 ** 64 for s in r.steps]
    for s, f in zip(steps, r.frequencies.tolist()):
        assert abs(s / 2 ** 64 - f / (2 * math.pi)) <= 2 ** -53
    # the angle of a far position, from the wrapped integer product
    p, i = 1234567, 3
    turn = (p * steps[i]) % 2 ** 64 / 2 ** 64
    want = math.fmod(p * float(r.frequencies[i]) / (2 * math.pi), 1.0)
    assert abs(turn - want) < 1e-9
    with pytest.raises(ValueError):
        Rotary(64, rotary_dim=128, device="cpu")
