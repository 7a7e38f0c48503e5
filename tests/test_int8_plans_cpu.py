"""How the 8-bit matrix product is cut: every channel and token tile once,
every part of K by one CTA of a cluster."""
import random

import pytest
import torch  # noqa: F401  (loads what the extension links)

SMS = 148


def _units(p):
    """(channel tile, token tile) of each unit, as the kernel counts them."""
    for u in range(p["channel_tiles"] * p["token_tiles"]):
        g, r = divmod(u, p["group"] * p["channel_tiles"])
        wide = min(p["group"], p["token_tiles"] - g * p["group"])
        yield r // wide, g * p["group"] + r % wide


@pytest.mark.parametrize("seed", range(8))
def test_every_tile_once(seed):
    native = pytest.importorskip("kunserve_b200._C")
    rng = random.Random(seed)
    for _ in range(150):
        m, n, k = (int(2 ** (rng.random() * b)) for b in (14, 17, 17))
        p = native.int8_plan(m, n, min(k, 131071), SMS)
        assert p["width"] % 16 == 0 and 16 <= p["width"] <= 256
        assert (p["token_tiles"] - 1) * p["width"] < m <= p["token_tiles"] * p["width"]
        assert (p["channel_tiles"] - 1) * 128 < n <= p["channel_tiles"] * 128
        blocks = -(-min(k, 131071) // 128)
        each = -(-blocks // p["splits"])
        assert 1 <= p["splits"] <= 8 and (p["splits"] - 1) * each < blocks <= p["splits"] * each
        units = p["channel_tiles"] * p["token_tiles"]
        if p["splits"] > 1:
            assert p["grid"] == units * p["splits"]
        else:
            assert 0 < p["grid"] <= units
        if units < 20000:
            seen = set(_units(p))
            assert len(seen) == units
            assert all(0 <= a < p["channel_tiles"] and 0 <= t < p["token_tiles"] for a, t in seen)
