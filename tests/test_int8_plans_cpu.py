"""How the 8-bit matrix product is cut: every channel and token tile once,
every part of K by one CTA of a cluster."""
import random

import pytest
import torch  # noqa: F401  (loads what the extension links)

# clusters of 1 to 8 CTAs that a B200 holds at once, one CTA an SM; and a device of few
B200 = [0, 148, 74, 45, 33, 26, 22, 15, 15]
SMALL = [0, 10, 5, 3, 2, 1, 1, 1, 1]
SHARED = {True: 232448, False: 115712}      # bytes a CTA may have, alone on its SM or one of two


def _units(p):
    """(channel tile, token tile) of each unit, as the kernel counts them."""
    for u in range(p["channel_tiles"] * p["token_tiles"]):
        g, r = divmod(u, p["group"] * p["channel_tiles"])
        wide = min(p["group"], p["token_tiles"] - g * p["group"])
        yield r // wide, g * p["group"] + r % wide


@pytest.mark.parametrize("slots", [B200, SMALL])
@pytest.mark.parametrize("seed", range(6))
def test_every_tile_once(seed, slots):
    native = pytest.importorskip("kunserve_b200._C")
    rng = random.Random(seed)
    for _ in range(150):
        m, n, k = (max(1, min(131071, int(2 ** (rng.random() * b)))) for b in (14, 17, 17))
        element = rng.choice([2, 4])
        p = native.int8_plan(m, n, k, element, slots)
        ctas = 2 if p["pair"] else 1
        assert p["width"] % (16 * ctas) == 0 and 16 * ctas <= p["width"] <= 256
        assert (p["token_tiles"] - 1) * p["width"] < m <= p["token_tiles"] * p["width"]
        assert (p["channel_tiles"] - 1) * 128 * ctas < n <= p["channel_tiles"] * 128 * ctas
        blocks = -(-k // 128)
        each = -(-blocks // p["splits"])
        assert 1 <= p["splits"] <= 8 // ctas and (p["splits"] - 1) * each < blocks <= p["splits"] * each
        units = p["channel_tiles"] * p["token_tiles"]
        assert p["grid"] % (ctas * p["splits"]) == 0
        if p["splits"] > 1:
            assert p["grid"] == ctas * units * p["splits"]
        else:
            assert 0 < p["grid"] <= ctas * units
        # shared memory: stages and barriers; of whole units two buffers for each epilogue group and two tiles' scales,
        # of split ones the parts of a share of the tokens, beside the stages or over them.  TMEM: two accumulators, of
        # each of two CTAs an SM
        stage = 128 * 128 + p["width"] // ctas * 128
        parts = -(-p["width"] // p["splits"]) * p["splits"] * 512
        assert 2 <= p["stages"] <= 8 and (p["splits"] > 1 or not p["apart"])
        if p["splits"] == 1:
            side = 4 * 16 * (128 * element + (16 if element == 2 else 0)) + 8 * p["width"]
        else:
            side = parts if p["apart"] else 0
            assert p["apart"] or parts <= p["stages"] * stage
        used = p["stages"] * stage + side + 21 * 8 + 16 + 1024
        assert used <= SHARED[bool(p["alone"])]
        # however many such CTAs an SM has room for, of one product or of several: their TMEM fits
        assert 233472 // (used + 1024) * p["tmem_columns"] <= 512
        assert 2 * p["width"] <= p["tmem_columns"] <= (512 if p["alone"] else 256)
        if units < 20000:
            seen = set(_units(p))
            assert len(seen) == units
            assert all(0 <= a < p["channel_tiles"] and 0 <= t < p["token_tiles"] for a, t in seen)
