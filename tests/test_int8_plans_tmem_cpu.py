"""TMEM of the 8-bit matrix product: CTAs wait for it without a limit, and
those of a cluster for one another.  Whatever meets on an SM has to fit, and
what waits while it holds some must not be kept from more by others that do."""
import itertools
import random

import pytest
import torch  # noqa: F401  (loads what the extension links)

# clusters of 1 to 8 CTAs that a B200 holds at once, one CTA an SM; and a device of few
B200 = [0, 148, 74, 45, 33, 26, 22, 15, 15]
SMALL = [0, 10, 5, 3, 2, 1, 1, 1, 1]
SM, KEPT, COLUMNS = 233472, 1024, 512      # bytes of an SM, what is kept of them for each CTA; an SM's TMEM

# tokens, channels, K: few k-blocks in wide tiles, clusters of eight in narrow ones
WIDE = [(992, 2560, 768), (3168, 768, 768), (3840, 768, 768), (1056, 2304, 768), (6176, 512, 512), (8400, 384, 128),
        (306, 5120, 5120), (8192, 28672, 4096)]
NARROW = [(8, 1024, 1024), (16, 768, 2048), (32, 512, 1024), (1, 6144, 4096), (48, 640, 1536)]


def _plans(slots):
    native = pytest.importorskip("kunserve_b200._C")
    rng = random.Random(1)
    drawn = [[max(1, min(131071, int(2 ** (rng.random() * b)))) for b in (14, 17, 14)] for _ in range(1500)]
    return [native.int8_plan(*s, el, slots) for s in WIDE + NARROW + drawn for el in (2, 4)]


@pytest.mark.parametrize("slots", [B200, SMALL])
def test_share_of_shared_memory_covers_the_share_of_tmem(slots):
    """Then any number of CTAs of any products that an SM's shared memory holds
    have room in its TMEM."""
    for p in _plans(slots):
        assert (p["smem"] + KEPT) * COLUMNS >= SM * p["tmem_columns"], p
        assert p["smem"] + KEPT <= (SM if p["alone"] else SM // 2)


def _waits(p):
    """For others of its cluster, while it holds TMEM: pairs, and splits that put their parts over the stages."""
    return p["pair"] or (p["splits"] > 1 and not p["apart"])


@pytest.mark.parametrize("slots", [B200, SMALL])
def test_what_waits_has_an_sm_or_half_of_it(slots):
    """Columns are given out on multiples of their number.  Beside a CTA that has
    half of them, on a multiple of half, one more such CTA always finds the other
    half once CTAs that wait for none have ended; beside one that has the SM's to
    itself no other starts."""
    plans = _plans(slots)
    least = min(p["smem"] for p in plans)
    kinds = set()
    for p in filter(_waits, plans):
        kinds.add((bool(p["alone"]), bool(p["pair"])))
        if p["alone"]:
            assert SM - (p["smem"] + KEPT) < least + KEPT
        else:
            assert p["tmem_columns"] == COLUMNS // 2 and p["smem"] + KEPT == SM // 2
    assert {(True, True), (True, False)} <= kinds and least >= 2 * (128 * 128 + 16 * 128)


def test_two_products_on_an_sm():
    native = pytest.importorskip("kunserve_b200._C")
    for a, b in itertools.product(WIDE, NARROW):
        for el in itertools.product((2, 4), (2, 4)):
            p, q = native.int8_plan(*a, el[0], B200), native.int8_plan(*b, el[1], B200)
            # as many of the second as fit beside one of the first
            beside = (SM - p["smem"] - KEPT) // (q["smem"] + KEPT)
            assert p["tmem_columns"] + beside * q["tmem_columns"] <= COLUMNS, (a, b)


def test_shared_memory_holds_what_the_kernel_lays_out():
    """Stages, results or parts beside them, barriers, and the first KB's alignment."""
    for p in _plans(B200):
        stages = p["stages"] * (128 * 128 + p["width"] // (2 if p["pair"] else 1) * 128)
        parts = -(-p["width"] // p["splits"]) * p["splits"] * 512
        side = 4 * 16 * 272 + 8 * p["width"] if p["splits"] == 1 else parts if p["apart"] else 0
        assert p["smem"] >= stages + side + 21 * 8 + 16 + 1024
