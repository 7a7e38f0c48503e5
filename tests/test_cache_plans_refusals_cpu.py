"""Batches that the cache operators' plans refuse (no GPU): the refusal comes
before anything is built for the device."""
from types import SimpleNamespace

import pytest

from kunserve_b200.ops import DecodePlan

KV = SimpleNamespace(block_size=16, pages_total=8, num_kv_heads=2)


@pytest.mark.parametrize("tables,lengths", [([[0, 1], [2, 1]], [20, 20]),     # a page of two requests
                                            ([[3, 3]], [17]),                 # twice in one
                                            ([[0, 1], [0, 2], [4]], [32, 32, 1])])
def test_decode_plan_refuses_shared_pages(tables, lengths):
    """Two requests would add to the same weights at once, and an eviction of
    one would move the other's keys."""
    with pytest.raises(ValueError, match="listed 2 times"):
        DecodePlan(tables, lengths, KV, 4)


def test_pages_past_the_tokens_are_not_compared():
    """Only pages that hold tokens count; the plan goes on to ask for the device."""
    with pytest.raises(AttributeError, match="pool"):
        DecodePlan([[0, 7], [1, 7], [0]], [16, 3, 0], KV, 4)
