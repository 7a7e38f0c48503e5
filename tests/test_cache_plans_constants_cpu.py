"""The host's plans and the kernels agree on how a plan is laid out."""
import pytest

from kunserve_b200 import ops
from kunserve_b200.ops import plans


@pytest.mark.skipif(not ops.available(), reason="the extension is not built")
def test_plan_constants_are_the_kernels():
    theirs = ops.native().PLAN_CONSTANTS
    assert set(theirs) == {"UNIT_INTS", "ROW_UNIT_ROWS", "TILE_UNIT_ROWS", "STAGE_KEYS", "TILE_KEYS", "CHUNK_KEYS",
                           "NO_LIMIT"}
    for name, value in theirs.items():
        assert getattr(plans, name) == value, name
