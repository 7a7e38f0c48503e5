"""Rules that the cache operators' kernels keep and no run can show: read from
their sources."""
import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kunserve_b200", "csrc", "kernels")
SOURCES = ["rotary.cu", "attention_prefix.cu", "attention_cached.cu", "evict.cu", "cache_elem.cuh"]


def _source(name):
    with open(os.path.join(KERNELS, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


# A plan's sections: the work units and lists that no kernel writes.
PLAN = r"(?:reinterpret_cast<const int4\*>\()?(?:a\.(?:row_units|tile_units|merge_off|merge|reqs|pages)\b|table\b|c\))"


@pytest.mark.parametrize("name", SOURCES)
def test_read_only_loads_are_of_plans(name):
    """A grid starts while the one before it still writes, so what other
    kernels write is not read-only for it: __ldg is for plans."""
    for arg in re.findall(r"__ldg\((.{0,60})", _source(name)):
        assert re.match(PLAN, arg), f"{name}: __ldg({arg}"
    assert "ld.global.nc" not in _source(name) and "__restrict__" not in _source(name)
