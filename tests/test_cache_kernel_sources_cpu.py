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


def test_tile_kernel_leaves_nothing_in_flight():
    """Copies and products end before the CTA does on every path: its roles
    wait for their own, by time alone, ahead of the last barrier."""
    body = _source("attention_prefix.cu")
    body = body[body.index("tile_kernel("):body.index("void launch(")]
    roles, end = body[:body.rindex("__syncthreads();")], body[body.rindex("__syncthreads();"):]
    producers, rest = roles.split("else if (warp == 10)")
    qk, rest = rest.split("else if (warp == 11)")
    pv, softmax = rest.rsplit("else {", 1)
    assert "mbar_wait<true>(&full[" in producers.split("row = row_of(i + 1);")[1]
    for role, i in ((qk, 0), (pv, 1)):
        after = role[role.rindex("umma_f16"):]
        commit, wait = (after.index(f"{call}(&bars->drained[{i}]") for call in ("umma_commit", "mbar_wait<true>"))
        assert commit < wait
        # behind the loop over units: neither a break nor a return skips it
        assert "break;" not in after[commit:] and "return" not in role
    assert "umma_" not in softmax and "tma_load" not in softmax + qk + pv
    assert "tmem_dealloc" in end and "mbar_init(&bars->drained[b], 1)" in body
