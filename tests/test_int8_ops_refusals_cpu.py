"""What the 8-bit operators refuse before anything touches a GPU, and rules that
their kernels keep and no run can show: read from their sources."""
import os
import re

import pytest
import torch

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kunserve_b200", "csrc", "kernels")


def test_tensors_of_the_host_are_refused():
    pytest.importorskip("kunserve_b200._C")
    from kunserve_b200 import ops
    x, w = torch.ones(2, 16).bfloat16(), torch.ones(16).bfloat16()
    q, s = torch.ones(2, 16, dtype=torch.int8), torch.ones(2)
    for f in (lambda: ops.quantize_int8(x), lambda: ops.add_rms_norm_int8(x, w), lambda: ops.silu_mul_int8(x, x),
              lambda: ops.dequantize_int8(q, s), lambda: ops.Int8Weight(q, s), lambda: ops.Int8Weight.quantize(x)):
        with pytest.raises(RuntimeError, match="must be a CUDA tensor"):
            f()


def _source(name):
    with open(os.path.join(KERNELS, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


@pytest.mark.parametrize("name", ["int8_rows.cu", "int8_gemm.cu"])
def test_nothing_is_read_as_constant_memory(name):
    """A grid starts while the one before it still writes."""
    text = _source(name)
    assert "__ldg" not in text and "ld.global.nc" not in text and "__restrict__" not in text


def _gemm_kernel():
    text = _source("int8_gemm.cu")
    return text[text.index("gemm_kernel(const __grid_constant__"):text.index("pack_kernel(")]


def test_weights_alone_are_loaded_ahead_of_the_wait():
    kernel = _gemm_kernel()
    setup, roles = kernel[:kernel.index("if (warp != 0)")], kernel[kernel.index("if (warp != 0)"):]
    # ahead of the roles only the weights' loads are issued, and by one thread
    assert setup.count("tma_load_2d(") == setup.count("tma_load_2d_pair(") == 1 and "&tmX" not in setup
    producer = roles[roles.index("if (warp == 0)"):roles.index("else if (warp == 1)")]
    ahead = producer[producer.index("prefetch_tmap"):producer.index("pdl_wait();")]
    assert "load_w(j" in ahead and "load_x(" not in ahead
    # every other role waits before it does anything
    assert re.match(r"if \(warp != 0\) \{\s*pdl_wait\(\);", roles)
    # and what writes weights lets nothing start before it has ended
    text = _source("int8_gemm.cu")
    pack = text[text.index("pack_kernel("):]
    pack = pack[:pack.index("align_kernel(")]
    assert "pdl_wait();" in pack and "pdl_trigger" not in pack
    launch = text[text.index("void int8_pack("):]
    assert "pack_kernel<<<" in launch[:launch.index("Int8Slots")]


def test_nothing_is_in_flight_at_the_end():
    """Copies and products end before their CTA on every path, and what a
    cluster's CTAs write to one another before they meet for the last time."""
    kernel = _gemm_kernel()
    producer, rest = kernel.split("else if (warp == 1)")
    assert "mbar_wait<true>(&full[" in producer[producer.rindex("load_x("):]
    issuer = rest[:rest.index("const int quarter")]
    after = issuer[issuer.rindex("umma_i8<PAIR>"):]
    assert after.index("commit<PAIR>(drained") < after.index("mbar_wait<true>(drained")
    assert after.count("mbar_wait<true>(drained") == 2      # of a pair's other CTA too
    shared = kernel[kernel.index("uint8_t* parts"):]
    # over the stages only once all have used them up; nothing is written to others past the last meeting
    assert re.search(r"if \(!PAIR\) cluster_wait\(\);\s*if \(!p.apart\) cluster_sync\(\);\s*if \(summed\)", shared)
    assert "st_cluster(" not in shared[shared.rindex("cluster_sync();"):]
    setup = kernel[:kernel.index("if (warp != 0)")]
    assert re.search(r"if \(PAIR\)\s*cluster_sync\(\);\s*else if \(SPLIT\)\s*cluster_arrive\(\);", setup)
