"""How many rows the 8-bit operators take: what their tiles can count."""
import pytest
import torch

from test_int8_ops_gpu import _no_device_error  # noqa: F401

pytestmark = pytest.mark.gpu


def test_rows_beyond_the_count_of_tiles_are_refused():
    from kunserve_b200 import ops
    row = torch.ones(1, 8, device="cuda").bfloat16()
    for n in (2 ** 31 - 511, 2 ** 31 - 1, 2 ** 31, 2 ** 33):
        many = row.expand(n, 8)
        for f in (lambda: ops.quantize_int8(many), lambda: ops.silu_mul_int8(many, many),
                  lambda: ops.add_rms_norm_int8(many, row[0])):
            with pytest.raises(RuntimeError, match="too many rows"):
                f()
