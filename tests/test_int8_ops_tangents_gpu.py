"""Forward-mode derivatives and the 8-bit operators: results carry none, so
arguments that carry a tangent are refused."""
import pytest
import torch
from torch.autograd import forward_ad

from test_int8_ops_gpu import BF, F32, _linear_inputs, _no_device_error, _randn  # noqa: F401

pytestmark = pytest.mark.gpu


def test_tangents_are_refused():
    from kunserve_b200 import ops
    x, w = _randn(1, 4, 32).bfloat16(), _randn(2, 32).bfloat16()
    q, s, wq, v = _linear_inputs(4, 32, 48)
    weight, bias = ops.Int8Weight(wq, v), torch.zeros(48, device="cuda", dtype=BF)
    plain = ops.int8_linear(q, s, weight, bias=bias)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t, torch.ones_like(t))

        calls = [lambda: ops.quantize_int8(dual(x)), lambda: ops.add_rms_norm_int8(dual(x), w),
                 lambda: ops.add_rms_norm_int8(x, dual(w)), lambda: ops.add_rms_norm_int8(x, w, residual=dual(x)),
                 lambda: ops.add_rms_norm_int8(x, w, residual=x, out=dual(torch.empty_like(x))),
                 lambda: ops.silu_mul_int8(dual(x), x), lambda: ops.silu_mul_int8(x, dual(x)),
                 lambda: ops.dequantize_int8(q, dual(s)),
                 lambda: ops.dequantize_int8(q, s, out=dual(torch.empty(4, 32, device="cuda"))),
                 lambda: ops.int8_linear(q, dual(s), weight), lambda: ops.int8_linear(q, s, weight, bias=dual(bias)),
                 lambda: ops.int8_linear(q, s, weight, out=dual(torch.empty(4, 48, device="cuda"))),
                 lambda: ops.Int8Weight(wq, dual(v))]
        for f in calls:
            with pytest.raises(ValueError, match="tangent"):
                f()
            with torch.no_grad(), pytest.raises(ValueError, match="tangent"):      # (which leaves tangents alone)
                f()
        # without one, inside a level, and detached
        assert torch.equal(ops.int8_linear(q, s, weight, bias=bias), plain)
        assert torch.equal(ops.quantize_int8(dual(x).detach())[0], ops.quantize_int8(x)[0])
        assert ops.Int8Weight.quantize(dual(wq.float())).in_features == 32
