"""What an 8-bit operator writes over a tensor that a gradient was recorded
with, the gradient's computation notices."""
import pytest
import torch

from test_int8_ops_gpu import BF, _linear_inputs, _no_device_error, _randn  # noqa: F401

pytestmark = pytest.mark.gpu


def _writers():
    from kunserve_b200 import ops
    q, s, wq, v = _linear_inputs(4, 32, 32)
    x, w = _randn(1, 4, 32).bfloat16(), _randn(2, 32).bfloat16()
    weight = ops.Int8Weight(wq, v)
    return {"norm": lambda out: ops.add_rms_norm_int8(x, w, residual=out, out=out),
            "values": lambda out: ops.dequantize_int8(q, s, out=out),
            "linear": lambda out: ops.int8_linear(q, s, weight, out=out)}


@pytest.mark.parametrize("name", ["norm", "values", "linear"])
def test_an_overwritten_tensor_of_a_recorded_product(name):
    write = _writers()[name]
    saved = _randn(3, 4, 32).bfloat16()
    p = torch.nn.Parameter(_randn(4, 4, 32).bfloat16())
    y = (p * saved).sum()
    was = saved._version
    write(saved)
    assert saved._version > was
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    # a view's writes are its base's
    base = _randn(5, 4, 64).bfloat16()
    y = (p * base[:, :32]).sum()
    write(base[:, 32:])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("name", ["norm", "values", "linear"])
def test_tensors_without_versions(name):
    write = _writers()[name]
    with torch.inference_mode():
        out = torch.zeros(4, 32, device="cuda", dtype=BF)
        write(out)
    write(out)
    assert out.is_inference() and out.isfinite().all()
