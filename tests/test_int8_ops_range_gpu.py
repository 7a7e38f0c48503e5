"""8-bit rows at the ends of fp32's range: every finite row comes back finite,
and what leaves the range is said by the scale."""
import pytest
import torch

from test_int8_ops_gpu import F32, TYPES, U, _no_device_error  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("k", [4, 37, 640, 4096, 40000])
@pytest.mark.parametrize("dtype", list(TYPES))
def test_largest_rows_come_back_finite(k, dtype):
    """127 times the nearest float to max / 127 can leave fp32; the scale is then
    the one below: off by one step, so every value is by two half steps more than
    the integer's half."""
    from kunserve_b200.ops import dequantize_int8, quantize_int8
    t = TYPES[dtype]
    big = torch.finfo(t).max
    x = torch.zeros(3, k, device="cuda", dtype=torch.float64)
    x[0, :4] = torch.tensor([big, -big, big / 2, big / 127], device="cuda", dtype=torch.float64)
    x[1, -1] = -big
    x[2] = big * torch.linspace(-1, 1, k, device="cuda", dtype=torch.float64)
    x = x.to(t)
    q, s = quantize_int8(x)
    v = dequantize_int8(q, s, F32)
    top = x.double().abs().amax(1, keepdim=True)
    assert v.isfinite().all() and (q.int().abs().amax(1) == 127).all()
    # the scale: a step, two U and the second order of both; the product's own rounding
    assert ((s.double() - top[:, 0] / 127).abs() <= 2 * U * (1 + 4 * U) * top[:, 0] / 127).all()
    assert ((v.double() - x.double()).abs() <= top / 127 * (0.5 + 127 * 6 * U)).all()
    if t != F32:
        assert torch.equal(s, top[:, 0].float() / 127)
    assert dequantize_int8(q, s, t).isfinite().all()
