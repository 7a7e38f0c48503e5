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
        assert torch.equal(s, (top[:, 0] / 127).float())
    assert dequantize_int8(q, s, t).isfinite().all()


@pytest.mark.parametrize("k", [64, 333, 4096, 40000])
def test_norms_that_leave_the_range_say_so(k):
    """h w is finite, its norm is not: scale NaN and integers 0, as of any row
    that leaves fp32 on the way.  Rows beside it, near the range's end too, keep
    their values."""
    from kunserve_b200.ops import add_rms_norm_int8, dequantize_int8
    w = torch.full((k,), 3e38, device="cuda").bfloat16()
    x = torch.zeros(4, k, device="cuda").bfloat16()
    x[0, 3] = 0.5                      # sqrt(k) times the weight
    x[1] = 0.5                         # the weight itself
    x[2, 3], x[2, 4:] = 1.0, 1e-3      # below sqrt(k) times it, above it for k > 1
    q, s, _ = add_rms_norm_int8(x, w, 1e-5)
    v = dequantize_int8(q, s, F32)
    total = x.double()
    y = total / (total.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    top = y.abs().amax(1)
    assert (top > torch.finfo(F32).max).tolist() == [True, False, True, False]
    assert s.isnan().tolist() == [True, False, True, False] and (q[[0, 2]] == 0).all()
    assert v.isnan().all(1).tolist() == [True, False, True, False]
    # 33 + 12: of the squares' sum and the factors (more where a row is read twice), as for other norms
    u = (10 + 8 * -(-k // 8192) + 32) * U
    assert v[[1, 3]].isfinite().all()
    assert ((v - y).abs()[[1, 3]] <= (0.5 / 127 + u) * top[[1, 3], None]).all()


def test_norms_near_the_range_keep_their_values():
    """A weight so large that the norm ends just inside fp32."""
    from kunserve_b200.ops import add_rms_norm_int8, dequantize_int8
    k, big = 64, torch.finfo(torch.bfloat16).max
    x = torch.zeros(1, k, device="cuda").bfloat16()
    x[0, 0] = 1.0                      # 8 times the weight, less 1 in 3200 for eps
    for share, inside in ((1.0, True), (1.01, False), (0.5, True)):
        w = torch.full((k,), big / 8 * share, device="cuda").bfloat16()
        q, s, _ = add_rms_norm_int8(x, w, 1e-5)
        v = dequantize_int8(q, s, F32)
        want = float(w[0].double()) / (1 / k + 1e-5) ** 0.5
        assert (want <= torch.finfo(F32).max) == inside
        if inside:
            assert q[0, 0] == 127 and abs(v[0, 0].item() - want) <= 45 * U * want and (v[0, 1:] == 0).all()
        else:
            assert (q == 0).all() and v.isnan().all()
