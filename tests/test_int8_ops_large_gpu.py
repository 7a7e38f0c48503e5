"""The norm's residual and sum past 2^31 elements, and the scales that a handle
of float weights is made with."""
import pytest
import torch

from test_int8_ops_gpu import BF, TYPES, _no_device_error, _randn  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("t,k", [(70001, 32768), (65603, 32771), (66000, 32776)])
def test_sums_past_32_bits(t, k):
    """Rows in registers, off the vectors, and read twice; the sum beside its inputs and over one of them."""
    from kunserve_b200 import ops
    assert (t - 3) * k > 2 ** 31
    x, r = (torch.empty(t, k, device="cuda", dtype=BF).fill_(v) for v in (1, 2))
    for i, a in enumerate((x, r)):
        a[:2], a[-3:] = _randn(2 * i, 2, k).bfloat16(), _randn(2 * i + 1, 3, k).bfloat16()
    w = _randn(9, k).bfloat16()
    edge = [torch.cat([a[:2], a[-3:]]) for a in (x, r)]
    q1, s1, h1 = ops.add_rms_norm_int8(edge[0], w, residual=edge[1])
    out = torch.empty_like(x)
    for total in (out, r):
        q, s, h = ops.add_rms_norm_int8(x, w, residual=r, out=total)
        assert h.data_ptr() == total.data_ptr()
        for a, b in ((q, q1), (s, s1), (h, h1)):
            assert torch.equal(torch.cat([a[:2], a[-3:]]), b)
        assert (h[2:-3:999] == 3).all() and (h[2:-3, ::4099] == 3).all()
        del q, s, h


@pytest.mark.parametrize("dtype", list(TYPES))
def test_scales_of_float_weights(dtype):
    from kunserve_b200 import ops
    w = (_randn(1, 200, 300) * torch.logspace(-3, 3, 200, device="cuda")[:, None]).to(TYPES[dtype])
    weight = ops.Int8Weight.quantize(torch.nn.Parameter(w))
    assert not weight.scales.requires_grad
    # the quotient rounded once: of two floats the one in 64 bits (2 * 24 + 2 and more) rounds to the same
    # (a float's by a number is taken as a product with 1 / 127 here, which is off by another half step)
    assert torch.equal(weight.scales, (w.double().abs().amax(1) / 127).float())
    # a unit token's product is a column of the integers times them
    one = torch.zeros(1, 300, dtype=torch.int8, device="cuda")
    one[0, 17] = 1
    q, s = ops.quantize_int8(w)
    y = ops.int8_linear(one, torch.ones(1, device="cuda"), weight, dtype=torch.float32)
    assert torch.equal(y[0], q[:, 17].float() * s)
