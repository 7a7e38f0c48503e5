"""Gradients through ``rotary_apply``: what autograd returns is the rotation's
transposed map, in the type of the input (one rounding, as in the operator)."""
import pytest
import torch

from test_cache_ops_gpu import BF, FP, U, YARN, _no_device_error, _positions, _rotated, _within  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("T,H,hd,rot", [(1, 1, 64, 64), (37, 5, 128, 96), (4, 3, 10, 6)])
def test_gradient_turns_back(dtype, interleaved, inverse, T, H, hd, rot):
    from kunserve_b200.ops import Rotary, rotary_apply
    torch.manual_seed(T)
    rotary, pos = Rotary(hd, rot, 10000.0, interleaved, YARN), _positions(T, 3)
    wide = torch.randn(T, H + 2, hd, device="cuda").to(dtype).requires_grad_()
    y = rotary_apply(wide[:, 1:H + 1], pos, rotary, inverse=inverse)     # a strided view
    with torch.no_grad():
        assert torch.equal(y, rotary_apply(wide[:, 1:H + 1], pos, rotary, inverse=inverse))
    g = torch.randn(T, H, hd, device="cuda").to(dtype)
    y.backward(g)
    want, slack = _rotated(g, pos, rotary, not inverse)
    _within(wide.grad[:, 1:H + 1], want, U[dtype] * want.abs() + slack + 2.0 ** -24)
    assert (wide.grad[:, 0] == 0).all() and (wide.grad[:, -1] == 0).all()


def test_gradient_of_a_sum_and_of_a_gradient():
    """A gradient broadcast from one number; and the map is linear, so the
    gradient of (gradient . v) by the incoming gradient is the turned v."""
    from kunserve_b200.ops import Rotary, rotary_apply
    torch.manual_seed(0)
    rotary, pos = Rotary(64), _positions(5, 1)
    x = torch.randn(5, 2, 64, device="cuda").half().requires_grad_()
    rotary_apply(x, pos, rotary).sum().backward()
    want, slack = _rotated(torch.ones_like(x), pos, rotary, True)
    _within(x.grad, want, U[FP] * want.abs() + slack + 2.0 ** -24)
    g = torch.randn_like(x).requires_grad_()
    v = torch.randn_like(x)
    first, = torch.autograd.grad(rotary_apply(x, pos, rotary), x, g, create_graph=True)
    second, = torch.autograd.grad(first, g, v)
    want, slack = _rotated(v, pos, rotary)
    _within(second, want, U[FP] * want.abs() + slack + 2.0 ** -24)


def test_gradient_is_not_lost_in_out():
    from kunserve_b200.ops import Rotary, rotary_apply
    rotary, pos = Rotary(64), _positions(2, 1)
    x = torch.randn(2, 1, 64, device="cuda").half().requires_grad_()
    for args in (dict(x=x, out=torch.empty_like(x, requires_grad=False)), dict(x=x.detach(), out=x)):
        with pytest.raises(ValueError, match="gradient"):
            rotary_apply(positions=pos, rotary=rotary, **args)
    with torch.no_grad():
        assert not rotary_apply(x, pos, rotary, out=torch.empty_like(x)).requires_grad
