"""SiLU * up in 8 bits over all gates: scales and integers of y = g / (1 + e^-g) u
to a few roundings of y itself, however small the sigmoid.

y is off by at most 11 U of itself, U = 2^-24: from -64 on e^-g is 2^n (4) times
1 + d (1, and 1 for what that leaves out or for d's own roundings), and a sum, a
reciprocal and two products follow (1, 2, 2); below, two exponentials of one
unit each and three products (8, 3).
"""
import pytest
import torch

from test_int8_ops_gpu import F32, TYPES, U, _no_device_error, _randn  # noqa: F401

pytestmark = pytest.mark.gpu

Y = 11
# an integer's quotient: of element and maximum, and its factor; a scale: of the maximum, and its quotient
ROUNDINGS = (2 * Y + 1, Y + 1)


def _exact(gate, up):
    g, u = gate.double(), up.double()
    return g / (1 + torch.exp(-g)) * u


def _check(q, s, y):
    top = y.abs().amax(1, keepdim=True)
    want = torch.where(top > 0, 127 * y / torch.where(top > 0, top, 1.0), 0.0)
    assert ((q.double() - want).abs() <= 0.5 + 127 * ROUNDINGS[0] * U).all()
    assert ((s.double() - top[:, 0] / 127).abs() <= ROUNDINGS[1] * U * top[:, 0] / 127).all()


@pytest.mark.parametrize("k", [8, 37, 1000, 5120, 14336, 40000])
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_scales_of_rows_far_from_zero(k, dtype):
    """Rows whose gates all lie near one value: nothing else hides its error."""
    from kunserve_b200.ops import silu_mul_int8
    near = [-1e-3, -0.5, -3, -8, -16.5, -31, -50, -62, -64, -79, 0, 1e-4, 2, 17, 79, 100, 1000]
    if dtype == "bf16":
        near += [-80, -81, -86.5, -87.5, -88, -88.75, -95, -103, -104, -120, -150, 1e30, 2e38]
    t = TYPES[dtype]
    gate = (torch.tensor(near, device="cuda")[:, None] * (1 + 0.01 * _randn(k, len(near), k)).clamp(0.97, 1.03)).to(t)
    # as large as the row's results leave the range (and fp16) room for
    size = torch.tensor([3e38 if n <= -80 else 1e-3 if n > 1e20 else 1.0 if t == TYPES["fp16"] else 1e30 if n < 20 else 1.0
                         for n in near], device="cuda")[:, None]
    up = ((0.5 + 0.4 * _randn(k + 1, len(near), k).clamp(-1, 1)) * size).to(t)
    y = _exact(gate, up)
    q, s = silu_mul_int8(gate, up)
    top = y.abs().amax(1)
    assert (top < torch.finfo(F32).max).all()
    keep = (top > 127 * 2.0 ** -126) | (top == 0)      # scales of normal size
    assert keep.sum() >= len(near) - 4
    _check(q[keep], s[keep], y[keep])
    # below that, a half step of the smallest float (and of y) for each rounding
    assert ((s.double() - top / 127).abs() <= (Y + 1) * U * top / 127 + 3 * 2.0 ** -149).all()


def test_a_gate_beyond_the_range_of_its_exponential():
    """e^88 and a product of 1e38: -53, not nothing."""
    from kunserve_b200.ops import dequantize_int8, silu_mul_int8
    gate = torch.tensor([[-88.0, -88.0, -3.0, -120.0]], device="cuda").bfloat16()
    up = torch.tensor([[1e38, -5e37, 1.0, 3e38]], device="cuda").bfloat16()
    q, s = silu_mul_int8(gate, up)
    y = _exact(gate, up)
    assert -54 < y[0, 0] < -53
    _check(q, s, y)
    assert ((dequantize_int8(q, s, F32).double() - y).abs() <= (0.5 / 127 + 30 * U) * y.abs().amax()).all()


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_every_gate_between(dtype):
    """A row for each of 4000 gates, eight ups each: the scale is y's."""
    from kunserve_b200.ops import silu_mul_int8
    t = TYPES[dtype]
    gate = torch.linspace(-110 if dtype == "bf16" else -95, 110, 4000, device="cuda").to(t)[:, None].repeat(1, 8)
    up = torch.tensor([2.0, 0.75, -1.5, 1.0, 0.0, 0.25, -0.125, 1.75], device="cuda").to(t).repeat(4000, 1)
    y = _exact(gate, up)
    q, s = silu_mul_int8(gate, up)
    keep = y.abs().amax(1) > 127 * 2.0 ** -126
    assert keep.sum() > 3500
    _check(q[keep], s[keep], y[keep])


def test_wide_and_narrow_gates_of_a_row():
    """Groups of eight with and without gates that have a formula of their own, rows on any element: the same bits wherever they lie."""
    from kunserve_b200.ops import silu_mul_int8
    for k in (100, 515, 4096, 33000):
        wide = (_randn(k, 6, 2 * k + 3) * 4).bfloat16()
        wide[torch.rand(6, 2 * k + 3, device="cuda") < 0.02] = -90
        wide[torch.rand(6, 2 * k + 3, device="cuda") < 0.01] = 300
        gate, up = wide[:, 1:k + 1], wide[:, k + 2:2 * k + 2]
        q, s = silu_mul_int8(gate, up)
        _check(q, s, _exact(gate, up))
        q2, s2 = silu_mul_int8(gate.contiguous(), up.contiguous())
        assert torch.equal(q, q2) and torch.equal(s, s2)


def test_gates_without_a_value():
    from kunserve_b200.ops import silu_mul_int8
    gate = torch.ones(7, 300, device="cuda").bfloat16()
    up = gate.clone()
    gate[0, 3], gate[1, 299], gate[2, 0], up[3, 7], up[4, 7] = float("nan"), float("inf"), -float("inf"), float("nan"), -float("inf")
    gate[5, 9] = -200                      # e^200 is no float: its y is zero
    gate[6, 9], up[6, 9] = 3e38, 2.0       # and this product none
    q, s = silu_mul_int8(gate, up)
    assert s.isnan().tolist() == [True] * 5 + [False, True] and (q[[0, 1, 2, 3, 4, 6]] == 0).all() and q[5, 9] == 0


@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_every_gate_there_is(dtype):
    """A row for each finite gate of the type: its scale is y / 127 to 12 U."""
    from kunserve_b200.ops import silu_mul_int8
    t = TYPES[dtype]
    gate = torch.arange(65536, device="cuda", dtype=torch.int32).to(torch.int16).view(t)
    gate = gate[gate.isfinite()][:, None].repeat(1, 8)
    for u in (1.0, 1.328125, 1e30 if dtype == "bf16" else 1000.0):
        up = torch.full_like(gate, u)
        y = _exact(gate[:, 0], up[:, 0]).abs()
        q, s = silu_mul_int8(gate, up)
        inside = y < 0.999 * torch.finfo(F32).max
        assert s[inside].isfinite().all()
        keep = inside & (y > 127 * 2.0 ** -126)
        assert ((s.double() - y / 127).abs() <= ROUNDINGS[1] * U * y / 127)[keep].all()
        assert (q[keep].abs() == 127).all()
