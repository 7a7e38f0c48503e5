"""The 8-bit operators against their formulas in 64 bits.

Bounds.  U = 2^-24 is half a step of fp32.  An integer is off by half, and by
what the roundings of its quotient make of 127; a result of the matrix product
by half a step of its type and by three fp32 roundings of its scaled sum.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
BF, HALF, F32 = torch.bfloat16, torch.float16, torch.float32
TYPES = {"bf16": BF, "fp16": HALF, "fp32": F32}


@pytest.fixture(autouse=True)
def _no_device_error():
    from kunserve_b200.ops import check_error
    yield
    check_error()


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _randn(seed, *shape):
    return torch.randn(*shape, generator=_gen(seed), device="cuda")


def check_rows(q, scales, y, roundings, scale_roundings):
    """q, scales: of the rows y (64 bits).  ``roundings``: of an integer's quotient, in U."""
    top = y.abs().amax(1, keepdim=True)
    assert q.dtype == torch.int8 and scales.dtype == F32 and q.shape == y.shape and scales.shape == y.shape[:1]
    assert (q.stride(0) % 16 == 0 or q.shape[0] <= 1) and q.data_ptr() % 16 == 0
    want = torch.where(top > 0, 127 * y / torch.where(top > 0, top, 1.0), 0.0)
    assert ((q.double() - want).abs() <= 0.5 + 127 * roundings * U).all()
    assert ((scales.double() - top[:, 0] / 127).abs() <= scale_roundings * U * top[:, 0] / 127).all()


# widths: one element, below a vector, whole vectors, odd, each variant's largest, read twice
WIDTHS = [1, 7, 8, 17, 100, 128, 255, 256, 257, 512, 513, 1000, 1024, 2047, 2048, 4096, 5119, 5120, 6144, 8192, 8195, 13824,
          16384, 32767, 32768, 32776]


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_quantize(k, dtype):
    from kunserve_b200.ops import dequantize_int8, quantize_int8
    x = (_randn(k, 5, k) * torch.tensor([1.0, 100.0, 1e-3, 0.0, 7.0], device="cuda")[:, None]).to(TYPES[dtype])
    q, s = quantize_int8(x)
    # 16-bit inputs: 127 x is exact in fp32, and a quotient of two 11-bit numbers is a half or far from one
    y = x.double()
    top = y.abs().amax(1, keepdim=True)
    check_rows(q, s, y, 2, 1)
    if dtype != "fp32":
        assert torch.equal(q.double(), torch.where(top > 0, 127 * y / top, 0.0).nan_to_num().round())
    for out in TYPES.values():
        v = dequantize_int8(q, s, out)
        assert v.dtype == out and torch.equal(v, (q.float() * s[:, None]).to(out))


def test_no_tokens():
    from kunserve_b200 import ops
    x = torch.empty(0, 48, device="cuda", dtype=BF)
    for q, s, *h in (ops.quantize_int8(x), ops.silu_mul_int8(x, x), ops.add_rms_norm_int8(
            x, torch.ones(48, device="cuda", dtype=BF), residual=x)):
        assert q.shape == (0, 48) and s.shape == (0,) and all(t.shape == (0, 48) for t in h)
    assert ops.dequantize_int8(*ops.quantize_int8(x)).shape == (0, 48)


@pytest.mark.parametrize("tokens", [0, 1, 3, 257])
def test_quantize_tokens(tokens):
    from kunserve_b200.ops import dequantize_int8, quantize_int8
    for k in (64, 200, 520, 1000, 4096):
        x = _randn(k, tokens, k).bfloat16()
        q, s = quantize_int8(x)
        check_rows(q, s, x.double(), 2, 1)
        assert dequantize_int8(q, s).shape == (tokens, k)


def test_halves_go_to_even():
    from kunserve_b200.ops import quantize_int8
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -126.5, 126.5]], device="cuda")
    for t in TYPES.values():
        q, s = quantize_int8((x * 4).to(t))
        assert q[0].tolist() == [127, 0, 2, 2, 0, -2, -126, 126] and s.item() == 4.0


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(k, dtype, residual):
    from kunserve_b200.ops import add_rms_norm_int8
    t = TYPES[dtype]
    x, w = (_randn(1, 4, k) * 3).to(t), (1 + 0.2 * _randn(2, k)).to(t)
    r = (_randn(3, 4, k) * 5).to(t) if residual else None
    q, s, h = add_rms_norm_int8(x, w, 1e-5, residual=r)
    total = x.double() + (r.double() if residual else 0)
    y = total / (total.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()
    # quotient: the sum, its product with w, of element and maximum; the product with 127, the quotient.
    # scale: a sum of squares adds at most 8 * 4 and 10 terms after one another (more where a row is read twice:
    # 8 * ceil(k / 8192)), half of their roundings count; rsqrt two steps, four products and quotients
    depth = 42 if k <= 32768 else 8 * math.ceil(k / 8192) + 10
    check_rows(q, s, y, 6, depth / 2 + 12)
    if residual:
        assert h.dtype == t and torch.equal(h, (x.float() + r.float()).to(t))
    else:
        assert h is x or h.data_ptr() == x.data_ptr()


@pytest.mark.parametrize("where", ["x", "residual", "columns"])
@pytest.mark.parametrize("k", [24, 37, 1000, 1003, 4096, 5119, 32776])
def test_norm_sum_in_place(where, k):
    """The sum over x, over the residual, or in other columns of their buffer."""
    from kunserve_b200.ops import add_rms_norm_int8
    wide = _randn(1, 6, 3 * k).bfloat16()
    x, r, o = wide[:, :k], wide[:, k:2 * k], wide[:, 2 * k:]
    w = _randn(2, k).bfloat16()
    x0, r0 = x.clone(), r.clone()
    want = add_rms_norm_int8(x0, w, 1e-6, residual=r0)
    out = {"x": x, "residual": r, "columns": o}[where]
    q, s, h = add_rms_norm_int8(x, w, 1e-6, residual=r, out=out)
    assert torch.equal(q, want[0]) and torch.equal(s, want[1]) and torch.equal(out, want[2])
    assert h.data_ptr() == out.data_ptr()
    if where != "x":
        assert torch.equal(x, x0)
    if where != "residual":
        assert torch.equal(r, r0)


def silu_roundings(g):
    """Of an integer's quotient and of a scale, in U.  y: e^-g is off by 2 + 1.173 |g| units in the last place (two U
    each; the bound that CUDA states for its fast exponential), the sum by one U, its reciprocal by a unit, two
    products by a U each: 9 + 2.35 |g|, of element and maximum.  The quotient's factor is off by one more, the scale
    by one for its quotient."""
    y = 9 + 2.35 * g.abs().max().item()
    return 2 * y + 1, y + 1


@pytest.mark.parametrize("k", WIDTHS)
@pytest.mark.parametrize("dtype", ["bf16", "fp16"])
def test_silu(k, dtype):
    from kunserve_b200.ops import silu_mul_int8
    wide = (_randn(1, 5, 2 * k) * 3).to(TYPES[dtype])
    gate, up = wide[:, :k], wide[:, k:]
    q, s = silu_mul_int8(gate, up)
    g = gate.double()
    check_rows(q, s, g / (1 + torch.exp(-g)) * up.double(), *silu_roundings(g))


def test_silu_large_gates():
    """Gates whose exponential leaves fp32: the limits 0 and the gate itself."""
    from kunserve_b200.ops import dequantize_int8, silu_mul_int8
    gate = torch.tensor([[-200.0, -1e4, 200.0, 1e4, 0.0, -89.0, 88.0, 3.0]], device="cuda").bfloat16()
    q, s = silu_mul_int8(gate, torch.ones_like(gate))
    v = dequantize_int8(q, s, F32)
    assert q[0, :3].tolist() == [0, 0, 3] and q[0, 3] == 127 and v[0, 3].item() == pytest.approx(float(gate[0, 3]), rel=4 * U)


def test_rows_of_any_stride():
    from kunserve_b200.ops import add_rms_norm_int8, dequantize_int8, quantize_int8, silu_mul_int8
    for k, wide, at in ((64, 72, 3), (64, 96, 16), (1000, 2048, 8), (37, 41, 1), (2051, 2100, 5)):
        buf = _randn(k, 9, wide).bfloat16()
        x = buf[:, at:at + k]
        w = _randn(1, k).bfloat16()
        c = x.clone()
        for f in (quantize_int8, lambda v: silu_mul_int8(v, v), lambda v: add_rms_norm_int8(v, w, residual=v)):
            for a, b in zip(f(x), f(c)):
                assert torch.equal(a, b)
        for shift in range(8):                      # sums around rows that start on any element
            flat = torch.full((9 * k + 16,), 3.0, device="cuda").bfloat16()
            out = flat[shift:shift + 9 * k].view(9, k)
            want = add_rms_norm_int8(x, w, residual=c)
            got = add_rms_norm_int8(x, w, residual=x, out=out)
            assert all(torch.equal(a, b) for a, b in zip(got, want))
            assert (flat[:shift] == 3).all() and (flat[shift + 9 * k:] == 3).all()
            v = dequantize_int8(*want[:2], out=out)
            assert torch.equal(v, dequantize_int8(*want[:2]))
            assert (flat[:shift] == 3).all() and (flat[shift + 9 * k:] == 3).all()
        rep = buf[:1, at:at + k].expand(9, k)       # one row for all tokens
        for a, b in zip(quantize_int8(rep), quantize_int8(rep.clone())):
            assert torch.equal(a, b)
        q, s = quantize_int8(x)
        q8 = torch.zeros(9, wide, dtype=torch.int8, device="cuda")
        q8[:, at:at + k] = q
        out = torch.full((9, wide), 5.0, device="cuda", dtype=HALF)
        v = dequantize_int8(q8[:, at:at + k], s, out=out[:, at:at + k])
        assert torch.equal(v, dequantize_int8(q, s, HALF)) and (out[:, :at] == 5).all() and (out[:, at + k:] == 5).all()


@pytest.mark.parametrize("k", [5, 256, 4096, 40000])
def test_rows_without_a_value(k):
    """A NaN or an infinity anywhere: scale NaN, integers 0; the other rows keep theirs."""
    from kunserve_b200.ops import Int8Weight, add_rms_norm_int8, dequantize_int8, int8_linear, quantize_int8, \
        silu_mul_int8
    x = _randn(1, 5, k).bfloat16()
    bad = x.clone()
    bad[1, k - 1], bad[2, 0], bad[4, k // 2] = math.nan, math.inf, -math.inf
    w = torch.ones(k, device="cuda").bfloat16()
    one = torch.ones_like(x)
    for f in (quantize_int8, lambda v: silu_mul_int8(one, v), lambda v: add_rms_norm_int8(v, w)[:2],
              lambda v: add_rms_norm_int8(v, w, residual=one)[:2]):
        (q, s), (q0, s0) = f(bad), f(x)
        assert s.isnan().tolist() == [False, True, True, False, True] and (q[[1, 2, 4]] == 0).all()
        assert torch.equal(q[[0, 3]], q0[[0, 3]]) and torch.equal(s[[0, 3]], s0[[0, 3]])
        assert dequantize_int8(q, s).isnan().all(1).tolist() == s.isnan().tolist()
        weight = Int8Weight(torch.ones(3, k, dtype=torch.int8, device="cuda"), torch.ones(3, device="cuda"))
        assert int8_linear(q, s, weight).isnan().all(1).tolist() == s.isnan().tolist()


def test_rows_at_the_ends_of_the_range():
    """Zeros, the largest and the smallest values of each type."""
    from kunserve_b200.ops import add_rms_norm_int8, dequantize_int8, quantize_int8
    for t in TYPES.values():
        big = torch.finfo(t).max
        x = torch.tensor([[0.0] * 4, [big, -big, big / 2, 0.0], [torch.finfo(t).tiny, 0, 0, -torch.finfo(t).tiny]],
                         device="cuda", dtype=torch.float64).to(t)
        q, s = quantize_int8(x)
        assert q.tolist()[0] == [0] * 4 and s[0] == 0 and q.tolist()[1] == [127, -127, 64, 0]
        assert q.tolist()[2] == [127, 0, 0, -127]
        v = dequantize_int8(q[1:2], s[1:2], F32)
        assert v[0, 2].item() == pytest.approx(64 / 127 * big, rel=3 * U)
    z = torch.zeros(2, 100, device="cuda", dtype=HALF)
    q, s, _ = add_rms_norm_int8(z, torch.ones_like(z[0]))
    assert (q == 0).all() and (s == 0).all()


def _linear_inputs(m, k, n, seed=0, channels_first=True):
    g = _gen(seed)
    q = torch.randint(-128, 128, (m, k), generator=g, device="cuda", dtype=torch.int8)
    w = torch.randint(-128, 128, (n, k), generator=g, device="cuda", dtype=torch.int8)
    s = torch.rand(m, generator=g, device="cuda") * 0.01
    v = torch.rand(n, generator=g, device="cuda") * 0.01
    return q, s, w, v


def check_linear(y, q, s, w, v, bias=None):
    acc = (q.double() @ w.double().t()) * s.double()[:, None] * v.double()
    want = acc if bias is None else acc + bias.double()
    half = torch.finfo(y.dtype).eps / 2
    bound = half * want.abs() * (1 + 8 * U) + (1 + half) * 3 * U * (acc.abs() + want.abs())
    if y.dtype == HALF:
        bound = bound + 2.0 ** -25
    assert ((y.double() - want).abs() <= bound).all()


# tokens: each tile width, ragged, more than one tile; K: below, at and past blocks, odd; N: odd, below a block, many
SHAPES = [(1, 128, 128), (1, 16, 1), (1, 4096, 6144), (2, 1, 3), (5, 100, 77), (16, 512, 130), (17, 4096, 256),
          (31, 1000, 333), (48, 129, 1000), (64, 5120, 2048), (65, 256, 127), (128, 640, 640), (130, 33, 129),
          (200, 2047, 515), (256, 1024, 384), (257, 300, 260), (306, 5120, 512), (513, 144, 1111), (700, 64, 4099),
          (1025, 384, 640), (16, 128, 40000), (64, 128, 40000), (130, 128, 20000), (300, 16384, 128)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", list(TYPES))
def test_linear(m, k, n, dtype):
    from kunserve_b200.ops import Int8Weight, int8_linear
    q, s, w, v = _linear_inputs(m, k, n)
    weight = Int8Weight(w, v)
    assert (weight.out_features, weight.in_features) == (n, k)
    bias = (0.1 * _randn(1, n)).to(TYPES[dtype])
    check_linear(int8_linear(q, s, weight, dtype=TYPES[dtype]), q, s, w, v)
    check_linear(int8_linear(q, s, weight, bias=bias, dtype=TYPES[dtype]), q, s, w, v, bias)


def test_linear_sums_are_exact():
    """The largest sums that 32 bits hold, and neighbours of them."""
    from kunserve_b200.ops import Int8Weight, int8_linear
    for k in (1 << 14, 131071):
        q = torch.full((3, k), -128, dtype=torch.int8, device="cuda")
        w = torch.full((130, k), -128, dtype=torch.int8, device="cuda")
        w[1, 7], w[129, k - 1], q[2, 11] = -127, 127, 0
        one = torch.ones(130, device="cuda")
        y = int8_linear(q, one[:3].contiguous(), Int8Weight(w, one), dtype=F32)
        assert torch.equal(y, (q.double() @ w.double().t()).float())


def test_linear_of_strided_tokens_and_results():
    from kunserve_b200.ops import Int8Weight, int8_linear
    for m, k, n in ((1, 100, 70), (3, 128, 128), (33, 200, 300), (300, 77, 150)):
        q, s, w, v = _linear_inputs(m, k, n, 3)
        want = int8_linear(q, s, Int8Weight(w, v))
        for wide, at in ((k + 5, 3), ((k + 31) // 16 * 16, 0), ((k + 47) // 16 * 16, 16)):
            buf = torch.full((m, wide + at), 99, dtype=torch.int8, device="cuda")
            buf[:, at:at + k] = q
            wb = torch.full((n, wide + at), 99, dtype=torch.int8, device="cuda")
            wb[:, at:at + k] = w
            weight = Int8Weight(wb[:, at:at + k], v)
            assert torch.equal(int8_linear(buf[:, at:at + k], s, weight), want)
            out = torch.full((m + 2, n + 9), 7.0, device="cuda", dtype=BF)
            got = int8_linear(buf[:, at:at + k], s, weight, out=out[1:m + 1, 4:n + 4])
            assert torch.equal(got, want) and got.data_ptr() == out[1:, 4:].data_ptr()
            out[1:m + 1, 4:n + 4] = 7
            assert (out == 7).all()                      # nothing around the result was written
        rep = q[:1].expand(m, k)
        assert torch.equal(int8_linear(rep, s, Int8Weight(w, v)), int8_linear(rep.clone(), s, Int8Weight(w, v)))


def test_linear_without_tokens():
    from kunserve_b200.ops import Int8Weight, int8_linear
    q, s, w, v = _linear_inputs(0, 64, 32)
    assert int8_linear(q, s, Int8Weight(w, v)).shape == (0, 32)


def test_weight_of_floats():
    from kunserve_b200.ops import Int8Weight, dequantize_int8, int8_linear, quantize_int8
    w = torch.nn.Parameter(_randn(1, 200, 300).bfloat16())
    x = _randn(2, 10, 300).bfloat16()
    q, s = quantize_int8(x)
    y = int8_linear(q, s, Int8Weight.quantize(w), dtype=F32)
    wq, ws = quantize_int8(w.detach())
    check_linear(y, q, s, wq, ws)
    # the handle holds copies
    weight = Int8Weight(wq, ws)
    wq.zero_(), ws.zero_()
    assert torch.equal(int8_linear(q, s, weight, dtype=F32), y)
    # each integer is off by half of its scale
    ref = x.double() @ w.detach().double().t()
    off = (0.5 * s.double()[:, None] * w.detach().double().abs().sum(1)
           + 0.5 * weight.scales.double().new_tensor(1) * dequantize_int8(q, s, F32).double().abs().sum(1)[:, None]
           * (w.detach().double().abs().amax(1) / 127))
    assert ((y.double() - ref).abs() <= off * (1 + 1e-4)).all()
