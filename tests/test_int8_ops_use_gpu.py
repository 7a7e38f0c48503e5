"""The 8-bit operators as they are used: refused arguments, a layer of them
together, captured in graphs, on several streams."""
import pytest
import torch

from test_cache_ops_streams_gpu import _behind_queued_work
from test_int8_ops_gpu import BF, F32, HALF, U, _linear_inputs, _no_device_error, _randn, check_linear, \
    check_rows, silu_roundings  # noqa: F401

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------- refusals
def test_refused_rows():
    from kunserve_b200 import ops
    x, w = _randn(1, 4, 32).bfloat16(), _randn(2, 32).bfloat16()
    refused = [
        (lambda: ops.quantize_int8(x[0]), "must be a CUDA tensor"),
        (lambda: ops.quantize_int8(x.t()), "contiguous rows"),
        (lambda: ops.quantize_int8(x[:, :0]), "at least one column"),
        (lambda: ops.quantize_int8(x.double()), "bfloat16, float16 or float32"),
        (lambda: ops.add_rms_norm_int8(x.float(), w.float()), "bfloat16 or float16"),
        (lambda: ops.add_rms_norm_int8(x, w.half()), "weight must be"),
        (lambda: ops.add_rms_norm_int8(x, w[:16]), "weight must be"),
        (lambda: ops.add_rms_norm_int8(x, w.repeat(2)[::2]), "weight must be"),
        (lambda: ops.add_rms_norm_int8(x, w, 0.0), "eps must be positive"),
        (lambda: ops.add_rms_norm_int8(x, w, float("nan")), "eps must be positive"),
        (lambda: ops.add_rms_norm_int8(x, w, 1e-60), "eps must be positive"),
        (lambda: ops.add_rms_norm_int8(x, w, residual=x[:2]), "residual must be"),
        (lambda: ops.add_rms_norm_int8(x, w, residual=x.half()), "residual must be"),
        (lambda: ops.add_rms_norm_int8(x, w, out=x), "without a residual"),
        (lambda: ops.add_rms_norm_int8(x, w, residual=x, out=x.half()), "out must be"),
        (lambda: ops.add_rms_norm_int8(x, w, residual=x, out=x[:1].expand(4, 32)), "rows overlap"),
        (lambda: ops.silu_mul_int8(x, x[:, :16]), "up must be"),
        (lambda: ops.silu_mul_int8(x, x.half()), "up must be"),
    ]
    # results that overlap an input without being it
    flat = _randn(3, 300).bfloat16()
    a, b = flat[:128].view(4, 32), flat[4:132].view(4, 32)
    wide = _randn(4, 4, 64).bfloat16()
    refused += [(lambda: ops.add_rms_norm_int8(a, w, residual=x, out=b), "overlaps x"),
                (lambda: ops.add_rms_norm_int8(x, w, residual=a, out=b), "overlaps residual"),
                (lambda: ops.add_rms_norm_int8(wide[:, :32], w, residual=x, out=wide[:, 16:48]), "overlaps x"),
                (lambda: ops.add_rms_norm_int8(x, flat[:32], residual=x.clone(), out=flat[:128].view(4, 32)),
                 "overlaps weight")]
    for f, message in refused:
        with pytest.raises(RuntimeError, match=message):
            f()
    ops.add_rms_norm_int8(wide[:, :32], w, residual=x, out=wide[:, 32:])


def test_refused_products():
    from kunserve_b200 import ops
    q, s, w, v = _linear_inputs(4, 32, 48)
    weight = ops.Int8Weight(w, v)
    out = torch.empty(4, 48, device="cuda", dtype=BF)
    bias = torch.zeros(48, device="cuda", dtype=BF)
    refused = [
        (lambda: ops.Int8Weight(w.short(), v), "must be int8"),
        (lambda: ops.Int8Weight(w, v[:5]), "scales must be"),
        (lambda: ops.Int8Weight(w, v.half()), "scales must be"),
        (lambda: ops.Int8Weight(w.t(), v[:32]), "contiguous rows"),
        (lambda: ops.Int8Weight(w[:0], v[:0]), "needs channels"),
        (lambda: ops.Int8Weight(torch.zeros(1, 131072, dtype=torch.int8, device="cuda"), v[:1]), "at most 131071"),
        (lambda: ops.int8_linear(q.float(), s, weight), "must be int8"),
        (lambda: ops.int8_linear(q[:, :16], s, weight), "has 16 columns"),
        (lambda: ops.int8_linear(q, s[:3], weight), "scales must be"),
        (lambda: ops.int8_linear(q, s.double(), weight), "scales must be"),
        (lambda: ops.int8_linear(q, s.cpu(), weight), "scales must be"),
        (lambda: ops.int8_linear(q, s, weight, dtype=torch.float64), "must be bfloat16"),
        (lambda: ops.int8_linear(q, s, weight, out=out[:2]), "out must be"),
        (lambda: ops.int8_linear(q, s, weight, out=out.t()), "contiguous rows"),
        (lambda: ops.int8_linear(q, s, weight, out=out[:1].expand(4, 48)), "rows overlap"),
        (lambda: ops.int8_linear(q, s, weight, bias=bias[:3]), "bias must be"),
        (lambda: ops.int8_linear(q, s, weight, bias=bias, dtype=F32), "bias must be"),
        (lambda: ops.dequantize_int8(q, s, torch.int32), "must be bfloat16"),
        (lambda: ops.dequantize_int8(q, s, out=out), "q's sizes"),
        (lambda: ops.dequantize_int8(q.float(), s), "must be int8"),
    ]
    for f, message in refused:
        with pytest.raises(RuntimeError, match=message):
            f()
    with pytest.raises(AttributeError):
        ops.int8_linear(q, s, w)


def test_gradients_are_refused():
    from kunserve_b200 import ops
    x, w = _randn(1, 4, 32).bfloat16(), _randn(2, 32).bfloat16()
    q, s, wq, v = _linear_inputs(4, 32, 48)
    weight = ops.Int8Weight(wq, v)
    g = x.clone().requires_grad_()
    calls = [lambda: ops.quantize_int8(g), lambda: ops.add_rms_norm_int8(g, w), lambda: ops.silu_mul_int8(x, g),
             lambda: ops.add_rms_norm_int8(x, w.clone().requires_grad_()),
             lambda: ops.add_rms_norm_int8(x, w, residual=g),
             lambda: ops.int8_linear(q, s.clone().requires_grad_(), weight),
             lambda: ops.dequantize_int8(q, s.clone().requires_grad_())]
    for f in calls:
        with pytest.raises(ValueError, match="requires a gradient"):
            f()
        with torch.no_grad():
            f()


@pytest.mark.parametrize("tokens", [2, 500])
def test_results_are_plain_tensors(tokens):
    """Whether they share their memory or not: copied, changed in place, kept
    apart from the others, used by what records gradients and by what does not."""
    import copy

    from kunserve_b200 import ops
    x, w = _randn(1, tokens, 200).bfloat16(), torch.ones(200, device="cuda", dtype=BF)
    q, s, h = ops.add_rms_norm_int8(x, w, residual=x)
    saved = [t.clone() for t in (q, s, h)]
    assert all(torch.equal(copy.deepcopy(t), c) and torch.equal(t.cpu(), c.cpu()) for t, c in zip((q, s, h), saved))
    h.add_(1)
    assert torch.equal(h, saved[2] + 1) and torch.equal(q, saved[0]) and torch.equal(s, saved[1])
    q.zero_(), s.fill_(3)
    assert torch.equal(h, saved[2] + 1) and (q == 0).all() and (s == 3).all()
    p = torch.nn.Parameter(torch.ones(200, device="cuda", dtype=BF))
    (h * p).sum().backward()
    assert p.grad is not None and not h.requires_grad
    with torch.inference_mode():
        q2, s2, h2 = ops.add_rms_norm_int8(x, w, residual=x)
        y = ops.int8_linear(q2, s2, ops.Int8Weight.quantize(w[None].repeat(3, 1)))
        h2.mul_(2)
    assert y.shape == (tokens, 3) and torch.equal(h2, saved[2] * 2)


# ------------------------------------------------------------- a layer of them
class Layer:
    """Projections of a decoder layer in 8 bits; every value's group of heads
    attends to itself alone (its attention is the value)."""

    def __init__(self, hidden, heads, kv_heads, hd, inner, seed=0):
        from kunserve_b200 import ops
        self.shape = (hidden, heads, kv_heads, hd, inner)

        def weight(n, k, seed):
            return ops.Int8Weight.quantize(_randn(seed, n, k).bfloat16() / k ** 0.5)

        self.norms = [(1 + 0.1 * _randn(seed + i, hidden)).bfloat16() for i in range(2)]
        self.qkv = weight((heads + 2 * kv_heads) * hd, hidden, seed + 2)
        self.o = weight(hidden, heads * hd, seed + 3)
        self.gate_up = weight(2 * inner, hidden, seed + 4)
        self.down = weight(hidden, inner, seed + 5)

    def run(self, x, residual, steps=None):
        """Output and residual; ``steps`` gathers what each operator took and gave."""
        from kunserve_b200 import ops
        hidden, heads, kv_heads, hd, inner = self.shape
        note = steps.append if steps is not None else lambda s: None
        q, s, h = ops.add_rms_norm_int8(x, self.norms[0], 1e-5, residual=residual)
        note(("norm", x, residual, self.norms[0], q, s, h))
        qkv = ops.int8_linear(q, s, self.qkv)
        note(("linear", q, s, self.qkv, qkv))
        v = qkv.view(-1, heads + 2 * kv_heads, hd)[:, heads + kv_heads:]
        att = v.repeat_interleave(heads // kv_heads, 1).flatten(1)
        q, s = ops.quantize_int8(att)
        note(("quantize", att, q, s))
        y = ops.int8_linear(q, s, self.o)
        note(("linear", q, s, self.o, y))
        q, s, h2 = ops.add_rms_norm_int8(y, self.norms[1], 1e-5, residual=h)
        note(("norm", y, h, self.norms[1], q, s, h2))
        gu = ops.int8_linear(q, s, self.gate_up)
        note(("linear", q, s, self.gate_up, gu))
        q, s = ops.silu_mul_int8(gu[:, :inner], gu[:, inner:])
        note(("silu", gu, q, s))
        y = ops.int8_linear(q, s, self.down)
        note(("linear", q, s, self.down, y))
        return y, h2


def unpacked(weight):
    """A handle's integers, through products with the unit tokens."""
    from kunserve_b200 import ops
    eye = torch.eye(weight.in_features, device="cuda").to(torch.int8)
    one = torch.ones(weight.in_features, device="cuda")
    return (ops.int8_linear(eye, one, weight, dtype=F32).double() / weight.scales.double()).round().t().to(torch.int8)


@pytest.mark.parametrize("tokens", [1, 37, 300])
@pytest.mark.parametrize("shape", [(256, 8, 2, 64, 768), (200, 3, 1, 40, 328)])
def test_layer(tokens, shape):
    """Every operator of the layer against its formula on what it was given."""
    layer, steps = Layer(*shape), []
    x, r = _randn(10, tokens, shape[0]).bfloat16(), _randn(11, tokens, shape[0]).bfloat16()
    layer.run(x, r, steps)
    assert len(steps) == 8
    for kind, *args in steps:
        if kind == "norm":
            a, b, w, q, s, h = args
            t = a.double() + b.double()
            check_rows(q, s, t / (t.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double(), 6, 42 / 2 + 12)
            assert torch.equal(h, (a.float() + b.float()).bfloat16())
        elif kind == "quantize":
            check_rows(args[1], args[2], args[0].double(), 2, 1)
        elif kind == "silu":
            g, u = args[0].double().chunk(2, 1)
            check_rows(args[1], args[2], g / (1 + torch.exp(-g)) * u, *silu_roundings(g))
        else:
            q, s, weight, y = args
            check_linear(y, q, s, unpacked(weight), weight.scales)


def test_layer_near_its_weights_in_full():
    """Of the layer in 64 bits without any integers the 8-bit one is off by what
    8 bits round: each of four products adds the rounding of its tokens and of
    its weights.  An integer is off by at most 1/2, evenly spread by 0.29; rows of
    K normal values have maxima of 3 to 5 times their root of mean squares, so
    that is 0.29 * 5 / 127 = 0.0115 of a value's size, twice a product and root 2
    of it together; the norms and the gated product carry it on at about its size
    (a gated product adds two of them).  Eight such and a margin of two: 0.13."""
    from kunserve_b200 import ops  # noqa: F401
    shape = (512, 8, 8, 64, 1024)
    layer = Layer(*shape)
    x, r = _randn(10, 64, 512).bfloat16(), _randn(11, 64, 512).bfloat16()
    y, h2 = layer.run(x, r)

    def weight(n, k, seed):
        return (_randn(seed, n, k).bfloat16() / k ** 0.5).double()

    def norm(t, w):
        return t / (t.square().mean(1, keepdim=True) + 1e-5).sqrt() * w.double()

    h = x.double() + r.double()
    v = norm(h, layer.norms[0]) @ weight(24 * 64, 512, 2)[16 * 64:].t()
    h = h + v @ weight(512, 512, 3).t()
    g, u = (norm(h, layer.norms[1]) @ weight(2048, 512, 4).t()).chunk(2, 1)
    want = (g / (1 + torch.exp(-g)) * u) @ weight(512, 1024, 5).t()
    assert (y.double() - want).norm() <= 0.13 * want.norm()
    assert (h2.double() - h).norm() <= 0.13 * h.norm()


# ------------------------------------------------------------ graphs, streams
@pytest.mark.parametrize("tokens", [1, 50, 290])
def test_layer_in_two_graphs(tokens):
    """Two captured layers, replayed in turn and with new inputs, give what calls give."""
    a, b = Layer(256, 8, 2, 64, 768), Layer(256, 8, 2, 64, 768, seed=50)
    x, r = _randn(1, tokens, 256).bfloat16(), _randn(2, tokens, 256).bfloat16()
    for layer in (a, b):
        layer.run(x, r)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for layer in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer.run(x, r))
        graphs.append(g)
    for seed in (3, 4):
        x.copy_(_randn(seed, tokens, 256)), r.copy_(_randn(seed + 10, tokens, 256))
        for g in graphs + graphs[::-1]:
            g.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in o] for o in outs]
        for layer, o in zip((a, b), got):
            assert all(torch.equal(m, n) for m, n in zip(o, layer.run(x, r)))


def test_first_product_of_a_size_inside_a_capture():
    from kunserve_b200 import ops
    q, s, w, v = _linear_inputs(219, 130, 260)
    weight = ops.Int8Weight(w, v)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        y = ops.int8_linear(q, s, weight)
    g.replay()
    check_linear(y, q, s, w, v)


def test_two_streams_at_once():
    layer = Layer(256, 8, 2, 64, 768)
    inputs = [(_randn(i, 40 + i, 256).bfloat16(), _randn(20 + i, 40 + i, 256).bfloat16()) for i in range(2)]
    want = [layer.run(*i) for i in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for k in range(2):
            with torch.cuda.stream(streams[k]):
                got[k].append(layer.run(*inputs[k]))
    torch.cuda.synchronize()
    for k in range(2):
        for o in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(o, want[k]))


def test_weight_made_on_one_stream_used_on_another():
    from kunserve_b200 import ops
    q, s, w, v = _linear_inputs(5, 512, 384)
    got, want = _behind_queued_work(lambda: ops.Int8Weight(w, v), lambda weight: ops.int8_linear(q, s, weight))
    assert torch.equal(got, want)


def test_weight_is_used_right_after_it_was_made():
    """A product's first loads run ahead of its wait for the kernel before it:
    never ahead of the one that writes the weights."""
    from kunserve_b200 import ops
    q, s, w, v = _linear_inputs(9, 4096, 4096)
    want = ops.int8_linear(q, s, ops.Int8Weight(w, v))
    flipped = (w.int() * -1).clamp(max=127).to(torch.int8)
    q[q == -128] = 0
    for i in range(20):
        # the same memory each time, with other weights
        for weights, sign in ((w, 1), (flipped, -1)):
            weight = ops.Int8Weight(weights, v)
            y = ops.int8_linear(q, s, weight, dtype=F32)
            ref = (q.double() @ weights.double().t()) * s.double()[:, None] * v.double()
            assert ((y.double() - ref).abs() <= 4 * U * (ref.abs() + 1e-30)).all(), (i, sign)
            del weight
    assert want.shape == (9, 4096)


def test_a_recorded_bad_index_stops_nothing():
    from kunserve_b200 import ops
    q, s, w, v = _linear_inputs(70, 3000, 700)
    weight = ops.Int8Weight(w, v)
    want = ops.int8_linear(q, s, weight)
    ops.native().raise_error_flag(6, 0)
    try:
        for _ in range(3):
            assert torch.equal(ops.int8_linear(q, s, weight), want)
    finally:
        with pytest.raises(RuntimeError, match="index out of bounds"):
            ops.check_error()


def test_results_repeat():
    """The same bits every time: integer sums have no order."""
    from kunserve_b200 import ops
    for m, k, n in ((3, 4096, 1000), (200, 2000, 3000), (1000, 512, 700)):
        q, s, w, v = _linear_inputs(m, k, n, 7)
        weight = ops.Int8Weight(w, v)
        want = ops.int8_linear(q, s, weight, dtype=HALF)
        for _ in range(10):
            assert torch.equal(ops.int8_linear(q, s, weight, dtype=HALF), want)


# ------------------------------------------------------- offsets past 32 bits
def test_rows_past_32_bits():
    from kunserve_b200 import ops
    t, k = 70001, 32768
    x = torch.empty(t, k, device="cuda", dtype=BF)
    x[-3:] = _randn(1, 3, k).bfloat16()
    x[:2] = _randn(2, 2, k).bfloat16()
    w = _randn(3, k).bfloat16()
    edge = torch.cat([x[:2], x[-3:]])
    for f in (ops.quantize_int8, lambda v: ops.silu_mul_int8(v, v), lambda v: ops.add_rms_norm_int8(v, w)[:2]):
        x[2:-3] = 1
        (q, s), (q1, s1) = f(x), f(edge)
        assert torch.equal(torch.cat([q[:2], q[-3:]]), q1) and torch.equal(torch.cat([s[:2], s[-3:]]), s1)
        v = ops.dequantize_int8(q, s)
        assert torch.equal(v[-3:], ops.dequantize_int8(q1, s1)[-3:])
        del q, v


def test_products_past_32_bits():
    from kunserve_b200 import ops
    # the result: 2.3e9 elements; the weights: 2.3e9 bytes
    for m, k, n in ((17001, 40, 135000), (5, 16400, 140001)):
        q, s, w, v = _linear_inputs(m, k, n)
        y = ops.int8_linear(q, s, ops.Int8Weight(w, v))
        rows, last = torch.tensor([0, m // 2, m - 1], device="cuda"), n - 200
        check_linear(y[rows][:, last:], q[rows], s[rows], w[last:], v[last:])
        check_linear(y[rows][:, :300], q[rows], s[rows], w[:300], v[:300])
        del y, w


def test_clusters_that_the_device_holds():
    """What cuts are chosen by: of single CTAs one an SM, of clusters no more than fit."""
    from kunserve_b200.ops import native
    slots = native().int8_slots()
    sms = native().num_sms()
    assert slots[1] == sms and all(1 <= slots[c] and c * slots[c] <= sms for c in range(2, 9))
