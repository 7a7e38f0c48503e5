"""Products whose waits run out: once some wait of the library has, the others
give up early.  The kernel then ends by itself, with nothing of its own in
flight, the error is reported, and later products are right.  No case here
waits for anything that is not on its way."""
import time

import pytest
import torch

from test_int8_ops_gpu import BF, F32, _linear_inputs

pytestmark = pytest.mark.gpu

# tokens, K, channels: pairs with whole units (one and several rounds), pairs that split K, single CTAs of both kinds
SHAPES = [(306, 5120, 5120), (3000, 2048, 9000), (1025, 384, 640), (500, 16384, 700), (64, 5120, 27648), (1, 4096, 6144)]


@pytest.mark.parametrize("m,k,n", SHAPES)
@pytest.mark.parametrize("dtype", [BF, F32], ids=["bf16", "fp32"])
def test_products_that_give_up_end_and_say_so(m, k, n, dtype):
    from kunserve_b200 import ops
    q, s, w, v = _linear_inputs(m, k, n)
    weight = ops.Int8Weight(w, v)
    want = ops.int8_linear(q, s, weight, dtype=dtype)
    wide = torch.full((m + 2, n + 8), 7.0, device="cuda", dtype=dtype)
    out = wide[1:m + 1, 4:n + 4]
    torch.cuda.synchronize()
    ops.check_error()
    for _ in range(5):
        ops.native().raise_error_flag(1, 0)      # as a wait that ran out would
        start = time.monotonic()
        for _ in range(4):
            ops.int8_linear(q, s, weight, out=out)
        torch.cuda.synchronize()
        # a wait for a copy that nobody made would take its whole limit, two seconds
        assert time.monotonic() - start < 1.0
        with pytest.raises(RuntimeError):
            ops.check_error()
        out.fill_(7)
        assert (wide == 7).all()                 # nothing around the result was written
        assert torch.equal(ops.int8_linear(q, s, weight, dtype=dtype), want)
        torch.cuda.synchronize()
        ops.check_error()
