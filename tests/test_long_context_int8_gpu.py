"""The long-context example with its projections in 8-bit integers."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "evaluation"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("mode", ["shared", "capped"])
def test_decodes(mode):
    import long_context
    from kunserve_b200.ops import Int8Weight, check_error
    model, pool = long_context.Decoder(300, layers=3, int8=True), long_context.Pages(300, 16)
    assert all(isinstance(w, Int8Weight) for w in model.w_qkv + model.w_o)
    prompts = long_context.random_prompts(3, 20, 60, 4096, 3)
    if mode == "shared":
        out, logits, _ = long_context.decode_shared(model, pool, long_context.random_prompts(1, 90, 90, 4096, 4)[0],
                                                    prompts, 4)
    else:
        out, logits, _, _ = long_context.decode_capped(model, pool, prompts, 4, 48, 8)
    check_error()
    assert out.shape == (3, 5) and logits.isfinite().all()


def test_first_layer_attends_to_nearly_the_same():
    """Queries, keys and values of the first layer come from the same hidden
    states in 16 and in 8 bits: each is off by two roundings to 8 bits, 0.0115 of
    its size each for rows whose maxima lie within 5 times their root of mean
    squares, so by 0.016.  A score, 128 products over sqrt(128), of unit queries
    and keys is then off by 0.023 standard deviations; a softmax weight by that
    share of itself, a value by 0.016: 0.03 together for normal scores, and a
    margin of two."""
    import long_context
    plain, quant = (long_context.Decoder(40, layers=1, int8=b) for b in (False, True))
    prompt = long_context.random_prompts(1, 200, 200, 4096, 1)[0]
    for m in (plain, quant):
        long_context.prefill(m, long_context.Pages(40, 16), [], prompt)
    a, b = plain.attended[0].float(), quant.attended[0].float()
    assert (a - b).norm() <= 0.06 * a.norm()
