"""The long-context example runs the cache operators together: logits agree
with whole per-request caches, capped requests give their pages back."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "evaluation"))

pytestmark = pytest.mark.gpu


def test_shared_and_uncapped_logits_agree():
    import long_context
    # two layers of bf16 activations: each of a handful of roundings is 2^-9
    # of its value, so a few percent bound what may add up
    assert max(long_context.check()) < 0.03


def test_capped_decoding_frees_pages():
    import long_context
    from kunserve_b200.ops import check_error
    model = long_context.Decoder(200, layers=2)
    pool = long_context.Pages(200, model.block)
    prompts = long_context.random_prompts(3, 90, 120, 4096, 3)
    out, logits, _, evictions = long_context.decode_capped(model, pool, prompts, 40, 48, 8)
    check_error()
    assert out.shape == (3, 41) and torch.isfinite(logits.float()).all()
    assert evictions >= 4
    assert 200 - len(pool.free) <= 3 * (-(-(48 + 8) // model.block))
