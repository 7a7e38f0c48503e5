"""The long-context example norms its hidden states alike in 16 and in 8 bits."""
import os
import sys

import pytest
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "evaluation"))

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("size", [1.0, 2.0 ** -6])
def test_small_hidden_states_attend_alike(size):
    """What is added under the norm's root is small beside hidden states of 1/64
    too: the first layer's attention is off by what 8 bits round alone, at most
    0.06 as for states of size one."""
    import long_context
    plain, quant = (long_context.Decoder(40, layers=1, int8=b) for b in (False, True))
    prompt = long_context.random_prompts(1, 200, 200, 4096, 1)[0]
    for m in (plain, quant):
        m.embed = m.embed * size
        long_context.prefill(m, long_context.Pages(40, 16), [], prompt)
    a, b = plain.attended[0].float(), quant.attended[0].float()
    assert (a - b).norm() <= 0.06 * a.norm()
