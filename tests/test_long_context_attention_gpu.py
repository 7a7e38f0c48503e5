"""The long-context example's attention, request by request and layer by layer,
against a decoder of plain operations over whole sequences.

Both sides round activations, queries, keys and outputs to bf16 at the same
places; they differ by roundings of 2^-9 (relative, in norm) of the products,
of probabilities and of outputs in each of two layers, some eight of them:
2^-6.  Keys left out change an output of n keys by about sqrt(lost / n): the
last page of the prefix by 0.2, one own key by 0.05; both are planted in the
plain side and have to exceed the bound.
"""
import math
import os
import sys

import pytest
import torch

from test_cache_ops_gpu import _no_device_error, _rotated  # noqa: F401

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "evaluation"))

pytestmark = pytest.mark.gpu

BOUND = 2.0 ** -6
PREFIX, BLOCK = 333, 16


def _plain(model, tokens, hidden=None):
    """Each layer's attention output of the last token of one sequence; keys of
    the places ``hidden`` are left out for it."""
    T, nq, nkv, hd = len(tokens), model.nq, model.nkv, model.hd
    h, out = model.embed[tokens], []
    pos = torch.arange(T, device="cuda", dtype=torch.int32)
    for layer in range(model.layers):
        x = torch.nn.functional.rms_norm(h, h.shape[-1:])
        qkv = (x @ model.w_qkv[layer].t()).view(T, -1, hd)
        turned = _rotated(qkv[:, :nq + nkv], pos, model.rotary)[0].bfloat16().double()
        q, k, v = turned[:, :nq], turned[:, nq:], qkv[:, nq + nkv:].double()
        k, v = (t.repeat_interleave(nq // nkv, 1) for t in (k, v))
        s = torch.einsum("thd,shd->hts", q, k) / math.sqrt(hd)
        s.masked_fill_(torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1), -math.inf)
        if hidden is not None:
            s[:, -1, hidden] = -math.inf
        a = torch.einsum("hts,shd->thd", s.softmax(-1), v).flatten(1).bfloat16()
        out.append(a[-1].float())
        h = h + a @ model.w_o[layer].t()
    return torch.stack(out)


def _off(a, b):
    return ((a - b).norm(dim=-1) / b.norm(dim=-1))


def test_attention_of_every_request_and_layer():
    import long_context
    model, pool = long_context.Decoder(400, layers=2, seed=3), long_context.Pages(400, BLOCK)
    prefix = long_context.random_prompts(1, PREFIX, PREFIX, 4096, 1)[0]
    prompts = long_context.random_prompts(4, 2, 40, 4096, 2)
    first = long_context.random_prompts(1, 4, 4, 4096, 3)[0]
    want = torch.stack([_plain(model, torch.cat([prefix, p, first[i:i + 1]])) for i, p in enumerate(prompts)], 1)
    long_context.decode_shared(model, pool, prefix, prompts, 1, first)
    shared = torch.stack([x.float() for x in model.attended])
    assert _off(shared, want).max() < BOUND
    long_context.decode_capped(model, pool, [torch.cat([prefix, p]) for p in prompts], 1, 4096, 1, first=first)
    assert _off(torch.stack([x.float() for x in model.attended]), want).max() < BOUND
    # what the bound tells apart
    for i, p in enumerate(prompts):
        tokens = torch.cat([prefix, p, first[i:i + 1]])
        for hidden in (range(PREFIX // BLOCK * BLOCK, PREFIX), range(PREFIX, PREFIX + len(p)), [PREFIX], [len(tokens) - 1]):
            lost = _plain(model, tokens, torch.tensor(list(hidden), device="cuda"))
            assert (_off(lost, want[:, i]) > BOUND).all(), (i, hidden)


def test_example_checks_itself():
    import long_context
    assert max(long_context.check()) < long_context.CHECK_BOUND == BOUND
