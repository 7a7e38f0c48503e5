"""Attention weights far below a row's largest one.

The kernels multiply the values by probabilities of 16 bits.  Every p is
rounded to the cache's type relative to a reference that is at most the row's
largest p times 2^11 (fp16) below fp16's range, so besides the relative
rounding of test_cache_ops_gpu a weight may be off by half of fp16's smallest
step, 2^-25, times 2^-11: 2^-36 of the row's largest.  bf16 has fp32's range.
"""
import math

import pytest
import torch

from test_cache_ops_gpu import BF, FP, U, _allot, _attend, _cache, _no_device_error, _rows, _within  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [FP, BF])
@pytest.mark.parametrize("gap", [13, 22, 26, 30])     # log2 of the heavy keys' weight over the others'
@pytest.mark.parametrize("n,requests", [(128, 2), (128, 20), (2500, 2), (2500, 20), (2500, 1)])
def test_light_keys_are_not_lost(dtype, gap, n, requests):
    """One key in 64 is heavy and has value zero: the output is what the light keys give."""
    from kunserve_b200.ops import PrefixGroup, SharedPrefixPlan, shared_prefix_attention
    nq, nkv, hd, bs = 4, 1, 64, 16
    pool, kv, lay = _cache(-(-n // bs) + requests, bs, nkv, hd, dtype)
    pages = _allot([n] + [1] * requests, bs, kv.pages_total, 1)
    g = torch.Generator(device="cuda").manual_seed(gap)
    heavy = torch.arange(n, device="cuda") % 64 == 0
    k, v = torch.zeros(n, hd, device="cuda"), 32 + 32 * torch.rand(n, hd, generator=g, device="cuda")
    k[heavy, 0], v[heavy] = gap * math.log(2) * math.sqrt(hd) / 8, 0.0
    for value, x in ((False, k), (True, v)):
        for i, p in enumerate(pages[0]):
            o = lay.kv_offset(p, 1, 1, value) // 2
            part = x[i * bs:(i + 1) * bs].reshape(-1).to(dtype)
            pool[o:o + part.numel()] = part
        for p in pages[1:]:                           # own keys: heavy, of value zero
            o = lay.kv_offset(p[0], 1, 1, value) // 2
            pool[o:o + hd] = 0 if value else k[0].to(dtype)
    q = torch.zeros(requests, nq, hd, device="cuda", dtype=dtype)
    q[..., 0] = 8.0
    plan = SharedPrefixPlan([PrefixGroup(pages[0], n, [(p, 1, 1) for p in pages[1:]])], kv, nq)
    got = shared_prefix_attention(q, kv, 1, plan)
    kk, vv = (torch.cat([_rows(pool, lay, pages[0], n, 1, 1, x), _rows(pool, lay, pages[1], 1, 1, 1, x)])
              for x in (False, True))
    o, tol, p, _ = _attend(q[0], kk, vv, 1 / math.sqrt(hd), U[dtype])
    assert o.min() > 0
    if dtype == FP:
        tol = tol + 2.0 ** -36 * p.max() * vv.double().abs().sum(0)
    for t in range(requests):
        _within(got[t], o, tol)
