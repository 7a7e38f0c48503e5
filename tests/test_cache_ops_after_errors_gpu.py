"""A bad index is recorded and its access left out; the calls after it run as
if it had not been, until ``check_error`` reports it."""
import pytest
import torch

from test_cache_ops_gpu import BF, _allot, _cache, _fill, _no_device_error  # noqa: F401

pytestmark = pytest.mark.gpu


def test_a_bad_row_does_not_reach_later_calls():
    """Kernels with long waits (many blocks a unit, a large product) behind an
    append with a page outside the cache."""
    from kunserve_b200.ops import (DecodePlan, PrefixGroup, Rotary, SharedPrefixPlan, check_error, native,
                                   rotary_append, shared_prefix_attention, weighted_decode_attention)
    nq, nkv, hd, bs, prefix, own = 32, 8, 128, 16, 4000, 40
    pool, kv, lay = _cache(1000, bs, nkv, hd, BF)
    pages = _allot([prefix] + [own] * 40 + [3000], bs, kv.pages_total, 1)
    for i, (p, n) in enumerate(zip(pages, [prefix] + [own] * 40 + [3000])):
        _fill(pool, lay, p, n, 1, 1, i)
    torch.manual_seed(0)
    q = torch.randn(40, nq, hd, device="cuda").to(BF)
    plan = SharedPrefixPlan([PrefixGroup(pages[0], prefix, [(p, own, 1) for p in pages[1:-1]])], kv, nq)
    decode = DecodePlan([pages[-1]], [3000], kv, nq)
    a, b = (torch.randn(n, 2048, device="cuda").to(BF) for n in (704, 1152))
    qkv, i32 = torch.zeros(1, nq + 2 * nkv, hd, device="cuda", dtype=BF), dict(dtype=torch.int32, device="cuda")
    rotary, position = Rotary(hd), torch.zeros(1, **i32)
    bad_page, slot = torch.tensor([kv.pages_total], **i32), torch.zeros(1, **i32)

    def results():
        w = torch.zeros(kv.pages_total, nkv, bs, device="cuda")
        out = torch.empty(704, 1152, device="cuda", dtype=BF)
        native().gemm(a, b, out, native().EPI_BF16, None, 0, 16)
        return [shared_prefix_attention(q, kv, 1, plan), weighted_decode_attention(q[:1], kv, 1, decode, w), w, out]

    want = results()
    torch.cuda.synchronize()
    check_error()
    for _ in range(5):
        rotary_append(qkv, position, bad_page, slot, rotary, kv, 1)
        *got, product = results()
        for x, y in zip(got, want):
            assert torch.equal(x, y)
        # the product's partial sums meet in no fixed order: fp32 sums, rounded once
        assert torch.allclose(product.float(), want[-1].float(), rtol=2.0 ** -7, atol=2.0 ** -6)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_error()
