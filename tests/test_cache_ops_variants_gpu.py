"""Every variant that the cache operators choose by size runs at least once
against the 64-bit forms (tolerances: test_cache_ops_gpu); each test asserts
from the plan or the sizes that its variant is the one taken."""
import math

import pytest
import torch

from test_cache_ops_gpu import (BF, FP, LLAMA3, U, _allot, _attend, _cache, _evict_case, _few, _fill,  # noqa: F401
                                _no_device_error, _positions, _rotated, _rows, _uniform, _within)

pytestmark = pytest.mark.gpu


@pytest.fixture
def tables(monkeypatch):
    """The section tables of the plans made during a test."""
    from kunserve_b200.ops import plans
    made, build = [], plans.build

    def keep(*args, **kwargs):
        blob, table = build(*args, **kwargs)
        made.append(table)
        return blob, table

    monkeypatch.setattr(plans, "build", keep)
    return made


# more than 32 parts a row: eight warps join it and the weights follow in a
# kernel of their own; more than 256: each of them takes a second round
@pytest.mark.parametrize("lens,nq,nkv,hd,dtype,parts", [([3000, 0, 40], 8, 2, 128, BF, 32), ([3001], 128, 1, 64, FP, 32),
                                                        ([20000, 7], 4, 1, 128, FP, 256), ([20011], 40, 2, 64, BF, 32)])
def test_weighted_decode_of_many_parts(lens, nq, nkv, hd, dtype, parts, tables):
    from kunserve_b200.ops import DecodePlan, weighted_decode_attention
    block = 16
    pool, kv, lay = _cache(sum(-(-n // block) for n in lens) + 1, block, nkv, hd, dtype, poison=True)
    pages = _allot(lens, block, kv.pages_total, 3)
    for i, (p, n) in enumerate(zip(pages, lens)):
        _fill(pool, lay, p, n, 0, 1, i)
    torch.manual_seed(len(lens))
    q = torch.randn(len(lens), nq, hd, device="cuda").to(dtype)
    plan = DecodePlan(pages, lens, kv, nq)
    assert tables[-1]["most_parts"] > parts
    w = torch.rand(kv.pages_total, nkv, block, device="cuda")
    w0 = w.clone()
    got = weighted_decode_attention(q, kv, 0, plan, w)
    want_w, tol_w = w0.double(), torch.zeros_like(w0, dtype=torch.float64)
    for i, (p, n) in enumerate(zip(pages, lens)):
        k, v = (_rows(pool, lay, p, n, 0, 1, x) for x in (False, True))
        o, tol, prob, rel = _attend(q[i], k, v, 1 / math.sqrt(hd), U[dtype])
        _within(got[i], o, tol)
        if n:
            s, at = prob.view(nkv, -1, n).sum(1), torch.arange(n)
            idx = (torch.tensor(p, dtype=torch.long)[at // block], slice(None), at % block)
            want_w[idx] += s.T
            tol_w[idx] = rel * s.T + 2.0 ** -23 * (w0[idx].double() + s.T)
    _within(w, want_w, tol_w)
    w2 = w0.clone()
    assert torch.equal(weighted_decode_attention(q, kv, 0, plan, w2), got) and torch.equal(w2, w)


@pytest.mark.parametrize("requests", [1, 6])       # the row kernel; tile units
def test_shared_prefix_of_many_parts(requests, tables):
    from kunserve_b200.ops import PrefixGroup, SharedPrefixPlan, shared_prefix_attention
    nq, nkv, hd, bs, n = 4, 1, 128, 16, 40000
    pool, kv, lay = _cache(n // bs + requests, bs, nkv, hd, BF)
    pages = _allot([n] + [5] * requests, bs, kv.pages_total, 2)
    for i, (p, m) in enumerate(zip(pages, [n] + [5] * requests)):
        _fill(pool, lay, p, m, 1, 1, i)
    q = torch.randn(requests, nq, hd, device="cuda").to(BF)
    plan = SharedPrefixPlan([PrefixGroup(pages[0], n, [(p, 5, 1) for p in pages[1:]])], kv, nq)
    assert tables[-1]["most_parts"] > (256 if requests == 1 else 32) and (tables[-1]["tile_units"] > 0) == (requests > 1)
    got = shared_prefix_attention(q, kv, 1, plan)
    kp, vp = (_rows(pool, lay, pages[0], n, 1, 1, x) for x in (False, True))
    for i in range(requests):
        k, v = (_rows(pool, lay, pages[1 + i], 5, 1, 1, x) for x in (False, True))
        o, tol, _, _ = _attend(q[i], torch.cat([kp, k]), torch.cat([vp, v]), 1 / math.sqrt(hd), U[BF])
        _within(got[i], o, tol)


# more than 256 vectors a token: several blocks take a token where tokens are
# few, several rounds of one block where they are many (296 and more)
@pytest.mark.parametrize("dtype,interleaved,rot", [(BF, False, 128), (FP, True, 128), (FP, False, 64), (BF, True, 96)])
@pytest.mark.parametrize("T", [3, 300])
def test_rotary_of_many_heads(dtype, interleaved, rot, T):
    from kunserve_b200.ops import Rotary, rotary_append, rotary_apply
    nq, nkv, hd, bs = 32, 8, 128, 16
    H = nq + 2 * nkv
    assert H * hd // 16 > 256
    torch.manual_seed(T)
    rotary, pos = Rotary(hd, rot, 500000.0, interleaved, LLAMA3), _positions(T, 1)
    x = torch.randn(T, H, hd, device="cuda").to(dtype)
    for inverse in (False, True):
        want, slack = _rotated(x, pos, rotary, inverse)
        _within(rotary_apply(x, pos, rotary, inverse=inverse), want, U[dtype] * want.abs() + slack + 2.0 ** -24)
    pool, kv, lay = _cache(-(-T // bs) + 1, bs, nkv, hd, dtype)
    spot = torch.randperm(kv.pages_total * bs, generator=torch.Generator().manual_seed(T))[:T]
    pages, slots = (spot // bs).int().cuda(), (spot % bs).int().cuda()
    qkv = x.clone()
    rotary_append(qkv, pos, pages, slots, rotary, kv, 1)
    want, slack = _rotated(x[:, :nq + nkv], pos, rotary)
    tol = U[dtype] * want.abs() + slack + 2.0 ** -24
    _within(qkv[:, :nq], want[:, :nq], tol[:, :nq])
    assert torch.equal(qkv[:, nq:], x[:, nq:])
    view = pool.view(kv.pages_total, 2, 2, bs, nkv, hd)    # page, layer, key or value
    assert lay.kv_offset(1, 1, 1, True) // 2 == view[1, 1, 1].storage_offset()
    k, v = (view[pages.long(), 1, i, slots.long()] for i in (0, 1))
    _within(k, want[:, nq:], tol[:, nq:])
    assert torch.equal(v, x[:, nq + nkv:])


@pytest.mark.parametrize("make", [_uniform, _few])
def test_select_of_rows_of_many_thousand_slots(make):
    """More than 4096 slots for each of a cluster's eight CTAs, kept in shared memory."""
    from kunserve_b200.ops import DecodePlan, select_evictions
    lens, keep, bs, nkv = [40001, 33000, 100], 20000, 64, 2
    assert 4096 < lens[0] / 8 < 40000
    pool, kv, _ = _cache(sum(-(-n // bs) for n in lens), bs, nkv, 8, BF, layers=1)
    pages = _allot(lens, bs, kv.pages_total, 1)
    g = torch.Generator().manual_seed(5)
    w = make((kv.pages_total, nkv, bs), g).cuda()
    pos = torch.randint(0, 40001, (kv.pages_total, nkv, bs), generator=g, dtype=torch.int32).cuda()
    moves, counts = select_evictions(w, pos, DecodePlan(pages, lens, kv, nkv), keep, 4, 500)
    for i, n in enumerate(lens):
        at = torch.arange(n)
        idx = (torch.tensor(pages[i])[at // bs], slice(None), at % bs)
        for h in range(nkv):
            x, p = w[idx][:, h].clone(), pos[idx][:, h]
            x[(p < 4) | (p > n - 1 - 500)] = math.inf
            left = min(n, keep)
            kept = torch.zeros(n, dtype=torch.bool, device="cuda")
            kept[x.sort(descending=True, stable=True).indices[:left]] = True
            dst, src = (~kept[:left]).nonzero().flatten(), left + kept[left:].nonzero().flatten()
            assert int(counts[i, h]) == len(dst)
            assert torch.equal(moves[i, h, :len(dst), 0].long(), dst)
            assert torch.equal(moves[i, h, :len(dst), 1].long(), src) and (moves[i, h, len(dst):] == -1).all()


@pytest.mark.parametrize("hd", [8, 80, 96])
def test_compaction_of_other_head_sizes(hd):
    _evict_case([70, 33, 200], 20, 2, 5, 3, 8, _uniform, hd=hd)
