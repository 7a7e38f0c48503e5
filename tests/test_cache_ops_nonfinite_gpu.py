"""NaN and infinite queries and keys of the cached-attention operators.

A row whose scores hold a NaN or +inf has no softmax: its outputs, and the
weights it adds, are NaN and not zeros.  A key of score -inf has weight zero;
rows without any other key give zeros.  Every other row is what it is without
the planted value.  Tolerances are those of finite rows (test_cache_ops_gpu).
"""
import math

import pytest
import torch

from test_cache_ops_gpu import BF, FP, U, _allot, _attend, _cache, _fill, _no_device_error, _rows, _within  # noqa: F401

pytestmark = pytest.mark.gpu

NQ, NKV, BS = 8, 2, 16
G = NQ // NKV


def _put(pool, lay, pages, key, head, dim, x):
    """One element of a key in layer 1."""
    o = lay.kv_offset(pages[key // BS], 1, 1, False) // 2
    pool[o + (key % BS * NKV + head) * lay.head_dim + dim] = x


def _check(got, rows, nan):
    """``rows``: (outputs, tolerance) of each token; ``nan`` [tokens, heads]: rows without a softmax."""
    for t, (o, tol) in enumerate(rows):
        assert got[t, nan[t]].isnan().all(), t
        _within(got[t, ~nan[t]], o[~nan[t]], tol[~nan[t]])


@pytest.mark.parametrize("hd,dtype", [(128, BF), (64, FP)])
@pytest.mark.parametrize("requests", [3, 24])      # 12 rows a prefix: the row kernel; 96: the tile kernel
@pytest.mark.parametrize("where", ["query", "infinite query", "first own key", "prefix key", "prefix block", "later own key"])
def test_shared_prefix_rows_without_a_softmax(where, requests, hd, dtype):
    from kunserve_b200.ops import PrefixGroup, SharedPrefixPlan, shared_prefix_attention
    prefix, own = 300, [1 + i % 3 for i in range(requests)]
    pool, kv, lay = _cache(60, BS, NKV, hd, dtype, poison=True)
    pages = _allot([prefix] + own, BS, kv.pages_total, 1)
    for i, (p, n) in enumerate(zip(pages, [prefix] + own)):
        _fill(pool, lay, p, n, 1, 1, 10 + i)
    torch.manual_seed(2)
    q = torch.randn(requests, NQ, hd, device="cuda").to(dtype)
    plan = SharedPrefixPlan([PrefixGroup(pages[0], prefix, [(p, n, 1) for p, n in zip(pages[1:], own)])], kv, NQ)
    assert (plan.num_q_heads, plan.tokens) == (NQ, requests)
    kp, vp = (_rows(pool, lay, pages[0], prefix, 1, 1, x) for x in (False, True))
    want = []
    for i, n in enumerate(own):
        k, v = (_rows(pool, lay, pages[1 + i], n, 1, 1, x) for x in (False, True))
        want.append(_attend(q[i], torch.cat([kp, k]), torch.cat([vp, v]), 1 / math.sqrt(hd), U[dtype])[:2])
    nan = torch.zeros(requests, NQ, dtype=torch.bool, device="cuda")
    if where == "query":
        q[1, 5, 3], nan[1, 5] = math.nan, True
    elif where == "infinite query":
        q[2, 0, 7], nan[2, 0] = math.inf, True       # scores of both signs: +inf among them
    elif where == "first own key":
        _put(pool, lay, pages[1], 0, 1, 9, math.nan)  # request 0 has no other own key
        nan[0, G:] = True
    elif where == "later own key":
        _put(pool, lay, pages[3], 2, 0, 0, math.nan)
        nan[2, :G] = True
    elif where == "prefix key":
        _put(pool, lay, pages[0], 130, 0, 1, math.nan)
        nan[:, :G] = True
    else:
        for key in range(128, 256):                  # all keys of one block of the tile kernel
            _put(pool, lay, pages[0], key, 1, 1, math.nan)
        nan[:, G:] = True
    got = shared_prefix_attention(q, kv, 1, plan)
    _check(got, want, nan)
    assert torch.equal(shared_prefix_attention(q, kv, 1, plan).isnan(), got.isnan())


@pytest.mark.parametrize("requests", [3, 24])
def test_shared_prefix_infinite_key(requests):
    """A key element of +inf: rows of positive queries there score +inf, rows of
    negative ones -inf, which is as if the key were not there."""
    from kunserve_b200.ops import PrefixGroup, SharedPrefixPlan, shared_prefix_attention
    hd, prefix = 64, 200
    pool, kv, lay = _cache(60, BS, NKV, hd, BF, poison=True)
    pages = _allot([prefix] + [2] * requests, BS, kv.pages_total, 4)
    for i, (p, n) in enumerate(zip(pages, [prefix] + [2] * requests)):
        _fill(pool, lay, p, n, 1, 1, 10 + i)
    torch.manual_seed(3)
    q = torch.randn(requests, NQ, hd, device="cuda").to(BF)
    plan = SharedPrefixPlan([PrefixGroup(pages[0], prefix, [(p, 2, 1) for p in pages[1:]])], kv, NQ)
    kp, vp = (_rows(pool, lay, pages[0], prefix, 1, 1, x) for x in (False, True))
    keep = torch.arange(prefix, device="cuda") != 77
    want = []
    for i in range(requests):
        k, v = (_rows(pool, lay, pages[1 + i], 2, 1, 1, x) for x in (False, True))
        with_, without = (_attend(q[i], torch.cat([kp[m], k]), torch.cat([vp[m], v]), 1 / math.sqrt(hd), U[BF])[:2]
                          for m in (slice(None), keep))
        head0 = (torch.arange(NQ, device="cuda") < G)[:, None]
        want.append(tuple(torch.where(head0, b, a) for a, b in zip(with_, without)))
    _put(pool, lay, pages[0], 77, 0, 5, math.inf)
    nan = (q[:, :, 5] > 0) & (torch.arange(NQ, device="cuda") < G)
    assert nan.any() and (q[:, :, 5] != 0).all()
    _check(shared_prefix_attention(q, kv, 1, plan), want, nan)


# 16 parts a row at most (weights beside the join), and more than 32 (weights behind it)
@pytest.mark.parametrize("n", [40, 600, 4000])
@pytest.mark.parametrize("where", ["query", "key", "infinite key"])
def test_weighted_rows_without_a_softmax(n, where):
    """Outputs and weights agree on which rows have no softmax."""
    from kunserve_b200.ops import DecodePlan, weighted_decode_attention
    hd = 64
    pool, kv, lay = _cache(-(-n // BS) + 3, BS, NKV, hd, BF, poison=True)
    pages = _allot([n, 20], BS, kv.pages_total, n)
    for i, m in enumerate((n, 20)):
        _fill(pool, lay, pages[i], m, 1, 1, i)
    torch.manual_seed(n)
    q = torch.randn(2, NQ, hd, device="cuda").to(BF)
    want = []
    for i, m in enumerate((n, 20)):
        k, v = (_rows(pool, lay, pages[i], m, 1, 1, x) for x in (False, True))
        want.append(_attend(q[i], k, v, 1 / math.sqrt(hd), U[BF]))
    nan = torch.zeros(2, NQ, dtype=torch.bool, device="cuda")
    if where == "query":
        q[0, 6, 0], nan[0, 6] = math.nan, True
    else:
        q[0, :G, 3] = 1.0 + torch.arange(G, device="cuda").to(BF)
        _put(pool, lay, pages[0], n - 7, 0, 3, math.nan if where == "key" else math.inf)
        nan[0, :G] = True
    w = torch.zeros(kv.pages_total, NKV, BS, device="cuda")
    got = weighted_decode_attention(q, kv, 1, DecodePlan(pages, [n, 20], kv, NQ), w)
    _check(got, [x[:2] for x in want], nan)
    for i, m in enumerate((n, 20)):
        added = w[pages[i]].transpose(0, 1).reshape(NKV, -1)[:, :m]
        lost = nan[i].view(NKV, G).any(1)
        p = want[i][2].view(NKV, G, m).sum(1)
        assert added[lost].isnan().all()
        _within(added[~lost], p[~lost], (want[i][3] + 2.0 ** -23) * p[~lost])


@pytest.mark.parametrize("n", [5, 3000])
def test_all_scores_minus_infinity(n):
    """No key of finite score: zeros, and no weight is added."""
    from kunserve_b200.ops import DecodePlan, weighted_decode_attention
    hd = 64
    pool, kv, lay = _cache(-(-n // BS) + 1, BS, NKV, hd, BF, poison=True)
    pages = _allot([n], BS, kv.pages_total, 1)
    _fill(pool, lay, pages[0], n, 1, 1, 0)
    for page in pages[0]:
        o = lay.kv_offset(page, 1, 1, False) // 2
        pool[o:o + BS * NKV * hd].view(BS, NKV, hd)[:, 0, 2] = -math.inf
    q = torch.rand(1, NQ, hd, device="cuda").to(BF) + 1.0
    w = torch.ones(kv.pages_total, NKV, BS, device="cuda")
    got = weighted_decode_attention(q, kv, 1, DecodePlan(pages, [n], kv, NQ), w)
    assert (got[0, :G] == 0).all() and torch.isfinite(got.float()).all()
    assert (w[:, 0] == 1).all() and torch.isfinite(w).all()
