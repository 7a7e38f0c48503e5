"""Long-context cache operators against plain 64-bit forms.

Tolerances.  u = half a unit in the last place of the output type, relative:
2^-8 (bf16), 2^-11 (fp16).  A rotated element is rounded once: u |y| plus
fp32 arithmetic on (a, b).  An attention output is rounded once, and the
kernels may round the probabilities to the cache's type before they meet the
values: u |y| + u sum p |v|, plus the score error d below on every p.  Scores
are fp32 sums of exact products: their error is at most d = hd 2^-23 scale
sum |q k|, and a probability's relative error 2 d plus a few fp32 units.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
BF, FP = torch.bfloat16, torch.float16


@pytest.fixture(autouse=True)
def _no_device_error():
    from kunserve_b200.ops import check_error
    check_error()
    yield
    torch.cuda.synchronize()
    check_error()


def _cache(pages, block, nkv, hd, dtype, layers=2, fusion=1, extend=0, seed=0, poison=False):
    """A filled pool, its handle and layout; with ``poison`` every slot starts as NaN."""
    from kunserve_b200.kv.layout import KVLayout
    from kunserve_b200.ops import PagedKV

    lay = KVLayout(pages, layers, block, nkv, hd, 2)
    n = (lay.base_bytes + extend * lay.extend_page_bytes(fusion)) // 2
    g = torch.Generator(device="cuda").manual_seed(seed)
    pool = torch.randn(n, generator=g, device="cuda").to(dtype)
    if poison:
        pool.fill_(math.nan)
    return pool, PagedKV(pool, lay, fusion), lay


def _rows(pool, lay, pages, n, layer, fusion, value):
    """Views are built from the layout's own offsets: [n, nkv, hd]."""
    bs, per = lay.block_size, lay.num_kv_heads * lay.head_dim
    got = []
    for i in range(-(-n // bs) if n else 0):
        o = lay.kv_offset(pages[i], layer, fusion, value) // 2
        got.append(pool[o:o + bs * per].view(bs, lay.num_kv_heads, lay.head_dim))
    return torch.cat(got)[:n] if got else pool.new_zeros(0, lay.num_kv_heads, lay.head_dim)


def _fill(pool, lay, pages, n, layer, fusion, seed, ramp=False):
    """Random keys and values in the first n slots behind a page list; with
    ``ramp`` the keys grow along the list."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    bs, per = lay.block_size, lay.num_kv_heads * lay.head_dim
    for value in (False, True):
        x = torch.randn(n, per, generator=g, device="cuda")
        if ramp and not value:
            x *= torch.linspace(0.2, 8.0, n, device="cuda")[:, None]
        x = x.to(pool.dtype)
        for i in range(-(-n // bs) if n else 0):
            o = lay.kv_offset(pages[i], layer, fusion, value) // 2
            part = x[i * bs:(i + 1) * bs]
            pool[o:o + part.numel()] = part.reshape(-1)


def _attend(q, k, v, scale, u):
    """64-bit attention of q [nq, hd] over k, v [n, nkv, hd]: outputs, tolerance,
    probabilities [nq, n] and their relative tolerance."""
    nq, hd = q.shape
    G = nq // k.shape[1]
    q, k, v = q.double(), k.double().repeat_interleave(G, 1), v.double().repeat_interleave(G, 1)
    if k.shape[0] == 0:
        z = torch.zeros_like(q)
        return z, z, q.new_zeros(nq, 0), 0.0
    s = scale * torch.einsum("hd,nhd->hn", q, k)
    d = hd * 2.0 ** -23 * scale * torch.einsum("hd,nhd->hn", q.abs(), k.abs()).max().item()
    p = torch.softmax(s, -1)
    o, a = torch.einsum("hn,nhd->hd", p, v), torch.einsum("hn,nhd->hd", p, v.abs())
    rel = 2 * d + 2.0 ** -20
    return o, u * o.abs() + (u + rel) * a + 2.0 ** -24, p, rel


def _within(got, want, tol):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), (int(bad.sum()), err[bad].max().item(), got.shape)


# ------------------------------------------------------------------- rotary
def _rotated(x, positions, rotary, inverse=False):
    """64-bit rotation, and the fp32 part of its tolerance."""
    f = rotary.frequencies.to(x.device)
    ang = positions.double()[:, None] * f
    c, s = (ang.cos() * rotary.scale)[:, None], (ang.sin() * rotary.scale * (-1 if inverse else 1))[:, None]
    y, r = x.double().clone(), rotary.rotary_dim
    i = torch.arange(r // 2, device=x.device)
    a, b = (2 * i, 2 * i + 1) if rotary.interleaved else (i, i + r // 2)
    xa, xb = y[..., a].clone(), y[..., b].clone()
    y[..., a], y[..., b] = xa * c - xb * s, xb * c + xa * s
    slack = torch.zeros_like(y)
    # the 64-bit angle itself is off by 2^-53 of its size
    off = (2.0 ** -20 + ang.abs()[:, None] * 2.0 ** -52) * rotary.scale * (xa.abs() + xb.abs())
    slack[..., a], slack[..., b] = off, off
    return y, slack


LLAMA3 = dict(rope_type="llama3", factor=8.0, low_freq_factor=1.0, high_freq_factor=4.0,
              original_max_position_embeddings=8192)
YARN = dict(rope_type="yarn", factor=16.0, original_max_position_embeddings=4096)


def _positions(T, seed):
    g = torch.Generator().manual_seed(seed)
    p = torch.randint(0, 1 << 20, (T,), generator=g, dtype=torch.int32)
    for i, v in enumerate((0, 1, 131071, -5, (1 << 31) - 1)):
        if i < T:
            p[i] = v
    return p.cuda()


@pytest.mark.parametrize("dtype", [BF, FP])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("T,H,hd,rot,scaling", [(1, 1, 128, 128, None), (7, 5, 128, 64, LLAMA3), (300, 3, 64, 48, YARN),
                                                (6, 3, 64, 2, None), (5, 2, 128, 24, dict(type="linear", factor=4.0)),
                                                (33, 9, 96, 96, None), (9, 1, 80, 32, None), (4, 2, 10, 6, None)])
def test_rotary_apply(dtype, interleaved, T, H, hd, rot, scaling):
    from kunserve_b200.ops import Rotary, rotary_apply
    torch.manual_seed(T)
    rotary = Rotary(hd, rot, 500000.0, interleaved, scaling)
    pos = _positions(T, 1)
    # plain, a strided view, a view off the 16-byte grid, in place
    wide = torch.randn(T, H + 3, hd, device="cuda").to(dtype)
    odd = torch.randn(T * H * hd + 1, device="cuda").to(dtype)[1:].view(T, H, hd)
    for x in (wide[:, :H].contiguous(), wide[:, 1:H + 1], odd, wide.transpose(0, 1).contiguous().transpose(0, 1)[:, :H]):
        for inverse in (False, True):
            want, slack = _rotated(x, pos, rotary, inverse)
            tol = U[dtype] * want.abs() + slack + 2.0 ** -24
            _within(rotary_apply(x, pos, rotary, inverse=inverse), want, tol)
            out = torch.full((T, H, 2 * hd), 7.0, device="cuda", dtype=dtype)
            rotary_apply(x, pos, rotary, out=out[..., :hd], inverse=inverse)
            _within(out[..., :hd], want, tol)
            assert (out[..., hd:] == 7).all()
    want, slack = _rotated(odd, pos, rotary)
    assert rotary_apply(odd, pos, rotary, out=odd) is odd
    _within(odd, want, U[dtype] * want.abs() + slack + 2.0 ** -24)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_gradient(interleaved):
    """The inverse with the factor kept is the transposed map: against the
    formula's own gradient, and against differences of the operator."""
    from kunserve_b200.ops import Rotary, rotary_apply
    torch.manual_seed(0)
    rotary = Rotary(64, 32, 10000.0, interleaved, YARN)
    T, H = 3, 2
    pos = torch.tensor([3, 70000, 0], dtype=torch.int32, device="cuda")
    x = torch.randn(T, H, 64, device="cuda").half()
    g = torch.randn(T, H, 64, device="cuda").half()
    got = rotary_apply(g, pos, rotary, inverse=True)
    xd = x.double().requires_grad_()
    f = rotary.frequencies.cuda()
    ang = pos.double()[:, None] * f
    c, s = (ang.cos() * rotary.scale)[:, None], (ang.sin() * rotary.scale)[:, None]
    i = torch.arange(16, device="cuda")
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + 16)
    y = torch.cat([xd[..., a] * c - xd[..., b] * s, xd[..., b] * c + xd[..., a] * s, xd[..., 32:]], -1)
    gg = torch.cat([g.double()[..., a], g.double()[..., b], g.double()[..., 32:]], -1)
    (y * gg).sum().backward()
    _within(got, xd.grad, U[FP] * xd.grad.abs() + 2.0 ** -18 * rotary.scale * 8)
    # differences: the map is linear, so a step of 1 in one element is exact up
    # to the two results' rounding
    y0 = rotary_apply(x, pos, rotary)
    for t, h, d in ((0, 0, 0), (1, 1, 5), (2, 0, 31), (1, 0, 40)):
        x1 = x.clone()
        x1[t, h, d] += 1
        step = (x1[t, h, d] - x[t, h, d]).double()
        y1 = rotary_apply(x1, pos, rotary)
        diff = ((y1.double() - y0.double()) * g.double()).sum() / step
        tol = (U[FP] * (y1.double().abs() + y0.double().abs() + 2.0 ** -9) * g.double().abs())[t, h].sum() + \
            U[FP] * got[t, h, d].double().abs()
        assert (diff - got[t, h, d].double()).abs() <= tol * 1.01


@pytest.mark.parametrize("dtype,interleaved,hd,rot,nq,nkv", [(BF, False, 128, 128, 8, 2), (FP, True, 64, 32, 3, 3),
                                                             (BF, True, 128, 96, 4, 1), (FP, False, 64, 20, 5, 1)])
@pytest.mark.parametrize("fusion,extend", [(1, 0), (2, 3)])
@pytest.mark.parametrize("T", [1, 40, 400])
def test_rotary_append(dtype, interleaved, hd, rot, nq, nkv, fusion, extend, T):
    from kunserve_b200.ops import Rotary, rotary_append
    bs, P = 16, 40
    pool, kv, lay = _cache(P, bs, nkv, hd, dtype, layers=4, fusion=fusion, extend=extend)
    assert kv.pages_total == fusion * P + extend
    before = pool.clone()
    g = torch.Generator().manual_seed(T)
    spot = torch.randperm(kv.pages_total * bs, generator=g)[:T]
    if T == 400 and extend:
        spot[-1] = kv.pages_total * bs - 1 if (kv.pages_total * bs - 1) not in spot else spot[-1]
    pages, slots = (spot // bs).int().cuda(), (spot % bs).int().cuda()
    rotary = Rotary(hd, rot, 10000.0, interleaved, LLAMA3)
    pos = _positions(T, 2)
    qkv = torch.randn(T, nq + 2 * nkv, hd, device="cuda").to(dtype)
    orig = qkv.clone()
    layer = 4 // fusion - 1
    w = torch.rand(kv.pages_total, nkv, bs, device="cuda")
    sp = torch.full((kv.pages_total, nkv, bs), -1, dtype=torch.int32, device="cuda")
    w0 = w.clone()
    rotary_append(qkv, pos, pages, slots, rotary, kv, layer, weights=w, slot_positions=sp)
    y, slack = _rotated(orig[:, :nq + nkv], pos, rotary)
    tol = U[dtype] * y.abs() + slack + 2.0 ** -24
    _within(qkv[:, :nq], y[:, :nq], tol[:, :nq])
    assert torch.equal(qkv[:, nq:], orig[:, nq:])
    touched = torch.zeros_like(pool, dtype=torch.bool)
    for t in range(T):
        for value in (False, True):
            o = lay.kv_offset(int(pages[t]), layer, fusion, value) // 2 + int(slots[t]) * nkv * hd
            got = pool[o:o + nkv * hd].view(nkv, hd)
            touched[o:o + nkv * hd] = True
            if value:
                assert torch.equal(got, orig[t, nq + nkv:])
            else:
                _within(got, y[t, nq:], tol[t, nq:])
    assert torch.equal(pool[~touched], before[~touched])
    pl, sl = pages.long(), slots.long()
    assert (w[pl, :, sl] == 0).all() and (sp[pl, :, sl] == pos[:, None]).all()
    w0[pl, :, sl] = 0
    assert torch.equal(w, w0) and int((sp != -1).sum()) <= T * nkv
    # out of place leaves qkv alone
    q2, out = orig.clone(), torch.empty(T, nq, hd, device="cuda", dtype=dtype)
    rotary_append(q2, pos, pages, slots, rotary, kv, layer, out=out)
    assert torch.equal(q2, orig) and torch.equal(out, qkv[:, :nq])


def test_rotary_append_drops_bad_rows():
    """A page or slot outside the cache is reported and not written; the rest is."""
    from kunserve_b200.ops import Rotary, check_error, rotary_append
    pool, kv, lay = _cache(3, 8, 2, 64, BF)
    before = pool.clone()
    qkv = torch.randn(4, 6, 64, device="cuda").to(BF)
    pages = torch.tensor([3, -1, 1, 2], dtype=torch.int32, device="cuda")
    slots = torch.tensor([0, 0, 8, 5], dtype=torch.int32, device="cuda")
    rotary_append(qkv, torch.arange(4, dtype=torch.int32, device="cuda"), pages, slots, Rotary(64), kv, 1)
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_error()
    changed = (pool != before).nonzero().flatten()
    for value in (False, True):
        o = lay.kv_offset(2, 1, 1, value) // 2 + 5 * 2 * 64
        inside = (changed >= o) & (changed < o + 128)
        assert inside.any()
        changed = changed[~inside]
    assert changed.numel() == 0


# -------------------------------------------------- shared-prefix attention
def _allot(lens, block, total, seed):
    """Distinct random pages for each length."""
    order = torch.randperm(total, generator=torch.Generator().manual_seed(seed)).tolist()
    out, at = [], 0
    for n in lens:
        k = -(-n // block)
        out.append(order[at:at + k])
        at += k
    assert at <= total
    return out


def _shared_case(groups, nq, nkv, hd, dtype, block, fusion=1, extend=0, amp=1.0, strided=False, seed=0,
                 ramp=False):
    """groups: [(prefix length, [(own tokens, queries), ...]), ...].  Runs the
    operator on a cache whose every other slot is NaN and checks every row."""
    from kunserve_b200.ops import PrefixGroup, SharedPrefixPlan, shared_prefix_attention
    lens = [n for p, reqs in groups for n in [p] + [o for o, _ in reqs]]
    total = sum(-(-n // block) for n in lens) + 2
    base = total if fusion == 1 else max(1, -(-(total - extend) // fusion))
    pool, kv, lay = _cache(base, block, nkv, hd, dtype, layers=2 * fusion, fusion=fusion, extend=extend, poison=True)
    pages = _allot(lens, block, kv.pages_total, seed)
    layer = 1
    for i, (p, n) in enumerate(zip(pages, lens)):
        _fill(pool, lay, p, n, layer, fusion, 100 + i, ramp)
    it = iter(pages)
    plan_groups = []
    for p, reqs in groups:
        pre = next(it)
        plan_groups.append(PrefixGroup(pre, p, [(next(it), o, n) for o, n in reqs]))
    T = sum(n for _, reqs in groups for _, n in reqs)
    torch.manual_seed(seed)
    q = (torch.randn(T, nq, hd, device="cuda") * amp).to(dtype)
    if strided:
        wide = torch.zeros(T, nq + 4, hd, device="cuda", dtype=dtype)
        wide[:, 2:2 + nq] = q
        q = wide[:, 2:2 + nq]
    plan = SharedPrefixPlan(plan_groups, kv, nq)
    assert plan.tokens == T
    scale = 1.0 / math.sqrt(hd)
    got = shared_prefix_attention(q, kv, layer, plan)
    assert got.shape == (T, nq, hd) and got.dtype == dtype
    t = 0
    for g in plan_groups:
        pk, pv = (_rows(pool, lay, g.pages, g.length, layer, fusion, x) for x in (False, True))
        for own, n, m in g.requests:
            ok, ov = (_rows(pool, lay, own, n, layer, fusion, x) for x in (False, True))
            for j in range(m):
                seen = n - m + j + 1
                o, tol, _, _ = _attend(q[t], torch.cat([pk, ok[:seen]]), torch.cat([pv, ov[:seen]]), scale, U[dtype])
                _within(got[t], o, tol)
                t += 1
    again = shared_prefix_attention(q, kv, layer, plan, scale, out=torch.empty_like(got))
    assert torch.equal(again, got), "the join order is fixed: a repeat gives the same bits"
    return got


ODD = [(37, [(1, 1), (5, 2), (16, 0)]), (0, [(3, 3), (40, 1)]), (200, [(17, 1)])]


@pytest.mark.parametrize("nq,nkv", [(4, 4), (6, 2), (8, 2), (8, 1), (16, 1), (20, 1), (40, 1), (14, 2)])
@pytest.mark.parametrize("hd,dtype", [(128, BF), (64, FP)])
def test_shared_prefix_heads(nq, nkv, hd, dtype):
    _shared_case(ODD, nq, nkv, hd, dtype, 16)


@pytest.mark.parametrize("block", [1, 5, 8, 24, 64, 128])
def test_shared_prefix_page_sizes(block):
    _shared_case(ODD + [(130, [(66, 1), (2, 1)])], 8, 2, 128, BF, block, seed=block)


@pytest.mark.parametrize("prefix", [1, 15, 16, 17, 63, 64, 65, 1023, 2500])
@pytest.mark.parametrize("requests", [1, 3, 9, 40])
def test_shared_prefix_lengths(prefix, requests):
    _shared_case([(prefix, [(1 + i % 5, 1) for i in range(requests)])], 8, 2, 128, BF if prefix % 2 else FP, 16)


@pytest.mark.parametrize("queries", [2, 16, 33, 90])
def test_shared_prefix_query_chunks(queries):
    """Chunks of query tokens: causal among the request's own tokens."""
    _shared_case([(100, [(queries, queries), (queries + 70, queries)]), (65, [(queries + 1, queries)])], 8, 2, 64, BF,
                 16)


def test_shared_prefix_fused_page_ids():
    _shared_case(ODD, 8, 2, 128, BF, 16, fusion=2, extend=4)
    _shared_case([(300, [(1 + i, 1) for i in range(9)])], 8, 2, 64, FP, 16, fusion=2, extend=9)   # the tile kernel


@pytest.mark.parametrize("hd,dtype", [(128, BF), (64, FP)])
def test_shared_prefix_growing_scores(hd, dtype):
    """Each block of keys outgrows the maxima of the ones before, in both kernels."""
    _shared_case([(1000, [(5, 1)] * 12), (900, [(150, 1)])], 8, 2, hd, dtype, 16, amp=4.0, ramp=True)


def test_shared_prefix_many_units():
    """More tile units than SMs: each CTA takes several, of ragged ends."""
    _shared_case([(650 + 17 * i, [(1 + j % 3, 1) for j in range(6)]) for i in range(12)], 32, 8, 128, FP, 16)
    _shared_case([(130 + 61 * i, [(2, 1 + j % 2) for j in range(20)]) for i in range(25)], 8, 8, 64, BF, 8, amp=3.0)


@pytest.mark.parametrize("amp", [0.0, 30.0])
def test_shared_prefix_flat_and_peaked(amp):
    """Equal scores, and scores of several hundred."""
    _shared_case([(300, [(20, 1)] * 20), (7, [(1, 1)])], 8, 2, 128, FP, 16, amp=amp)


def test_shared_prefix_strided_queries_and_empty():
    from kunserve_b200.ops import PrefixGroup, SharedPrefixPlan, shared_prefix_attention
    _shared_case(ODD, 8, 2, 128, BF, 16, strided=True)
    pool, kv, _ = _cache(4, 16, 2, 128, BF)
    empty = torch.empty(0, 4, 128, device="cuda", dtype=BF)
    for groups in ([], [PrefixGroup([0], 5, [])], [PrefixGroup([0], 5, [([1], 3, 0)])]):
        plan = SharedPrefixPlan(groups, kv, 4)
        assert shared_prefix_attention(empty, kv, 0, plan).shape == (0, 4, 128)


def test_attention_across_32_bit_offsets():
    """Pages past 2^31 elements of a large pool."""
    from kunserve_b200.kv.layout import KVLayout
    from kunserve_b200.ops import DecodePlan, PagedKV, weighted_decode_attention
    nkv, hd, bs = 8, 128, 16
    lay = KVLayout(70000, 1, bs, nkv, hd, 2)
    pool = torch.empty(lay.base_bytes // 2, device="cuda", dtype=BF)
    assert pool.numel() > 1 << 31
    kv = PagedKV(pool, lay)
    pages, n = [69999, 65536, 65535, 3], 50
    _fill(pool, lay, pages, n, 0, 1, 5)
    q = torch.randn(1, 16, hd, device="cuda").to(BF)
    w = torch.zeros(kv.pages_total, nkv, bs, device="cuda")
    got = weighted_decode_attention(q, kv, 0, DecodePlan([pages], [n], kv, 16), w)
    k, v = (_rows(pool, lay, pages, n, 0, 1, x) for x in (False, True))
    o, tol, p, rel = _attend(q[0], k, v, 1 / math.sqrt(hd), U[BF])
    _within(got[0], o, tol)
    want = p.view(nkv, 2, n).sum(1)
    _within(w[pages].transpose(0, 1).reshape(nkv, -1)[:, :n], want, rel * want)
    # the same pages as a prefix of 15 requests: 30 rows, the tile kernel
    from kunserve_b200.ops import PrefixGroup, SharedPrefixPlan, shared_prefix_attention
    own = [68000 + i for i in range(15)]
    for i, page in enumerate(own):
        _fill(pool, lay, [page], 3, 0, 1, 50 + i)
    q = torch.randn(15, 16, hd, device="cuda").to(BF)
    plan = SharedPrefixPlan([PrefixGroup(pages, n, [([page], 3, 1) for page in own])], kv, 16)
    got = shared_prefix_attention(q, kv, 0, plan)
    for i, page in enumerate(own):
        ok, ov = (_rows(pool, lay, [page], 3, 0, 1, x) for x in (False, True))
        o, tol, _, _ = _attend(q[i], torch.cat([k, ok]), torch.cat([v, ov]), 1 / math.sqrt(hd), U[BF])
        _within(got[i], o, tol)


# ------------------------------------------------ weighted decode attention
@pytest.mark.parametrize("nq,nkv,hd,dtype", [(4, 2, 64, BF), (8, 1, 128, FP), (5, 5, 128, BF), (40, 2, 64, FP)])
@pytest.mark.parametrize("block", [16, 5, 64])
def test_weighted_decode(nq, nkv, hd, dtype, block):
    from kunserve_b200.ops import DecodePlan, weighted_decode_attention
    lens = [1, 0, 15, 16, 17, 511, 512, 513, 1300, 64]
    pool, kv, lay = _cache(sum(-(-n // block) for n in lens) + 1, block, nkv, hd, dtype, poison=True)
    pages = _allot(lens, block, kv.pages_total, 3)
    for i, (p, n) in enumerate(zip(pages, lens)):
        _fill(pool, lay, p, n, 0, 1, i)
    q = torch.randn(len(lens), nq, hd, device="cuda").to(dtype)
    plan = DecodePlan(pages, lens, kv, nq)
    w = torch.rand(kv.pages_total, nkv, block, device="cuda")
    w0 = w.clone()
    got = weighted_decode_attention(q, kv, 0, plan, w)
    want_w, tol_w = w0.double(), torch.zeros_like(w0, dtype=torch.float64)
    for i, (p, n) in enumerate(zip(pages, lens)):
        k, v = (_rows(pool, lay, p, n, 0, 1, x) for x in (False, True))
        o, tol, prob, rel = _attend(q[i], k, v, 1 / math.sqrt(hd), U[dtype])
        _within(got[i], o, tol)
        s = prob.view(nkv, -1, n).sum(1) if n else prob.new_zeros(nkv, 0)
        at = torch.arange(n)
        idx = (torch.tensor(p, dtype=torch.long)[at // block], slice(None), at % block) if n else None
        if n:
            want_w[idx] += s.T
            tol_w[idx] = rel * s.T + 2.0 ** -23 * (w0[idx].double() + s.T)
            gain = (w[idx].double() - w0[idx].double()).sum(0)
            assert (gain - nq // nkv).abs().max() <= n * 2.0 ** -22 + rel * nq
    _within(w, want_w, tol_w)
    w2 = w0.clone()
    assert torch.equal(weighted_decode_attention(q, kv, 0, plan, w2), got) and torch.equal(w2, w)


def test_weighted_decode_on_another_stream():
    from kunserve_b200.ops import DecodePlan, weighted_decode_attention
    pool, kv, lay = _cache(80, 16, 2, 128, BF)
    q = torch.randn(1, 4, 128, device="cuda").to(BF)
    pages = list(range(70))
    want_w, got_w = (torch.zeros(kv.pages_total, 2, 16, device="cuda") for _ in range(2))
    want = weighted_decode_attention(q, kv, 1, DecodePlan([pages], [1111], kv, 4), want_w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = weighted_decode_attention(q, kv, 1, DecodePlan([pages], [1111], kv, 4), got_w)
        for _ in range(20):   # the plans above are freed while the stream still runs
            weighted_decode_attention(q, kv, 1, DecodePlan([pages], [900], kv, 4), torch.zeros_like(got_w))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and torch.equal(got_w, want_w)


# ----------------------------------------------------------------- eviction
def _evict_case(lens, keep, sinks, recent, nkv, block, make, seed=0, hd=64, fusion=1, newest=None):
    """Select and compact against a plain sort; ``make(shape)`` gives weights."""
    from kunserve_b200.ops import DecodePlan, compact_cache, select_evictions
    total = sum(-(-n // block) for n in lens) + 1
    pool, kv, lay = _cache(-(-total // fusion), block, nkv, hd, BF, layers=2 * fusion, fusion=fusion, seed=seed)
    pages = _allot(lens, block, kv.pages_total, seed)
    g = torch.Generator().manual_seed(seed)
    w = make((kv.pages_total, nkv, block), g)
    pos = torch.zeros(kv.pages_total, nkv, block, dtype=torch.int32)
    table = []
    for p, n in zip(pages, lens):
        at = torch.arange(n)
        table.append((torch.tensor(p, dtype=torch.long)[at // block], at % block))
        pg, sl = table[-1]
        for h in range(nkv):
            pos[pg, h, sl] = torch.randperm(n, generator=g).int()
    newest = newest if newest is not None else [n - 1 for n in lens]
    w, pos = w.cuda(), pos.cuda()
    w0, p0, pool0 = w.clone(), pos.clone(), pool.clone()
    plan = DecodePlan(pages, lens, kv, nkv, newest)
    moves, counts = select_evictions(w, pos, plan, keep, sinks, recent)
    assert torch.equal(w, w0) or w0.isnan().any()
    compact_cache(kv, 1, plan, moves, counts, w, pos)
    cap = max([min(keep, n - keep) for n in lens] + [0])
    assert moves.shape == (len(lens), nkv, cap, 2)
    want_pool, want_w, want_p = pool0.clone(), w0.clone(), p0.clone()
    for i, n in enumerate(lens):
        pg, sl = table[i]
        left = min(n, keep)
        for h in range(nkv):
            x, q = w0[pg, h, sl].cpu().double(), p0[pg, h, sl].cpu()
            x = torch.where(x.isnan(), -math.inf, x) + 0.0
            rank = torch.zeros(n, 3, dtype=torch.float64)
            rank[:, 0] = ((q < sinks) | (q > newest[i] - recent)).double()       # protected first
            rank[:, 1] = 1.0 - w0[pg, h, sl].cpu().isnan().double() * (1 - rank[:, 0])   # NaN last
            rank[:, 2] = torch.where(rank[:, 0] > 0, 0.0, x)
            order = sorted(range(n), key=lambda j: (-rank[j, 0].item(), -rank[j, 1].item(), -rank[j, 2].item(), j))
            kept = torch.zeros(n, dtype=torch.bool)
            kept[order[:left]] = True
            dst, src = (~kept[:left]).nonzero().flatten(), left + kept[left:].nonzero().flatten()
            assert int(counts[i, h]) == len(dst)
            got = moves[i, h].cpu()
            assert torch.equal(got[:len(dst), 0].long(), dst) and torch.equal(got[:len(dst), 1].long(), src)
            assert (got[len(dst):] == -1).all()
            for a, b in zip(dst.tolist(), src.tolist()):
                for value in (False, True):
                    o1, o2 = ((lay.kv_offset(int(pg[j]), 1, fusion, value) // 2 + (int(sl[j]) * nkv + h) * hd)
                              for j in (a, b))
                    want_pool[o1:o1 + hd] = pool0[o2:o2 + hd]
                want_w[pg[a], h, sl[a]], want_p[pg[a], h, sl[a]] = w0[pg[b], h, sl[b]], p0[pg[b], h, sl[b]]
    assert torch.equal(pool, want_pool) and torch.equal(pos, want_p)
    assert torch.equal(w.nan_to_num(-9), want_w.nan_to_num(-9))


def _uniform(shape, g):
    return torch.rand(shape, generator=g)


def _few(shape, g):
    return torch.randint(0, 3, shape, generator=g).float()


def _strange(shape, g):
    vals = torch.tensor([0.0, -0.0, math.nan, math.inf, -math.inf, 1e-45, -1e-45, 1.0, -2.0, 3.4e38])
    return vals[torch.randint(0, len(vals), shape, generator=g)]


@pytest.mark.parametrize("make", [_uniform, _few, _strange, lambda s, g: torch.ones(s)])
@pytest.mark.parametrize("lens,keep,sinks,recent", [([40, 7, 33, 0, 32, 200], 32, 4, 8), ([65], 64, 0, 0),
                                                    ([300, 299], 1, 0, 1), ([1000, 31, 513], 500, 0, 500),
                                                    ([130, 129], 129, 100, 29)])
def test_evict(make, lens, keep, sinks, recent):
    _evict_case(lens, keep, sinks, recent, 2, 16, make)


@pytest.mark.parametrize("lens,keep", [([9001], 3000), ([5000, 20, 4097], 4096), ([12000], 11999)])
@pytest.mark.parametrize("make", [_uniform, _few])
def test_evict_long_rows(lens, keep, make):
    """Rows cut over the CTAs of a cluster, ties across their borders."""
    _evict_case(lens, keep, 4, 100, 1, 64, make, hd=64)


def test_evict_layouts():
    _evict_case([70, 33], 20, 2, 5, 3, 5, _uniform, hd=128)
    _evict_case([70, 33], 20, 2, 5, 2, 8, _uniform, fusion=2)
    # newest positions ahead of the slots: earlier evictions
    _evict_case([70, 33], 20, 2, 5, 2, 8, _uniform, newest=[68, 40])


def test_evict_very_long_row_matches_sort():
    """A row too long for the shared memory of its cluster."""
    from kunserve_b200.ops import DecodePlan, select_evictions
    n, keep, bs = 420001, 100003, 64
    pool, kv, _ = _cache(-(-n // bs), bs, 1, 8, BF, layers=1)
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.rand(kv.pages_total, 1, bs, generator=g, device="cuda")
    pos = torch.arange(kv.pages_total * bs, device="cuda", dtype=torch.int32).view_as(w)
    plan = DecodePlan([list(range(kv.pages_total))], [n], kv, 1)
    moves, counts = select_evictions(w, pos, plan, keep, 5, 1000)
    x = w.flatten()[:n].clone()
    x[:5], x[n - 1000:] = math.inf, math.inf
    kept = torch.zeros(n, dtype=torch.bool, device="cuda")
    kept[x.sort(descending=True, stable=True).indices[:keep]] = True
    dst, src = (~kept[:keep]).nonzero().flatten(), keep + kept[keep:].nonzero().flatten()
    assert int(counts) == len(dst)
    assert torch.equal(moves[0, 0, :len(dst), 0].long(), dst) and torch.equal(moves[0, 0, :len(dst), 1].long(), src)


def test_compact_reports_bad_moves():
    """Moves outside a request are reported and not made."""
    from kunserve_b200.ops import DecodePlan, check_error, compact_cache
    pool, kv, _ = _cache(4, 16, 1, 64, BF)
    before = pool.clone()
    plan = DecodePlan([[0, 1]], [20], kv, 1)
    moves = torch.tensor([[[[3, 20], [-1, 4]]]], dtype=torch.int32, device="cuda")
    compact_cache(kv, 0, plan, moves, torch.full((1, 1), 2, dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    with pytest.raises(RuntimeError, match="out of bounds"):
        check_error()
    assert torch.equal(pool, before)


def test_evicted_cache_attends_to_what_is_kept():
    """Attention over the compacted slots equals attention over the kept tokens."""
    from kunserve_b200.ops import DecodePlan, compact_cache, select_evictions, weighted_decode_attention
    nq, nkv, hd, bs, n, keep = 8, 2, 128, 16, 300, 100
    pool, kv, lay = _cache(20, bs, nkv, hd, BF)
    pages = list(range(1, 20))
    q = torch.randn(1, nq, hd, device="cuda").to(BF)
    w = torch.zeros(kv.pages_total, nkv, bs, device="cuda")
    pos = torch.zeros(kv.pages_total, nkv, bs, dtype=torch.int32, device="cuda")
    pos[pages] = torch.arange(19 * bs, dtype=torch.int32, device="cuda").view(19, 1, bs)
    plan = DecodePlan([pages], [n], kv, nq)
    weighted_decode_attention(q, kv, 0, plan, w)
    k, v = (_rows(pool, lay, pages, n, 0, 1, x).clone() for x in (False, True))
    score = w[pages].transpose(0, 1).reshape(nkv, -1)[:, :n].clone()
    moves, counts = select_evictions(w, pos, plan, keep, 4, 16)
    compact_cache(kv, 0, plan, moves, counts, w, pos)
    got = weighted_decode_attention(q, kv, 0, DecodePlan([pages], [keep], kv, nq, newest=[n - 1]), w)
    for h in range(nkv):
        s = score[h].clone()
        s[:4], s[n - 16:] = math.inf, math.inf
        kept = s.topk(keep).indices
        o, tol, _, _ = _attend(q[0, 4 * h:4 * h + 4], k[kept, h:h + 1], v[kept, h:h + 1], 1 / math.sqrt(hd), U[BF])
        _within(got[0, 4 * h:4 * h + 4], o, tol)
        assert sorted(pos[pages].transpose(0, 1).reshape(nkv, -1)[h, :keep].tolist()) == sorted(kept.tolist())


# ----------------------------------------------------------------- refusals
def test_refusals():
    from kunserve_b200.kv.layout import KVLayout
    from kunserve_b200.ops import (DecodePlan, PagedKV, PrefixGroup, Rotary, SharedPrefixPlan, compact_cache,
                                   rotary_append, rotary_apply, select_evictions, shared_prefix_attention,
                                   weighted_decode_attention)
    pool, kv, lay = _cache(6, 16, 2, 64, BF)
    bad = pytest.raises((RuntimeError, ValueError))
    with bad:
        PagedKV(pool.float(), lay)
    with bad:
        PagedKV(pool[:-64], lay)
    with bad:
        PagedKV(pool.cpu(), lay)
    with bad:
        PagedKV(pool, lay, 3)
    with bad:
        PagedKV(pool, KVLayout(6, 2, 16, 2, 64, 4))
    rot = Rotary(64)
    i32 = dict(dtype=torch.int32, device="cuda")
    x, pos = torch.zeros(3, 4, 64, device="cuda", dtype=BF), torch.zeros(3, **i32)
    for args in ((x.float(), pos), (x, pos.long()), (x, pos[:2]), (x[..., :32], pos), (x, pos.cpu()),
                 (x.transpose(1, 2), pos)):
        with bad:
            rotary_apply(*args, rot)
    with bad:
        rotary_apply(x, pos, rot, out=x[:2])
    with bad:
        rotary_append(x, pos, pos, pos, rot, kv, 2)
    with bad:
        rotary_append(x[:, :3], pos, pos, pos, rot, kv, 0)
    with bad:
        rotary_append(x.to(FP), pos, pos, pos, rot, kv, 0)
    with bad:
        rotary_append(x, pos, pos, pos, rot, kv, 0, weights=torch.zeros(6, 2, 16, device="cuda"))
    for groups in ([PrefixGroup([0], 17, [([1], 1, 1)])], [PrefixGroup([6], 1, [([1], 1, 1)])],
                   [PrefixGroup([0], 1, [([-1], 1, 1)])], [PrefixGroup([0], 1, [([1], 1, 2)])],
                   [PrefixGroup([0], -1, [([1], 1, 1)])]):
        with bad:
            SharedPrefixPlan(groups, kv, 4)
    with bad:
        SharedPrefixPlan([PrefixGroup([0], 1, [([1], 1, 1)])], kv, 5)
    plan = SharedPrefixPlan([PrefixGroup([0], 1, [([1], 1, 1)])], kv, 4)
    q = torch.zeros(1, 4, 64, device="cuda", dtype=BF)
    other = _cache(6, 8, 2, 64, BF)[1]
    for args in ((q.to(FP), kv, 0), (q[:, :2], kv, 0), (q, kv, 2), (q, other, 0), (q.cpu(), kv, 0),
                 (torch.zeros(1, 4, 66, device="cuda", dtype=BF)[..., 1:65], kv, 0)):
        with bad:
            shared_prefix_attention(*args, plan)
    with bad:
        shared_prefix_attention(q, kv, 0, plan, out=torch.zeros(2, 4, 64, device="cuda", dtype=BF))
    w, sp = torch.zeros(6, 2, 16, device="cuda"), torch.zeros(6, 2, 16, **i32)
    with bad:
        weighted_decode_attention(q, kv, 0, plan, w)   # not a decode plan
    with bad:
        DecodePlan([[0]], [17], kv, 4)
    with bad:
        DecodePlan([[0]], [1, 1], kv, 4)
    dec = DecodePlan([[0, 1]], [20], kv, 4)
    for bw in (w[:5], w.double(), w[:, :1], w.cpu(), w.transpose(1, 2)):
        with bad:
            weighted_decode_attention(q, kv, 0, dec, bw)
    for kw in (dict(keep=0), dict(keep=4, sinks=3, recent=2), dict(keep=4, sinks=-1)):
        with bad:
            select_evictions(w, sp, dec, **kw)
    with bad:
        select_evictions(w, sp.long(), dec, 4)
    moves, counts = select_evictions(w, sp, dec, 4)
    with bad:
        compact_cache(kv, 0, dec, moves[..., :1], counts)
    with bad:
        compact_cache(kv, 0, dec, moves, counts[:, :1].contiguous())
    with bad:
        compact_cache(kv, 5, dec, moves, counts)


def test_empty_batches():
    """No tokens, no heads, no requests: empty results, nothing launched."""
    from kunserve_b200.ops import (DecodePlan, Rotary, compact_cache, rotary_append, rotary_apply, select_evictions,
                                   weighted_decode_attention)
    pool, kv, _ = _cache(6, 16, 2, 64, BF)
    before = pool.clone()
    i32 = torch.zeros(0, dtype=torch.int32, device="cuda")
    rot = Rotary(64)
    assert rotary_apply(torch.zeros(0, 4, 64, device="cuda", dtype=BF), i32, rot).shape == (0, 4, 64)
    assert rotary_apply(torch.zeros(3, 0, 64, device="cuda", dtype=BF), torch.zeros(3, dtype=torch.int32, device="cuda"),
                        rot).shape == (3, 0, 64)
    rotary_append(torch.zeros(0, 6, 64, device="cuda", dtype=BF), i32, i32, i32, rot, kv, 0)
    plan = DecodePlan([], [], kv, 4)
    w, sp = torch.zeros(6, 2, 16, device="cuda"), torch.zeros(6, 2, 16, dtype=torch.int32, device="cuda")
    assert weighted_decode_attention(torch.zeros(0, 4, 64, device="cuda", dtype=BF), kv, 0, plan, w).shape == (0, 4, 64)
    moves, counts = select_evictions(w, sp, plan, 4)
    assert moves.shape == (0, 2, 0, 2) and counts.shape == (0, 2)
    compact_cache(kv, 0, plan, moves, counts, w, sp)
    # one request that needs no eviction: no moves
    moves, counts = select_evictions(w, sp, DecodePlan([[0]], [4], kv, 4), 4)
    assert moves.shape == (1, 2, 0, 2) and (counts == 0).all()
    assert torch.equal(pool, before)
    # one token whose row has a stride that no second row uses
    q = torch.zeros(70 + 4 * 64, device="cuda", dtype=BF)[64:64 + 256].view(1, 4, 64)
    q = q.as_strided((1, 4, 64), (13, 64, 1))
    assert weighted_decode_attention(q, kv, 0, DecodePlan([[0]], [4], kv, 4), w).shape == (1, 4, 64)


def test_nan_in_unused_places_reaches_nothing():
    """Slots past a request's tokens hold NaN in the cache and in the weights."""
    from kunserve_b200.ops import DecodePlan, select_evictions, weighted_decode_attention
    pool, kv, lay = _cache(5, 16, 2, 64, BF, poison=True)
    pages, n = [4, 1], 19
    _fill(pool, lay, pages, n, 0, 1, 1)
    w = torch.full((kv.pages_total, 2, 16), math.nan, device="cuda")
    at = torch.arange(n)
    idx = (torch.tensor(pages)[at // 16], slice(None), at % 16)
    w[idx] = 0.0
    sp = torch.zeros(kv.pages_total, 2, 16, dtype=torch.int32, device="cuda")
    plan = DecodePlan([pages], [n], kv, 4)
    out = weighted_decode_attention(torch.randn(1, 4, 64, device="cuda").to(BF), kv, 0, plan, w)
    assert torch.isfinite(out.float()).all() and torch.isfinite(w[idx]).all()
    assert int(torch.isfinite(w).sum()) == 2 * n
    moves, counts = select_evictions(w, sp + 100, plan, 10)
    assert (counts >= 0).all() and (moves < n).all()
