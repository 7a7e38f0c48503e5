"""What the operators keep on the device (plans, rotary frequencies) outlives
the work queued on whatever stream used it, also when the caller lets go of it
first."""
import pytest
import torch

from test_cache_ops_gpu import BF, _allot, _cache, _fill, _no_device_error  # noqa: F401

pytestmark = pytest.mark.gpu


def _behind_queued_work(make, call):
    """``call`` with what ``make`` makes on the current stream, on another stream
    behind queued work; the handle is dropped and its memory offered to others
    before that stream gets there.  Returns the result, and that of a plain call."""
    def offered():
        return [torch.zeros(n, dtype=torch.int32, device="cuda") for n in (128, 512, 2048, 8192, 32768) * 40]

    want, side, handle = call(make()), torch.cuda.Stream(), make()
    offered()
    with torch.cuda.stream(side):           # the allocator has memory for both streams from here on:
        call(handle)                        # asking the driver for more could wait for the GPU
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(400_000_000)      # a good 0.1 s
        got = call(handle)
    busy = not side.query()
    del handle
    # whatever the allocator hands out now on this stream is written at once
    # (zeros: a plan of them has no keys, and frequencies of them do not turn)
    filled = offered()
    torch.cuda.current_stream().synchronize()
    assert busy and not side.query(), "the work was to be still queued"
    side.synchronize()
    del filled
    return got, want


def test_plan_made_on_one_stream_used_on_another():
    from kunserve_b200.ops import DecodePlan, PrefixGroup, SharedPrefixPlan, shared_prefix_attention, \
        weighted_decode_attention
    pool, kv, lay = _cache(80, 16, 2, 128, BF)
    pages = _allot([700, 30, 30], 16, kv.pages_total, 1)
    for i, (p, n) in enumerate(zip(pages, (700, 30, 30))):
        _fill(pool, lay, p, n, 1, 1, i)
    q = torch.randn(2, 8, 128, device="cuda").to(BF)

    def weighted(plan):
        w = torch.zeros(kv.pages_total, 2, 16, device="cuda")
        return torch.cat([weighted_decode_attention(q, kv, 1, plan, w).float().flatten(), w.flatten()])

    got, want = _behind_queued_work(lambda: DecodePlan(pages[:2], [700, 30], kv, 8), weighted)
    assert torch.equal(got, want)
    group = PrefixGroup(pages[0], 700, [(pages[1], 30, 1), (pages[2], 30, 1)])
    got, want = _behind_queued_work(lambda: SharedPrefixPlan([group], kv, 8),
                                    lambda plan: shared_prefix_attention(q, kv, 1, plan))
    assert torch.equal(got, want)


def test_rotary_made_on_one_stream_used_on_another():
    from kunserve_b200.ops import Rotary, rotary_apply
    x = torch.randn(3, 4, 128, device="cuda").to(BF)
    pos = torch.tensor([5, 1000, 70000], dtype=torch.int32, device="cuda")
    got, want = _behind_queued_work(lambda: Rotary(128), lambda rotary: rotary_apply(x, pos, rotary))
    assert torch.equal(got, want)
