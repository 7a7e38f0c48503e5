"""Arguments that the cache operators refuse at the edges of their types."""
import pytest
import torch

from test_cache_ops_gpu import BF, _cache, _no_device_error  # noqa: F401

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sinks,recent", [(1 << 62, 1 << 62), (5, 0), (0, 5), (2, 3), ((1 << 63) - 1, 4)])
def test_protected_tokens_must_fit(sinks, recent):
    """Also where their sum leaves 64 bits."""
    from kunserve_b200.ops import DecodePlan, select_evictions
    pool, kv, _ = _cache(4, 16, 2, 64, BF)
    w, sp = torch.zeros(4, 2, 16, device="cuda"), torch.zeros(4, 2, 16, dtype=torch.int32, device="cuda")
    plan = DecodePlan([[0, 1]], [20], kv, 4)
    with pytest.raises(RuntimeError, match="must fit in keep"):
        select_evictions(w, sp, plan, 4, sinks, recent)
    select_evictions(w, sp, plan, 4, 2, 2)
