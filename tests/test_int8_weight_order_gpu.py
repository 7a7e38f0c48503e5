"""A product loads its first weights ahead of its wait for the kernel before
it, which alone makes that kernel's writes visible.  So it may start early
behind any kernel but the one that packs the weights."""
import pytest
import torch

from test_int8_ops_gpu import F32, U, _linear_inputs, _no_device_error  # noqa: F401

pytestmark = pytest.mark.gpu


def _edges(graph):
    """(from, to, programmatic) between the nodes of a captured graph, nodes by their place in the chain."""
    driver = pytest.importorskip("cuda.bindings.driver")
    raw = driver.CUgraph(graph.raw_cuda_graph())
    err, _, _, _, n = driver.cuGraphGetEdges_v2(raw)
    assert err == driver.CUresult.CUDA_SUCCESS
    err, start, end, data, n = driver.cuGraphGetEdges_v2(raw, n)
    assert err == driver.CUresult.CUDA_SUCCESS
    start, end = [int(x) for x in start[:n]], [int(x) for x in end[:n]]
    after = dict(zip(start, end))
    assert len(after) == n                      # a chain
    node, place = next(x for x in start if x not in end), {}
    while node is not None:
        place[node] = len(place)
        node = after.get(node)
    kind = driver.CUgraphDependencyType.CU_GRAPH_DEPENDENCY_TYPE_PROGRAMMATIC
    return sorted((place[a], place[b], int(e.type) == int(kind)) for a, b, e in zip(start, end, data[:n]))


@pytest.mark.parametrize("m", [1, 40, 600])
def test_first_product_waits_for_the_packing(m):
    from kunserve_b200 import ops
    q, s, w, v = _linear_inputs(m, 640, 384)
    ops.int8_linear(q, s, ops.Int8Weight(w, v), dtype=F32)      # (a kernel's first launch of all would start early behind none)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        weight = ops.Int8Weight(w, v)
        for _ in range(3):
            y = ops.int8_linear(q, s, weight, dtype=F32)
    edges = _edges(graph)
    # what makes the handle, then three products: those start early behind one another, the first does not
    last = edges[-1][1]
    assert [(a, b) for a, b, early in edges if early] == [(last - 2, last - 1), (last - 1, last)]
    for _ in range(2):
        graph.replay()
    ref = (q.double() @ w.double().t()) * s.double()[:, None] * v.double()
    assert ((y.double() - ref).abs() <= 4 * U * ref.abs()).all()


def test_products_of_other_streams_wait_for_the_packing():
    """A handle's first product on another stream says nothing of its own: the order is the handle's."""
    from kunserve_b200 import ops
    q, s, w, v = _linear_inputs(9, 2048, 2048)
    side = torch.cuda.Stream()
    want = ops.int8_linear(q, s, ops.Int8Weight(w, v))
    torch.cuda.synchronize()
    for _ in range(10):
        weight = ops.Int8Weight(w, v)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            a = ops.int8_linear(q, s, weight)
        b = ops.int8_linear(q, s, weight)
        torch.cuda.synchronize()
        assert torch.equal(a, want) and torch.equal(b, want)
        del weight
