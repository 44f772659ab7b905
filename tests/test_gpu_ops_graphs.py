"""Captured graphs of the sequence operators: each with a workspace of its own."""
import gc

import pytest
import torch

pytestmark = pytest.mark.gpu


def scan_inputs(T, seed):
    """A scan whose chunks go through the workspace."""
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(T, 1, 512, generator=g).cuda() for _ in range(2)]


def captured(ops, z, x, stream):
    out = (torch.empty_like(x), torch.empty(x.shape[1:], device="cuda"))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        ops.gated_scan(z, x, out=out)
    return graph, out


def test_graphs_and_calls_do_not_share_workspaces():
    """Two captures after one warm-up on their stream, and that stream's own calls:
    three blocks. Replayed together on streams of their own, with calls on the
    capture stream between, each gives what it gives alone."""
    from phyz_amd.ops import Ops
    ops = Ops(0)
    (z1, x1), (z2, x2), (z3, x3) = (scan_inputs(20000, k) for k in range(3))
    want = [tuple(t.clone() for t in ops.gated_scan(z, x)) for z, x in ((z1, x1), (z2, x2), (z3, x3))]
    plain = ops.workspace_bytes
    side, a, b = (torch.cuda.Stream() for _ in range(3))
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.gated_scan(z1, x1)
    side.synchronize()
    block = ops.workspace_bytes - plain
    assert block > 0 and ops._L.phz_ops_graph_bytes(ops._h) == 0
    g1, out1 = captured(ops, z1, x1, side)
    assert ops.workspace_bytes == plain + block and ops._L.phz_ops_graph_bytes(ops._h) == block
    g2, out2 = captured(ops, z2, x2, side)
    assert ops.workspace_bytes == plain + 2 * block and ops._L.phz_ops_graph_bytes(ops._h) == 2 * block
    torch.cuda.synchronize()
    for k in range(5):
        for out in (out1, out2):
            out[0].fill_(7.0), out[1].fill_(7.0)
        torch.cuda.synchronize()
        with torch.cuda.stream(a):
            g1.replay()
        with torch.cuda.stream(b):
            g2.replay()
        with torch.cuda.stream(side):
            h3, l3 = ops.gated_scan(z3, x3)
        torch.cuda.synchronize()
        for got, expect in ((out1, want[0]), (out2, want[1]), ((h3, l3), want[2])):
            assert torch.equal(got[0], expect[0]) and torch.equal(got[1], expect[1]), k
    assert ops.workspace_bytes == plain + 3 * block


def test_calls_of_one_capture_share_its_workspace():
    from phyz_amd.ops import Ops
    ops = Ops(0)
    z, x = scan_inputs(20000, 4)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ops.gated_scan(z, x)
    side.synchronize()
    before = ops.workspace_bytes
    outs = [(torch.empty_like(x), torch.empty(1, 512, device="cuda")) for _ in range(3)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        for out in outs:
            ops.gated_scan(z, x, out=out)
    graph.replay()
    torch.cuda.synchronize()
    want = ops.gated_scan(z, x)
    assert ops._L.phz_ops_graph_bytes(ops._h) == before
    for out in outs:
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_a_graph_outlives_its_handle():
    """With a workspace, and with the zeros that products read past their ends."""
    from phyz_amd.ops import Ops
    z, x = scan_inputs(20000, 5)
    w, xs = torch.randn(512, 1096, device="cuda"), torch.randn(2000, 1096, device="cuda")
    other = Ops(0)
    want, y_want = tuple(t.clone() for t in other.gated_scan(z, x)), other.linear(xs, w)
    ops = Ops(0)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.gated_scan(z, x)
    side.synchronize()
    graph, out = captured(ops, z, x, side)
    product, y = torch.cuda.CUDAGraph(), torch.empty(2000, 512, device="cuda")
    third = Ops(0)
    with torch.cuda.graph(product, stream=side):
        third.linear(xs, w, out=y)
    del ops, third
    gc.collect()
    filler = [torch.full((1 << 20,), 3.0, device="cuda") for _ in range(8)]
    for _ in range(3):
        out[0].zero_(), y.zero_()
        graph.replay()
        product.replay()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1]) and torch.equal(y, y_want)
    assert all(bool((f == 3).all()) for f in filler)
