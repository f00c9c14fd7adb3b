"""The paged cache where it went wrong once: workspaces of graphs, extreme scores and positions."""

import pytest
import torch

from paged_cases import Batch, attend_oracle, check_attention

pytestmark = pytest.mark.gpu

DEV = "cuda"
BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def ops():
    import m5kernels_b200 as m
    from m5kernels_b200 import _lib

    yield m
    assert _lib.device_status() == 0  # no bounded wait gave up


# ---------------------------------------------------------------- workspaces

@pytest.mark.parametrize("hint", [1, 64])
def test_a_graph_keeps_its_workspace(ops, hint):
    """A stream's workspace is replaced by a larger one after a graph was captured there."""
    batch = Batch([1, 1], [9000, 40], q_heads=8, kv_heads=1, dim=64, page=16, dtype=BF16)
    wide = Batch([1, 1], [9000, 40], q_heads=8, kv_heads=1, dim=128, page=16, dtype=BF16)
    want, want_lse, spread = attend_oracle(batch)
    q, args = batch.q.to(DEV), batch.on(DEV)
    wide_q, wide_args = wide.q.to(DEV), wide.on(DEV)
    out, graph, side = torch.empty_like(q), torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        first = ops.paged_attention(q, *args, max_query_len=hint)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        ops.paged_attention(q, *args, max_query_len=hint, out=out)
    with torch.cuda.stream(side):
        ops.paged_attention(wide_q, *wide_args, max_query_len=hint)
        taken = [torch.full((1 << 20,), i, dtype=torch.int32, device=DEV) for i in range(32)]
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    check_attention(out, None, want, want_lse, spread, BF16)
    assert torch.equal(out, first)
    assert all((t == i).all() for i, t in enumerate(taken))


def test_graphs_replayed_beside_each_other(ops):
    """Two graphs captured on one stream, and that stream's own calls, on three streams at once."""
    batch = Batch([1, 1], [9000, 40], q_heads=8, kv_heads=1, dim=128, page=16, dtype=BF16)
    q, args = batch.q.to(DEV), batch.on(DEV)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    with torch.cuda.stream(streams[0]):
        want = ops.paged_attention(q, *args, max_query_len=1)
    torch.cuda.synchronize()
    outs, graphs = [], []
    for _ in range(2):
        out, graph = torch.empty_like(q), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=streams[0]):
            for _ in range(3):
                ops.paged_attention(q, *args, max_query_len=1, out=out)
        outs.append(out)
        graphs.append(graph)
    for _ in range(20):
        for graph, stream in zip(graphs, streams[1:]):
            with torch.cuda.stream(stream):
                graph.replay()
        with torch.cuda.stream(streams[0]):
            got = ops.paged_attention(q, *args, max_query_len=1)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and all(torch.equal(out, want) for out in outs)
