"""8-bit calls captured into graphs of a caller's own, without a workspace."""
import math

import pytest
import torch

from tests.test_float8_gpu import E4M3, ops  # noqa: F401 (the fixture)

pytestmark = pytest.mark.gpu


def captured(call):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    return graph


def test_graphs_without_a_workspace_share_nothing(ops):  # noqa: F811
    """What a captured call needs cleared is cleared in its graph, and what one call leaves behind is no other's: graphs captured on one stream are
    replayed in any order, after other calls, some never, and scratch memory that the kernel set keeps is not theirs."""
    g = torch.Generator(device="cuda").manual_seed(2)
    M, N, K = 480, 130, 11008                                  # tiles in parts, joined by counters
    a = torch.randn(M, K, generator=g, device="cuda").to(torch.bfloat16)
    w8 = ops.float8_weight(torch.randn(N, K, generator=g, device="cuda"))
    heads, kv_heads, hd, page, n, R = 8, 8, 64, 32, 4000, 20          # requests in parts, joined by counters
    q = torch.randn(R, heads, hd, generator=g, device="cuda").to(torch.bfloat16)
    pages = -(-n // page)
    pools = [(100 * torch.randn(pages, kv_heads, page, hd, generator=g, device="cuda")).clamp(-448, 448).to(E4M3) for _ in range(2)]
    scales = [torch.full((pages, kv_heads), 2.0 ** -7, device="cuda") for _ in range(2)]
    table = torch.arange(pages, dtype=torch.int32, device="cuda").repeat(R, 1)
    cu = torch.arange(R + 1, dtype=torch.int32, device="cuda")
    kv = torch.full((R,), n, dtype=torch.int32, device="cuda")
    want = [torch.empty(M, N, device="cuda"), torch.empty(R, heads * hd, dtype=torch.bfloat16, device="cuda")]
    got = [[torch.full_like(t, math.nan) for t in want] for _ in range(3)]

    def both(out):
        ops.linear_float8(a, w8, out[0])
        ops.paged_attention_float8(q, *pools, *scales, table, cu, kv, out[1], 0.1, 0, page, R, 1, n)

    both(want)
    torch.cuda.synchronize()
    graphs = [captured(lambda out=out: both(out)) for out in got]
    torch.cuda.synchronize()
    for ws in ops._float8_scratch.values():                    # whatever the set keeps was never cleared by a graph that did not run
        for buffer in ws._bufs.values():
            buffer.fill_(0x55)
    ops._float8_scratch.clear()
    for i in (2, 1, 2):
        graphs[i].replay()
    torch.cuda.synchronize()
    for i in (1, 2):
        assert all(torch.equal(x, y) for x, y in zip(got[i], want))
    both(got[0])
    assert all(torch.equal(x, y) for x, y in zip(got[0], want))
    ops.check_float8_errors()
