"""Captured paged decodes and the scratch of eager ones: graphs captured of the split decode replay
at the same time as each other and as eager calls, after larger calls and release_workspaces() have
given every kept buffer back, and match the eager results bit for bit."""
import pytest
import torch

import attnkernels as ak
from oracle.reference import make_paged_cache

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("warm", [True, False])
@pytest.mark.parametrize("partials", [True, False])
def test_graphs_replay_beside_each_other_and_eager_calls(warm, partials):
    gen = torch.Generator().manual_seed(5)
    kc, vc, tables, lens = make_paged_cache([5000, 700, 33], 8, 128, device="cuda", generator=gen)
    qs = [torch.randn(3, 32, 128, generator=gen).half().cuda() for _ in range(3)]
    fn = ak.paged_decode_partials if partials else ak.paged_decode

    def call(i):
        out = fn(qs[i], kc, vc, tables, lens, 5000, partition_size=256)
        return out if partials else (out,)

    want = [call(i) for i in range(3)]
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    if warm:
        with torch.cuda.stream(side):
            call(0)
        side.synchronize()
    else:
        ak.release_workspaces()
    graphs = []
    for i in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = call(i)
        graphs.append((g, out))
    # A larger call on the capture's stream, then all kept buffers given back and their memory
    # taken by someone else, who must not see it written.
    big_q = torch.randn(3, 64, 128, generator=gen).half().cuda()
    with torch.cuda.stream(side):
        ak.paged_decode(big_q, kc, vc, tables, lens, 5000, partition_size=256)
        side.synchronize()
        ak.release_workspaces()
        others = [torch.full((1 << 20,), 7, dtype=torch.uint8, device="cuda") for _ in range(64)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                graphs[i][0].replay()
        with torch.cuda.stream(side):
            eager = call(2)
    torch.cuda.synchronize()
    for got, w in zip([graphs[0][1], graphs[1][1], eager], want):
        assert all(torch.equal(a, b) for a, b in zip(got, w))
    assert all((t == 7).all() for t in others)
    ak.check_device_status()
