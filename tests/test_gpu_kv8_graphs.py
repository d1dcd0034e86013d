"""One batch in several CUDA graphs (needs a B200): each graph has an attention workspace of its own, so graphs captured on
one stream may be replayed on any streams, beside each other and beside calls on the capturing stream."""
import pytest
import torch

from kv8_helpers import Pool

pytestmark = pytest.mark.gpu


def test_graphs_of_one_batch_replayed_together(pkg):
    lens = [9000, 8000]
    pool = Pool(pkg, lens, 2, 64, 256, seed=7, fill=lens)
    batch = pool.batch([1, 1], lens)
    side = torch.cuda.Stream()
    q = [torch.randn((2, 8, 64), device="cuda").half() for _ in range(3)]
    want, out = [torch.zeros_like(x) for x in q], [torch.zeros_like(x) for x in q]
    for x, o in zip(q, want):
        pool.cache.attention(batch, x, o, 0.125)
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    held = []
    with torch.cuda.stream(side):
        pool.cache.attention(batch, q[2], out[2], 0.125)
        for i, g in enumerate(graphs):
            side.synchronize()
            before = set(batch._workspaces)
            with torch.cuda.graph(g, stream=side):
                for _ in range(20):
                    pool.cache.attention(batch, q[i], out[i], 0.125)
            held.append(set(batch._workspaces) - before)
    assert [len(h) for h in held] == [1, 1], "one workspace for each graph, whatever the calls in it"
    spaces = [t.data_ptr() for t in batch._workspaces.values()]
    assert len(set(spaces)) == len(spaces) >= 3
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(10):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
        with torch.cuda.stream(side):
            pool.cache.attention(batch, q[2], out[2], 0.125)
    torch.cuda.synchronize()
    pool.cache.check()
    assert all(torch.equal(a, b) for a, b in zip(want, out))
