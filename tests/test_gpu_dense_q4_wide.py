"""The int8 copy of a Q4_0 layer's weights that its first call of many rows
makes (trit_dense_q4_0), when there is no memory for it."""
import numpy as np
import pytest

from tests.test_gpu_dense_q4 import layer
from trit_b200 import Dense, TritError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_a_failed_copy_leaves_nothing_behind():
    """Most of the memory is taken; the calls that cannot have their copy fail and keep nothing, the layer's others go on,
    and the copy is made once there is room."""
    n, k, rows = 16384, 8192, 33
    blocks = np.tile(layer(64, k, 1)[0], (n // 64, 1, 1))
    dense = Dense.q4_0(blocks, n, k)
    x = torch.randn(rows, k, device="cuda")
    out = torch.empty(rows, n, device="cuda")
    want = torch.empty(4, n, device="cuda")
    torch.cuda.synchronize()
    dense.forward_device(x.data_ptr(), 4, want.data_ptr())
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    taken = torch.empty(torch.cuda.mem_get_info()[0] - n * k * 3 // 4, dtype=torch.uint8, device="cuda")
    free = torch.cuda.mem_get_info()[0]
    assert n * k // 4 < free < n * k
    for _ in range(3):
        with pytest.raises(TritError, match="out of memory"):
            dense.forward_device(x.data_ptr(), rows, out.data_ptr())
        assert torch.cuda.mem_get_info()[0] == free
    dense.forward_device(x.data_ptr(), 4, out.data_ptr())
    torch.cuda.synchronize()
    assert torch.equal(out[:4], want)
    del taken
    torch.cuda.empty_cache()
    dense.forward_device(x.data_ptr(), rows, out.data_ptr())
    torch.cuda.synchronize()
    size = float(want.abs().max())
    assert float((out[:4] - want).abs().max()) <= 1e-4 * size
    dense.close()


def test_captured_calls_of_many_rows():
    """Refused before the layer has its int8 copy; afterwards a graph's scratch is its own: graphs replay at once, and after
    a larger call, which replaces the layer's."""
    n, k = 256, 512
    dense = Dense.q4_0(layer(n, k, 2)[0], n, k)
    xs = [torch.randn(r, k, device="cuda") for r in (40, 70)]
    wants, outs = ([torch.zeros(x.shape[0], n, device="cuda") for x in xs] for _ in range(2))
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=streams[0]):
        with pytest.raises(TritError, match="being captured"):
            dense.forward_device(xs[0].data_ptr(), 40, outs[0].data_ptr(), streams[0].cuda_stream)
        outs[0].add_(1)
    g.replay()
    torch.cuda.synchronize()
    assert bool((outs[0] == 1).all())
    for x, want in zip(xs, wants):
        dense.forward_device(x.data_ptr(), x.shape[0], want.data_ptr())
    torch.cuda.synchronize()
    graphs = []
    for x, out, stream in zip(xs, outs, streams):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=stream):
            for _ in range(4):
                dense.forward_device(x.data_ptr(), x.shape[0], out.data_ptr(), stream.cuda_stream)
    big = torch.randn(5000, k, device="cuda")
    large = torch.empty(5000, n, device="cuda")
    torch.cuda.synchronize()
    dense.forward_device(big.data_ptr(), 5000, large.data_ptr())
    torch.cuda.synchronize()
    for _ in range(3):
        for out in outs:
            out.zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, wants))
