"""Products by pairs of blocks with the next kernels right behind them: a block that ends hands its shared memory to a block
of the kernel behind it, which starts early, so nothing of the pair's may still be on its way there."""
import pytest

from tests.test_gpu_dense_fp8 import check, layer, rows
from trit_b200 import rms_norm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


@pytest.mark.parametrize("n, k, m", [(12288, 2048, 1024), (8192, 1024, 1000), (12288, 4096, 513)])
def test_kernels_behind_a_pair(n, k, m):
    """Pairs, few rows, one block an SM and norms after one another, without a wait and from a recorded graph: all as alone."""
    dense, w = layer(n, k, 1)
    small, ws = layer(700, k, 2)
    codes, scales, x = rows(m, k, 3)
    few, few_scales, xf = rows(5, k, 4)
    some, some_scales, xm = rows(130, k, 5)
    weight = torch.ones(k, device="cuda")
    values = torch.randn(64, k, device="cuda")
    stream = torch.cuda.Stream()

    def outputs():
        return [torch.zeros(m, n, dtype=torch.bfloat16, device="cuda"), torch.zeros(5, 700, device="cuda"),
                torch.zeros(130, 700, device="cuda"), torch.zeros(64, k, dtype=torch.uint8, device="cuda"),
                torch.zeros(64, k // 128, device="cuda")]

    def calls(out, wait=lambda: None):
        s = stream.cuda_stream
        for _ in range(2):
            dense.forward_codes(codes.data_ptr(), scales.data_ptr(), m, out[0].data_ptr(), dtype="bf16", stream=s)
            wait()
            small.forward_codes(few.data_ptr(), few_scales.data_ptr(), 5, out[1].data_ptr(), stream=s)
            wait()
            dense.forward_codes(codes.data_ptr(), scales.data_ptr(), m, out[0].data_ptr(), dtype="bf16", stream=s)
            wait()
            rms_norm(values.data_ptr(), weight.data_ptr(), 64, k, codes_ptr=out[3].data_ptr(), scales_ptr=out[4].data_ptr(), stream=s)
            wait()
            small.forward_codes(some.data_ptr(), some_scales.data_ptr(), 130, out[2].data_ptr(), stream=s)
            wait()

    alone = outputs()
    torch.cuda.synchronize()
    calls(alone, torch.cuda.synchronize)
    check(alone[0], x, w)
    check(alone[1], xf, ws)
    check(alone[2], xm, ws)
    behind = outputs()
    torch.cuda.synchronize()
    for _ in range(20):
        calls(behind)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, behind))
    graph, replayed = torch.cuda.CUDAGraph(), outputs()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        calls(replayed)
    for _ in range(20):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(alone, replayed))
