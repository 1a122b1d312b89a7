"""Row operators from several threads at once, on one layer and one handle: as one after another."""
from concurrent.futures import ThreadPoolExecutor

import pytest

from tests.test_gpu_dense_fp8 import layer
from trit_b200 import Rotary, rms_norm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

WORKERS = 6


def test_threads():
    dense, _ = layer(700, 512, 1)
    rotary = Rotary(64, theta=1e4)
    g = torch.Generator("cuda").manual_seed(2)
    sizes = [1, 5, 40, 70, 300, 9][:WORKERS]
    inputs = [(torch.randn(m, 512, generator=g, device="cuda"), torch.randn(512, generator=g, device="cuda"),
               torch.randint(0, 9999, (m,), generator=g, device="cuda")) for m in sizes]

    def work(i, turns):
        x, w, at = inputs[i]
        m, stream = x.shape[0], torch.cuda.Stream()
        results = []
        with torch.cuda.stream(stream):
            for _ in range(turns):
                h, codes, scales = x.clone(), torch.empty(m, 512, dtype=torch.uint8, device="cuda"), torch.empty(m, 4, device="cuda")
                y, z = torch.empty(m, 700, device="cuda"), torch.empty(m, 700, device="cuda")
                s = stream.cuda_stream
                rms_norm(x.data_ptr(), w.data_ptr(), m, 512, codes_ptr=codes.data_ptr(), scales_ptr=scales.data_ptr(), stream=s)
                dense.forward_codes(codes.data_ptr(), scales.data_ptr(), m, y.data_ptr(), stream=s)
                dense.forward_rows(x.data_ptr(), m, z.data_ptr(), stream=s)
                rotary.apply(at.data_ptr(), m, h.data_ptr(), 8, stream=s)
                results.append((h, codes, scales, y, z))
            stream.synchronize()
        return results

    torch.cuda.synchronize()
    alone = [work(i, 1)[0] for i in range(WORKERS)]
    with ThreadPoolExecutor(WORKERS) as pool:
        for i, results in enumerate(pool.map(lambda i: work(i, 30), range(WORKERS))):
            for r in results:
                assert all(torch.equal(a, b) for a, b in zip(r, alone[i]))
