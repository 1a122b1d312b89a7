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
