"""Attention over the 8-bit cache (trit_cuda_kv_attend) for f32 rows whose
scores are far from zero."""
import numpy as np
import pytest

from trit_b200 import KvCache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# One row takes the kernel of few rows, 200 rows of 32 heads that of many.
@pytest.mark.parametrize("rows", [1, 200])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("size", [-1e20, -1e29, -1e31, -1e36, 1e36])
def test_equal_scores_of_any_size(rows, hd, size):
    """Equal keys have equal scores, whatever their size: the output is the mean of the values. (They stay f16, so that
    their products are the same to the bit.) t sums at 2^-24 and the weights' and values' f32."""
    heads = 32
    for t in (1, 5, 40):
        k = torch.zeros(t, 1, hd, device="cuda")
        k[:, 0, 0] = 1.0
        v = torch.randn(t, 1, hd, device="cuda").half().float()
        q = torch.zeros(rows, heads, hd, device="cuda")
        q[:, :, 0] = size
        out = torch.full_like(q, float("nan"))
        torch.cuda.synchronize()
        with KvCache(kv_heads=1, pages=1, head_dim=hd, page_tokens=128, sequences=1, max_tokens=128) as kv:
            s = kv.open(1)
            kv.extend(s, [t])
            kv.append(0, s, [t], k.data_ptr(), v.data_ptr())
            kv.attend(0, s, [rows], q.data_ptr(), out.data_ptr(), heads=heads, scale=0.5, causal=False)
            torch.cuda.synchronize()
        want = v.double().mean(0)[None]
        assert float((out.double() - want).abs().max()) <= float(v.abs().max()) * (t + 8) * 2.0**-23
