"""Attention of f16 rows over the 8-bit cache (trit_cuda_kv_attend): the weights
keep more bits than the output."""
import math

import numpy as np
import pytest

from tests.kv_oracle import attend, held
from trit_b200 import KvCache

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


# A row of 8 heads takes the kernel of few rows, 300 rows of 32 that of many.
@pytest.mark.parametrize("rows, heads", [(1, 8), (300, 32)])
@pytest.mark.parametrize("hd, page", [(64, 16), (128, 64)])
@pytest.mark.parametrize("t", [1, 2, 3, 17, 64, 200, 1500])
def test_the_output_is_rounded_once(rows, heads, hd, page, t):
    """Before its rounding to f16 the output is off by the tolerance of f32 rows at most (rounding is monotone, so what is
    rounded lies between the two ends rounded). One position gives back its value to the bit."""
    rng = np.random.default_rng(t)
    k, v = (torch.from_numpy(rng.standard_normal((t, 1, hd)).astype(np.float16)).cuda() for _ in range(2))
    q = torch.from_numpy(rng.standard_normal((rows, heads, hd)).astype(np.float16)).cuda()
    out = torch.full_like(q, float("nan"))
    scale = 1 / math.sqrt(hd)
    torch.cuda.synchronize()
    with KvCache(kv_heads=1, pages=t // page + 1, head_dim=hd, page_tokens=page, sequences=1, max_tokens=t) as kv:
        s = kv.open(1)
        kv.extend(s, [t])
        kv.append(0, s, [t], k.data_ptr(), v.data_ptr(), dtype="f16")
        kv.attend(0, s, [rows], q.data_ptr(), out.data_ptr(), heads=heads, scale=scale, dtype="f16", causal=False)
        torch.cuda.synchronize()
    got = out.cpu().numpy()
    hk, hv = (held(x.double().cpu().numpy(), page) for x in (k, v))
    want, tol = attend(q.double().cpu().numpy(), hk, hv, scale, False)
    low, high = (want - tol).astype(np.float16), (want + tol).astype(np.float16)
    bad = ~((low <= got) & (got <= high))
    assert not bad.any(), f"{bad.sum()} of {bad.size} values off, {np.abs(got.astype(np.float64) - want).max()}"
    if t == 1:
        assert np.array_equal(got, np.broadcast_to(v.cpu().numpy(), got.shape))
