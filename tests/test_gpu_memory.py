"""Calls after one that found no memory: nothing is lost, and the next call is
not blamed for it."""
import pytest

from trit_b200 import KvCache, TritError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_a_call_after_a_failed_allocation():
    """A cache larger than any GPU's memory is refused; calls of another are not."""
    hd = 64
    x = torch.ones(16, 1, hd, device="cuda")
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    with KvCache(kv_heads=1, pages=4, head_dim=hd, page_tokens=16, sequences=1, max_tokens=64) as kv:
        s = kv.open(1)
        for _ in range(2):
            with pytest.raises(TritError, match="out of memory"):
                KvCache(kv_heads=64, pages=1 << 24, head_dim=128, page_tokens=128)
            kv.extend(s, [16])
            with pytest.raises(TritError, match="out of memory"):
                KvCache(kv_heads=64, pages=1 << 24, head_dim=128, page_tokens=128)
            kv.append(0, s, [16], x.data_ptr(), x.data_ptr())
        kv.read(0, s, [16], [16], out.data_ptr(), None)
        torch.cuda.synchronize()
    assert bool((out == 1).all())
