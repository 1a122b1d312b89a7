"""Counts of rows that no call can have (trit_cuda_kv_attend)."""
import pytest

from trit_b200 import KvCache, TritError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_counts_past_64_bits():
    """Rows without causal order need no position of their own, so only the call bounds their count; counts whose sum
    wraps to a small number are refused, and the cache goes on."""
    hd = 64
    x = torch.ones(16, 1, hd, device="cuda")
    out = torch.zeros_like(x)
    torch.cuda.synchronize()
    with KvCache(kv_heads=1, pages=2, head_dim=hd, page_tokens=16, sequences=1, max_tokens=32) as kv:
        s = kv.open(1)
        kv.extend(s, [16])
        kv.append(0, s, [16], x.data_ptr(), x.data_ptr())
        for counts in ([2**63 - 1, 2**63 - 1, 7], [2**62] * 4 + [1], [2**31], [2**31 - 1, 1], [2**63 - 1]):
            with pytest.raises(TritError, match="more than 2\\^31 rows"):
                kv.attend(0, s * len(counts), counts, x.data_ptr(), out.data_ptr(), heads=1, scale=1.0, causal=False)
        kv.attend(0, s, [16], x.data_ptr(), out.data_ptr(), heads=1, scale=1.0, causal=False)
        torch.cuda.synchronize()
    # A weight holds 22 bits, its page's value scale comes as a logarithm (2^-22 of it) and as an inverse (2 units in the
    # last place, 2^-22), and 16 products and a quotient round: all below 2^-19.
    assert float((out - 1).abs().max()) <= 2.0**-19
