"""What a stream capture takes of the 8-bit cache's calls (trit_cuda_kv_*)."""
import pytest

from trit_b200 import KvCache, TritError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_an_extension_without_a_new_page():
    """It touches no device memory, and is refused in a capture as every call that changes a sequence; the capture and the
    cache go on."""
    side = torch.cuda.Stream()
    x = torch.zeros(4, device="cuda")
    with KvCache(kv_heads=1, pages=2, head_dim=64, page_tokens=16, sequences=1, max_tokens=32) as kv:
        s = kv.open(1)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            with pytest.raises(TritError, match="extend: the stream is being captured"):
                kv.extend(s, [1], stream=side.cuda_stream)
            kv.extend(s, [0], stream=side.cuda_stream)  # a call of nothing
            x.add_(1)
        assert kv.length(s[0]) == 0
        g.replay()
        kv.extend(s, [1], stream=side.cuda_stream)
        assert kv.length(s[0]) == 1
        torch.cuda.synchronize()
    assert bool((x == 1).all())
