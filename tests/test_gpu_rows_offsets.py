"""Row operators where elements lie more than 2^31 and 2^32 behind their tensor's first."""
import pytest

from tests.test_gpu_dense_fp8 import check, layer, numbers, rows
from trit_b200 import Dense, Rotary, rms_norm

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

FAR = 2**31 + 24  # elements between two rows: the third one begins behind 2^32


@pytest.fixture(autouse=True)
def memory():
    free = torch.cuda.mem_get_info()[0]
    if free < 30 * 2**30:
        pytest.skip(f"{free >> 30} GB free")
    yield
    torch.cuda.empty_cache()


def far_rows(n, width, dtype):
    """n rows FAR elements apart, and the memory around them."""
    flat = torch.empty((n - 1) * FAR + width + 8, dtype=dtype, device="cuda")
    for r in range(n):
        flat[r * FAR:r * FAR + width + 8] = 7
    return flat, torch.as_strided(flat, (n, width + 8), (FAR, 1))


@pytest.mark.parametrize("width", [264, 263, 20000])
def test_norm(width):
    g = torch.Generator("cuda").manual_seed(width)
    flat, x = far_rows(3, width, torch.bfloat16)
    near = torch.randn(3, width, generator=g, device="cuda").to(torch.bfloat16)
    x[:, :width] = near
    residual = torch.randn(3, width, generator=g, device="cuda").to(torch.bfloat16)
    w = torch.randn(width, generator=g, device="cuda")
    outs = []
    for at, stride, kept in ((x, FAR, True), (near.clone(), 0, False)):
        res, codes, scales = residual.clone(), torch.zeros(3, width, dtype=torch.uint8, device="cuda"), torch.zeros(3, (width + 127) // 128, device="cuda")
        rms_norm(at.data_ptr(), w.data_ptr(), 3, width, out_ptr=at.data_ptr(), codes_ptr=codes.data_ptr(), scales_ptr=scales.data_ptr(),
                 residual_ptr=res.data_ptr(), dtype="bf16", x_stride=stride, out_stride=stride)
        torch.cuda.synchronize()
        outs.append((at[:, :width].clone(), res, codes, scales))
        assert not kept or bool((at[:, width:] == 7).all())
    assert all(torch.equal(a, b) for a, b in zip(*outs))


@pytest.mark.parametrize("layout", ["halves", "interleaved"])
def test_rotary(layout):
    g = torch.Generator("cuda").manual_seed(1)
    rotary, at = Rotary(64, layout=layout), torch.tensor([5, 70000, 3], device="cuda")
    flat, q = far_rows(3, 256, torch.bfloat16)
    near = torch.randn(3, 256, generator=g, device="cuda").to(torch.bfloat16)
    q[:, :256] = near
    rotary.apply(at.data_ptr(), 3, q.data_ptr(), 3, q.data_ptr() + 2 * 192, 1, dtype="bf16", q_stride=FAR, k_stride=FAR)
    rotary.apply(at.data_ptr(), 3, near.data_ptr(), 4, dtype="bf16")
    torch.cuda.synchronize()
    assert torch.equal(q[:, :256], near) and bool((q[:, 256:] == 7).all())


@pytest.mark.parametrize("m", [3, 40, 130])
def test_product_into_far_rows(m):
    """Rows of out so far apart that the last one begins around 2^32."""
    dense, w = layer(200, 256, 1)
    codes, scales, x = rows(m, 256, 2)
    stride = (2**32 // m + 8) // 8 * 8
    for more in (0, 1):
        out = torch.empty((m - 1) * (stride + more) + 208, dtype=torch.bfloat16, device="cuda")
        view = torch.as_strided(out, (m, 208), (stride + more, 1))
        view[:] = 7
        dense.forward_codes(codes.data_ptr(), scales.data_ptr(), m, out.data_ptr(), dtype="bf16", out_stride=stride + more)
        torch.cuda.synchronize()
        check(view[:, :200], x, w)
        assert bool((view[:, 200:] == 7).all())
        del out, view


def test_product_of_many_rows():
    """More than 2^31 numbers of x and of the output; a sample of rows against 64 bits."""
    n, k, m = 2064, 2048, 1100003
    dense, w = layer(n, k, 3)
    g = torch.Generator("cuda").manual_seed(4)
    codes = torch.empty(m, k, dtype=torch.float8_e4m3fn, device="cuda")
    for a in range(0, m, 100000):
        codes[a:a + 100000] = numbers(g, min(100000, m - a), k)
    scales = 0.01 * (0.1 + torch.rand(m, k // 128, generator=g, device="cuda"))
    out = torch.full((m + 1, n), 7.0, dtype=torch.bfloat16, device="cuda")
    dense.forward_codes(codes.data_ptr(), scales.data_ptr(), m, out.data_ptr(), dtype="bf16")
    torch.cuda.synchronize()
    some = torch.cat([torch.arange(0, 300, device="cuda"), torch.randint(0, m, (700,), generator=g, device="cuda"),
                      torch.arange(m - 300, m, device="cuda")])
    x = codes[some].double() * scales[some].double().repeat_interleave(128, 1)
    check(out[some], x, w)
    assert bool((out[-1] == 7).all())


def test_product_with_many_weights():
    """More than 2^31 numbers of w."""
    n, k = 1049000, 2064
    g = torch.Generator("cuda").manual_seed(5)
    w = torch.empty(n, k, dtype=torch.float8_e4m3fn, device="cuda")
    for a in range(0, n, 100000):
        w[a:a + 100000] = numbers(g, min(100000, n - a), k)
    ws = 1e-3 * (0.1 + torch.rand((n + 127) // 128, (k + 127) // 128, generator=g, device="cuda"))
    dense = Dense.fp8(w.view(torch.uint8).cpu().numpy(), ws.cpu().numpy(), n, k)
    some = torch.cat([torch.arange(0, 200, device="cuda"), torch.randint(0, n, (600,), generator=g, device="cuda"),
                      torch.arange(n - 200, n, device="cuda")])
    ref = w[some].double() * ws[some // 128].double().repeat_interleave(128, 1)[:, :k]
    for m in (3, 40, 130, 600):
        codes, scales, x = rows(m, k, m)
        out = torch.zeros(m, n, device="cuda")
        dense.forward_codes(codes.data_ptr(), scales.data_ptr(), m, out.data_ptr())
        torch.cuda.synchronize()
        check(out[:, some], x, ref)
