"""Products of 8-bit floating point with block scales (trit_dense_fp8) against 64 bits."""
import numpy as np
import pytest

from trit_b200 import Dense, TritError
from tests import rows_oracle

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def numbers(g, *shape, size=100.0):
    """e4m3 numbers of a normal distribution."""
    return (torch.randn(*shape, generator=g, device="cuda") * size).clamp(-448, 448).to(torch.float8_e4m3fn)


def layer(n, k, seed):
    """(the layer, its weights in 64 bits on the GPU)."""
    g = torch.Generator("cuda").manual_seed(seed)
    codes = numbers(g, n, k)
    scales = 1e-4 * (0.1 + 2 * torch.rand((n + 127) // 128, (k + 127) // 128, generator=g, device="cuda"))
    w = codes.double() * scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return Dense.fp8(codes.view(torch.uint8).cpu().numpy(), scales.cpu().numpy(), n, k), w


def rows(m, k, seed):
    """8-bit rows (16-byte aligned), their scales, and what they stand for."""
    g = torch.Generator("cuda").manual_seed(seed)
    codes = numbers(g, m, k)
    scales = 0.01 * (0.1 + torch.rand(m, (k + 127) // 128, generator=g, device="cuda"))
    return codes, scales, codes.double() * scales.double().repeat_interleave(128, 1)[:, :k]


def check(got, x, w):
    """A block's sum: four steps of 32 products on the tensor cores, where each of 33 terms may lose what lies 2^-24 below
    the largest, so 4 * 33 * 2^-24 of the terms' absolute sum at most; then two f32 roundings a block (the scales' product,
    the addition), of sums that are at most the absolute sum; then the output's own."""
    want, size = x @ w.t(), x.abs() @ w.abs().t()
    blocks = (x.shape[1] + 127) // 128
    off = (got.double() - want).abs()
    eps = torch.finfo(got.dtype).eps
    tiny = torch.finfo(got.dtype).smallest_normal * eps
    tol = size * ((4 * 33 + 2 * blocks + 2) * 2.0**-24) + want.abs() * eps / 2 * 1.01 + tiny
    assert got.shape == want.shape and bool((off <= tol).all()), f"{int((off > tol).sum())} off, worst {float((off / size).max())}"
    if got.dtype == torch.float32:  # far from the bound as a whole
        assert float(off.norm()) <= 2.0**-20 * float(size.norm())


def codes_call(dense, codes, scales, dtype, stream=None, out_stride=0):
    m, wide = codes.shape[0], out_stride or dense.n
    out = torch.full((m + 2, wide), 5.0, dtype=TYPES[dtype], device="cuda")
    dense.forward_codes(codes.data_ptr(), scales.data_ptr(), m, out[1:].data_ptr(), dtype=dtype, out_stride=out_stride, stream=stream)
    torch.cuda.synchronize()
    assert bool((out[0] == 5).all() and (out[-1] == 5).all() and (out[:, dense.n:] == 5).all())
    return out[1:-1, :dense.n]


@pytest.mark.parametrize("n, k", [(1, 16), (7, 128), (33, 48), (64, 144), (127, 256), (129, 1040), (300, 2064), (513, 4096), (1000, 8208)])
@pytest.mark.parametrize("m", [1, 2, 9, 16, 17, 33, 64, 65, 127, 128, 129, 300])
def test_sizes(n, k, m):
    dense, w = layer(n, k, n + k)
    codes, scales, x = rows(m, k, m)
    dtype = ["f32", "f16", "bf16"][(n + m) % 3]
    check(codes_call(dense, codes, scales, dtype), x, w)


@pytest.mark.parametrize("n, stride", [(4, 0), (8, 0), (8, 24), (40, 48), (64, 72), (129, 136), (256, 264), (257, 258)])
@pytest.mark.parametrize("m", [1, 16, 17, 64, 65, 150, 700])
def test_places_of_the_output(n, stride, m):
    """Rows of the output that tensor copies take (16-byte aligned), narrower than their boxes too, and rows that they do not;
    what lies between and around them stays."""
    dense, w = layer(n, 272, n)
    codes, scales, x = rows(m, 272, m)
    for dtype in ("f32", "f16", "bf16"):
        check(codes_call(dense, codes, scales, dtype, out_stride=stride), x, w)


@pytest.mark.parametrize("n, k, m", [(12288, 2048, 1), (4096, 4096, 5), (2048, 6144, 64), (32768, 256, 20), (5001, 2064, 333), (2560, 1024, 2100),
                                     (129, 128, 5000), (40, 16384, 3), (3000, 512, 1037), (256, 11008, 260)])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_larger(n, k, m, dtype):
    dense, w = layer(n, k, 1)
    codes, scales, x = rows(m, k, 2)
    got = codes_call(dense, codes, scales, dtype)
    check(got, x, w)
    assert torch.equal(got, codes_call(dense, codes, scales, dtype)), "two calls differ"


@pytest.mark.parametrize("n, k, m", [(357, 2112, 225), (20001, 400, 333), (3825, 672, 621), (3824, 672, 621), (2049, 4112, 389), (2064, 4112, 389),
                                     (110, 1360, 83), (257, 8208, 1131), (2561, 528, 6400), (20001, 400, 50),
                                     (23001, 2064, 50), (5001, 4112, 33), (1000, 8208, 64), (9417, 5200, 35)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_many_rows(n, k, m, dtype):
    """Tiles of one block or two an SM and of pairs, k split or not, whole 16 bytes or odd rows to write."""
    dense, w = layer(n, k, 3)
    codes, scales, x = rows(m, k, 4)
    got = codes_call(dense, codes, scales, dtype)
    check(got, x, w)
    assert torch.equal(got, codes_call(dense, codes, scales, dtype)), "two calls differ"


@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("n, k, m", [(96, 272, 5), (700, 1024, 70), (1024, 2048, 600)])
def test_rows_of_values(n, k, m, dtype):
    """Rows are rounded first, also those of a wider tensor; the host's call and the plain device call agree."""
    dense, w = layer(n, k, 4)
    g = torch.Generator("cuda").manual_seed(m)
    wide = torch.randn(m, k + 40, generator=g, device="cuda") * (0.5 + 30 * (torch.rand(1, k + 40, generator=g, device="cuda") > 0.98))
    wide = wide.to(TYPES[dtype])
    for first in (0, 3):
        x = wide[:, first:first + k]
        codes, scales = rows_oracle.rows_of(x.float().cpu().numpy())
        want = torch.from_numpy(rows_oracle.values_of(codes, scales)).cuda()
        out = torch.full((m, n + 3), 5.0, dtype=x.dtype, device="cuda")
        dense.forward_rows(x.data_ptr(), m, out.data_ptr(), dtype=dtype, x_stride=k + 40, out_stride=n + 3)
        torch.cuda.synchronize()
        check(out[:, :n], want, w)
        assert bool((out[:, n:] == 5).all())
    if dtype == "f32":
        x = x.contiguous()
        assert np.array_equal(dense.forward(x.cpu().numpy()), out[:, :n].cpu().numpy())
        again = torch.empty(m, n, device="cuda")
        torch.cuda.synchronize()
        dense.forward_device(x.data_ptr(), m, again.data_ptr())
        torch.cuda.synchronize()
        assert torch.equal(again, out[:, :n])


@pytest.mark.parametrize("m", [3, 40, 200, 700])
def test_rows_that_are_not_numbers(m):
    """A NaN scale or number spoils its row alone; a NaN weight its column alone."""
    n, k = 260, 1040
    g = torch.Generator("cuda").manual_seed(1)
    codes = numbers(g, n, k)
    codes.view(torch.uint8)[5, 700] = 0x7F
    scales = torch.full(((n + 127) // 128, (k + 127) // 128), 0.001, device="cuda")
    dense = Dense.fp8(codes.view(torch.uint8).cpu().numpy(), scales.cpu().numpy(), n, k)
    w = codes.double() * 0.001
    xc, xs, x = rows(m, k, 3)
    xs[1, 4] = float("nan")
    xc.view(torch.uint8)[2, 1039] = 0xFF
    got = codes_call(dense, xc, xs, "f32")
    assert bool(got[1].isnan().all() and got[2].isnan().all() and got[:, 5].isnan().all())
    keep_r = [r for r in range(m) if r not in (1, 2)]
    keep_c = [c for c in range(n) if c != 5]
    w32 = codes.double() * scales.double()[0, 0]
    check(got[keep_r][:, keep_c], x[keep_r], w32[keep_c])


def test_largest_numbers():
    """Sums of 448 * 448 over every block, and scales that bring them beyond f16: infinity there, as a rounding gives."""
    n, k, m = 130, 4096, 66
    dense = Dense.fp8(np.full((n, k), 0x7E, np.uint8), np.full((2, 32), 1e-3, np.float32), n, k)
    codes = torch.full((m, k), 0x7E, dtype=torch.uint8, device="cuda")
    scales = torch.full((m, 32), 0.5, device="cuda")
    want = 448.0 * 448.0 * k * 0.5 * float(np.float32(1e-3))
    got = codes_call(dense, codes, scales, "f32")
    assert bool(((got - want).abs() <= want * 2.0**-18).all())
    assert bool(codes_call(dense, codes, scales, "f16").isinf().all())


def test_streams_and_replay():
    """Calls overlap, those that round their rows too; a captured call has scratch of its own."""
    n, k = 700, 1536
    dense, w = layer(n, k, 6)
    xs = [torch.randn(m, k, device="cuda") for m in (3, 150)]
    outs = [torch.empty(x.shape[0], n, device="cuda") for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    for _ in range(20):
        for x, out, s in zip(xs, outs, streams):
            dense.forward_rows(x.data_ptr(), x.shape[0], out.data_ptr(), stream=s.cuda_stream)
    torch.cuda.synchronize()
    want = []
    for x, out in zip(xs, outs):
        c, s = rows_oracle.rows_of(x.cpu().numpy())
        want.append(torch.from_numpy(rows_oracle.values_of(c, s)).cuda())
        check(out, want[-1], w)
    graphs = []
    first = [out.clone() for out in outs]
    for x, out, s in zip(xs, outs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            dense.forward_rows(x.data_ptr(), x.shape[0], out.data_ptr(), stream=s.cuda_stream)
        graphs.append(g)
    for out in outs:
        out.fill_(5)
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for out, f in zip(outs, first):
        assert torch.equal(out, f)
    # The graphs go before the layer, which gives back what they had.
    del g
    graphs.clear()
    dense.close()


def test_refusals():
    dense, _ = layer(40, 64, 1)
    codes, scales, _ = rows(4, 64, 1)
    out = torch.zeros(4, 40, device="cuda")
    host = torch.zeros(4, 40)
    with pytest.raises(TritError, match="codes is not aligned to 16"):
        dense.forward_codes(codes.data_ptr() + 8, scales.data_ptr(), 1, out.data_ptr())
    with pytest.raises(TritError, match="out is not device memory"):
        dense.forward_codes(codes.data_ptr(), scales.data_ptr(), 4, host.data_ptr())
    with pytest.raises(TritError, match="shorter than a row"):
        dense.forward_codes(codes.data_ptr(), scales.data_ptr(), 4, out.data_ptr(), out_stride=39)
    with pytest.raises(TritError, match="not one of"):
        dense.forward_rows(out.data_ptr(), 4, out.data_ptr(), dtype="f8")
    with pytest.raises(TritError, match="scales is NULL"):
        dense.forward_codes(codes.data_ptr(), None, 4, out.data_ptr())
    dense.forward_codes(None, None, 0, None)
    other = Dense.q8_0(np.zeros(32 * 4 * 34, np.uint8), 32, 128)
    with pytest.raises(TritError, match="not 8-bit floating point"):
        other.forward_codes(codes.data_ptr(), scales.data_ptr(), 1, out.data_ptr())
