"""Products of 8-bit floating point over the range of scales that the header gives: the two scales' product is 0 or a normal
f32, near either end of those, and each scale may be anything, a denormal number too."""
import pytest

from tests.test_gpu_dense_fp8 import check, codes_call, numbers
from trit_b200 import Dense

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def power(g, lo, hi, *shape):
    """f32 numbers of 2^lo up to 2^hi in size, of either sign."""
    e = torch.randint(lo, hi, shape, generator=g, device="cuda")
    sign = 1.0 - 2.0 * torch.randint(0, 2, shape, generator=g, device="cuda")
    return (sign * (1 + torch.rand(*shape, generator=g, device="cuda")).double() * torch.exp2(e.double())).float()


def layer(codes, scales):
    n, k = codes.shape
    w = codes.double() * scales.double().repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]
    return Dense.fp8(codes.view(torch.uint8).cpu().numpy(), scales.cpu().numpy(), n, k), w


def values(codes, scales):
    return codes.double() * scales.double().repeat_interleave(128, 1)[:, :codes.shape[1]]


# Few rows, up to 64 with one block an SM and two, more with one block, two, pairs; k split over a cluster and not.
SHAPES = [(300, 1040, 3), (20001, 400, 5), (300, 1040, 40), (16384, 4096, 33), (357, 2112, 225), (4096, 4096, 600), (8192, 1024, 1000)]


@pytest.mark.parametrize("n, k, m", SHAPES)
@pytest.mark.parametrize("way", ["small", "large", "small and large"])
def test_ends_of_the_range(n, k, m, way):
    """Sums of a block are around 2^17 for numbers around 100, 2^-13 for the type's smallest."""
    g = torch.Generator("cuda").manual_seed(n + m)
    shape, rows = ((n + 127) // 128, (k + 127) // 128), (m, (k + 127) // 128)
    if way == "small":  # products 2^-126 .. 2^-118
        codes, xc = numbers(g, n, k), numbers(g, m, k)
        scales, xs = power(g, -63, -60, *shape), power(g, -63, -58, *rows)
    elif way == "large":  # products 2^112 .. 2^127
        codes, xc = numbers(g, n, k, size=0.004), numbers(g, m, k, size=0.004)
        scales, xs = power(g, 60, 63, *shape), power(g, 52, 64, *rows)
    else:  # denormal scales of w, those of x beyond the others' reach
        codes, xc = numbers(g, n, k), numbers(g, m, k)
        scales, xs = power(g, -140, -126, *shape), power(g, 120, 127, *rows)
    dense, w = layer(codes, scales)
    x = values(xc, xs)
    for dtype in ("f32", "bf16"):
        check(codes_call(dense, xc, xs, dtype), x, w)


@pytest.mark.parametrize("m", [3, 40, 130])
def test_no_scale(m):
    """A scale of 0 leaves its blocks out."""
    g = torch.Generator("cuda").manual_seed(m)
    codes, xc = numbers(g, 260, 512), numbers(g, m, 512)
    scales, xs = torch.ones(3, 4, device="cuda"), torch.ones(m, 4, device="cuda")
    scales[0, 1] = scales[2, :] = 0.0
    xs[0] = 0.0
    xs[1, 2] = xs[2, 1] = 0.0
    dense, w = layer(codes, scales)
    got = codes_call(dense, xc, xs, "f32")
    check(got, values(xc, xs), w)
    assert bool((got[0] == 0).all() and (got[:, 256:] == 0).all())
