"""Rotary positions far behind 32 bits against angles formed in whole numbers, where a 64-bit product has lost the angle."""
import math
from fractions import Fraction

import numpy as np
import pytest

from trit_b200 import Rotary

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def pi_fraction(bits=300):
    """pi = 16 atan(1/5) - 4 atan(1/239)."""
    one = 1 << bits + 20

    def atan(n):
        term = total = one // n
        k, sign = 1, -1
        while term:
            term //= n * n
            k += 2
            total += sign * (term // k)
            sign = -sign
        return total

    return Fraction(4 * (4 * atan(5) - atan(239)), one)


PI = pi_fraction()


def remainder(position, frequency):
    """position * frequency less whole turns, the product exact."""
    x = Fraction(position) * Fraction(frequency) / (2 * PI)
    return float((x - round(x)) * 2 * PI)


POSITIONS = [2**31 + 5, -(2**33) - 1, 2**40 + 7, 2**45 + 12345, -(2**48) + 1, 2**52 + 3, 2**53, -(2**53) + 1]


@pytest.mark.parametrize("layout", ["halves", "interleaved"])
@pytest.mark.parametrize("options", [dict(theta=1e4), dict(theta=1e6, scaling="yarn", factor=16.0, trained=4096), dict(theta=1.5),
                                     dict(scaling="linear", factor=1e-6), dict(frequencies=[1.0, -0.1, 1000.1, 2.0**27 - 0.3, 1e-9] + [0.0] * 27)])
def test_far_positions(layout, options):
    """cos and sin off by 2^-23 (half a step from the angle's rounding, up to 2 steps of the function, the factor's
    product), so a value by 2^-22 (|a| + |b|) with the products' own roundings; the angle's own error is below 2^-24 up to
    2^80 radians, the farthest here, and counts once for each of a pair's two terms."""
    rotary = Rotary(64, layout=layout, **options)
    f, factor = rotary.frequencies()
    g = torch.Generator("cuda").manual_seed(1)
    q = torch.randn(len(POSITIONS), 3, 64, generator=g, device="cuda")
    out, at = torch.empty_like(q), torch.tensor(POSITIONS, device="cuda")
    rotary.apply(at.data_ptr(), len(POSITIONS), q.data_ptr(), 3, dtype="f32", q_out_ptr=out.data_ptr())
    torch.cuda.synchronize()
    x, got = q.double().cpu().numpy(), out.double().cpu().numpy()
    a, b = (slice(0, 64, 2), slice(1, 64, 2)) if layout == "interleaved" else (slice(0, 32), slice(32, 64))
    angle = np.array([[remainder(p, w) for w in f] for p in POSITIONS])[:, None, :]
    cos, sin = factor * np.cos(angle), factor * np.sin(angle)
    size = factor * (np.abs(x[..., a]) + np.abs(x[..., b])) * (2.0**-22 + 2.0**-24)
    for part, want in ((a, x[..., a] * cos - x[..., b] * sin), (b, x[..., b] * cos + x[..., a] * sin)):
        off = np.abs(got[..., part] - want)
        assert (off <= size + np.abs(want) * 2.0**-24).all(), float((off / size).max())


def test_remainder():
    """The oracle itself at angles that 64 bits still hold."""
    for p, w in ((12345, 0.5), (-3, 0.001), (2**20, 1.0)):
        assert abs(math.cos(remainder(p, w)) - math.cos(p * w)) < 1e-9
