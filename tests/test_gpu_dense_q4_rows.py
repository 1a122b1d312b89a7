"""Rows at the edges of the numbers through a Q4_0 layer's 8-bit activations
(trit_dense_q4_0 with table = 0): one rule for every count of rows."""
import numpy as np
import pytest

from tests.test_gpu_dense_q4 import layer
from trit_b200 import Dense

pytestmark = pytest.mark.gpu

# The 4-bit kernel takes up to 32 rows, the int8 tensor cores more.
ROWS = [1, 5, 32, 33, 70]


def rounded(x):
    """Rows as their int8 codes stand for them. The largest of a group may be so small that the inverse of its scale is
    infinite: what is not zero is then the largest code, and what is zero stays code zero."""
    g = x.reshape(x.shape[0], -1, 32)
    top = np.abs(g).max(-1, keepdims=True)
    with np.errstate(all="ignore"):
        scale = np.where(top > 0, top / np.float32(127), np.float32(1)).astype(np.float32)
        code = np.where(g == 0, 0.0, np.clip(np.rint(g * (np.float32(1) / scale)), -127, 127))
    return (code.astype(np.float64) * scale.astype(np.float16).astype(np.float64)).reshape(x.shape)


def check(got, x, w):
    """f32 sums of k / 32 exact group sums, each times a product of two scales (2^-23 a step, as the last round on the
    tensor cores need not be to nearest)."""
    want, size = rounded(x) @ w.T, np.abs(rounded(x)) @ np.abs(w).T
    tol = size * (x.shape[1] / 32 + 12) * 2.0**-23
    assert np.isfinite(got).all()
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("tiny", [3.7e-37, 1e-38, 1e-44])
def test_groups_of_tiny_values_and_zeros(rows, tiny):
    """A group's largest value is so small that the inverse of its scale overflows: its zeros are zeros."""
    n, k = 64, 256
    blocks, w = layer(n, k, 3)
    x = np.random.default_rng(rows).standard_normal((rows, k)).astype(np.float32)
    x[0, :32] = 0
    x[0, 5] = tiny
    x[0, 6] = -tiny / 3
    x[-1, 64:] = 0
    x[-1, 96:128:2] = tiny
    check(Dense.q4_0(blocks, n, k).forward(x), x, w)


@pytest.mark.parametrize("rows", ROWS)
def test_rows_that_are_not_numbers(rows):
    """A row with NaN or an infinity gives no numbers, and changes no other."""
    n, k = 64, 256
    blocks, w = layer(n, k, 4)
    x = np.random.default_rng(rows).standard_normal((rows, k)).astype(np.float32)
    bad = {r: v for r, v in zip((0, rows // 2, rows - 1), (np.nan, np.inf, -np.nan))}
    for i, (r, v) in enumerate(bad.items()):
        x[r, 37 * i + 3] = v
    got = Dense.q4_0(blocks, n, k).forward(x)
    assert not np.isfinite(got[list(bad)]).any()
    good = [r for r in range(rows) if r not in bad]
    if good:
        check(got[good], x[good], w)
