"""What Dense.fp8 takes for e4m3 numbers: their bytes reach the library as they are, and nothing else does."""
import ctypes

import numpy as np
import pytest

from trit_b200 import Dense, TritError, lm

N, K = 6, 32


class Library:
    """Keeps what a layer was made of."""

    def trit_dense_fp8(self, codes, scales, n, k, device):
        self.codes = np.frombuffer(ctypes.string_at(codes, n * k), np.uint8).reshape(n, k)
        return 1

    def trit_dense_free(self, handle):
        pass


@pytest.fixture
def made(monkeypatch):
    lib = Library()
    monkeypatch.setattr(lm, "library", lambda: lib)
    return lib


def numbers():
    return np.random.default_rng(1).integers(0, 256, (N, K), dtype=np.uint8)


SCALES = np.ones((1, 1), np.float32)


@pytest.mark.parametrize("make", [lambda b: b, lambda b: b.view(np.int8), lambda b: b.astype(np.int64), lambda b: b.astype(np.uint16).tolist(),
                                  lambda b: b.reshape(-1), lambda b: np.asfortranarray(b), lambda b: np.repeat(b, 2, 0)[::2]])
def test_bytes(made, make):
    Dense.fp8(make(numbers()), SCALES, N, K)
    assert np.array_equal(made.codes, numbers())


def test_e4m3_type(made):
    """The numbers of a float8 type keep their bits: 1.5 is 0x3C and -2 is 0xC0, not 1 and 254."""
    f8 = pytest.importorskip("ml_dtypes").float8_e4m3fn
    codes = np.tile(np.array([1.5, -2.0], np.float32).astype(f8), (N, K // 2))
    Dense.fp8(codes, SCALES, N, K)
    assert np.array_equal(made.codes, np.tile(np.array([0x3C, 0xC0], np.uint8), (N, K // 2)))
    Dense.fp8(numbers().view(f8), SCALES, N, K)
    assert np.array_equal(made.codes, numbers())


@pytest.mark.parametrize("codes", [np.ones((N, K), np.float32), np.ones((N, K), np.float16), np.ones((N, K)), np.ones((N, K), bool),
                                   np.full((N, K), 256), np.full((N, K), -1), np.full((N, K), 1j), np.ones((N, K), "V1")])
def test_refused(made, codes):
    with pytest.raises(TritError, match="neither bytes nor e4m3 numbers"):
        Dense.fp8(codes, SCALES, N, K)


@pytest.mark.parametrize("name", ["float8_e5m2", "float8_e4m3fnuz", "float8_e4m3b11fnuz", "float8_e8m0fnu"])
def test_other_one_byte_types(made, name):
    kind = getattr(pytest.importorskip("ml_dtypes"), name, None)
    if kind is None:
        pytest.skip(f"no {name} here")
    with pytest.raises(TritError, match="neither bytes nor e4m3 numbers"):
        Dense.fp8(numbers().view(kind), SCALES, N, K)
