"""What the row operators refuse before any device work, and the frequencies of rotary positions."""
import ctypes
import math

import numpy as np
import pytest

from trit_b200 import Dense, Rotary, TritError, lm, rms_norm

P = 4096  # stands for an address: a refused call reads nothing


@pytest.mark.parametrize("args, words", [
    (dict(width=0), "width is from 1"),
    (dict(width=2**24 + 1), "width is from 1"),
    (dict(rows=2**31), "a call has at most"),
    (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"),
    (dict(dtype="f64"), "not one of"),
    (dict(dtype="f16", weight_dtype="bf16"), "weight's type"),
    (dict(weight_ptr=None), "weight is NULL"),
    (dict(out_ptr=None), "neither out nor codes"),
    (dict(codes_ptr=P), "come together"),
    (dict(scales_ptr=P), "come together"),
    (dict(sum_ptr=P), "sum without a residual"),
    (dict(residual_stride=64), "residual_stride without"),
    (dict(sum_stride=64), "sum_stride without"),
    (dict(x_stride=63), "shorter than a row"),
    (dict(residual_ptr=2 * P, residual_stride=63), "shorter than a row"),
    (dict(out_stride=63), "shorter than a row"),
    (dict(out_ptr=None, codes_ptr=P, scales_ptr=P, out_stride=64), "out_stride without"),
    (dict(out_ptr=P, out_stride=65), "x and out are one tensor with two strides"),
    (dict(residual_ptr=2 * P, sum_ptr=P, sum_stride=65), "x and sum are one tensor with two strides"),
    (dict(residual_ptr=2 * P, out_ptr=2 * P), "out and sum are one tensor"),
    (dict(residual_ptr=2 * P, sum_ptr=3 * P, out_ptr=2 * P), "out and residual are one tensor"),
])
def test_norm_refusals(args, words):
    call = dict(x_ptr=P, weight_ptr=P, rows=4, width=64, out_ptr=5 * P)
    call.update(args)
    with pytest.raises(TritError, match=words):
        rms_norm(**call)


def test_no_rows_is_no_work():
    rms_norm(None, P, 0, 64, out_ptr=P)
    Rotary(64).apply(None, 0, P, 4)


@pytest.mark.parametrize("options, words", [
    (dict(head_dim=0), "head_dim must be a whole number from 2 to 512"),
    (dict(head_dim=514), "head_dim must be a whole number"),
    (dict(head_dim=63), "head_dim must be even"),
    (dict(head_dim=64, rotary_dim=66), "rotary_dim must be even and at most head_dim"),
    (dict(head_dim=64, rotary_dim=33), "rotary_dim must be even"),
    (dict(head_dim=64, layout="thirds"), "layout is"),
    (dict(head_dim=64, layout=2), "layout must be a string"),
    (dict(head_dim=64, scaling="square"), "scaling is"),
    (dict(head_dim=64, scaling="linear"), "needs factor"),
    (dict(head_dim=64, scaling="yarn", factor=2), "needs trained"),
    (dict(head_dim=64, scaling="yarn", factor=2, trained=4096, fast=1, slow=1), "fast must be more"),
    (dict(head_dim=64, scaling="bands", factor=2, trained=4096, low=4, high=1), "high must be more"),
    (dict(head_dim=64, factor=2), "factor is not a setting"),
    (dict(head_dim=64, scaling="linear", factor=2, trained=4096), "trained is not a setting"),
    (dict(head_dim=64, scaling="yarn", factor=2, trained=4096, low=1), "low is not a setting"),
    (dict(head_dim=64, theta=1), "theta must be a number"),
    (dict(head_dim=64, theta="big"), "theta must be a number"),
    (dict(head_dim=64, frequencies=[1.0]), "1 frequencies for 32 pairs"),
    (dict(head_dim=4, frequencies=[1.0, "x"]), "each of frequencies"),
    (dict(head_dim=4, frequencies=[1.0, 0.1], scaling="linear", factor=2), "not scaled"),
    (dict(head_dim=4, frequencies=[1.0, 0.1], theta=1e4), "theta is not a setting"),
    (dict(head_dim=64, base=1e4), "unknown key base"),
])
def test_rotary_options(options, words):
    with pytest.raises(TritError, match=words):
        Rotary(**options)


def test_rotary_needs_an_object():
    lib = lm.library()
    for text in (None, b"", b"[64]", b"{"):
        assert lib.trit_cuda_rotary_new(text) is None
        assert lib.trit_cuda_last_error()


@pytest.mark.parametrize("args, words", [
    (dict(q_heads=-1), "heads are from 0"),
    (dict(q_heads=65536), "heads are from 0 to 65535"),
    (dict(k_ptr=2 * P, k_heads=65536), "heads are from 0 to 65535"),
    (dict(q_heads=0, k_ptr=2 * P, k_heads=2), "q is given with no heads"),
    (dict(q_ptr=None, q_heads=0), "neither q nor k"),
    (dict(k_ptr=P), "k is given with no heads"),
    (dict(rows=2**31), "a call has at most"),
    (dict(q_stride=255), "q_stride is shorter"),
    (dict(q_out_stride=256), "q_out_stride without q_out"),
    (dict(q_out_ptr=P, q_out_stride=257), "one tensor with two strides"),
    (dict(k_ptr=P, k_heads=4, rows=0), "q_out and k_out are one tensor"),
    (dict(q_out_ptr=2 * P, k_ptr=2 * P, k_heads=4, k_out_ptr=3 * P), "q_out and k are one tensor"),
    (dict(q_out_ptr=2 * P, k_ptr=3 * P, k_heads=4, k_out_ptr=P), "k_out and q are one tensor"),
    (dict(dtype="f8"), "not one of"),
])
def test_rotary_refusals(args, words):
    call = dict(positions_ptr=P, rows=0 if args.get("rows") == 0 else args.get("rows", 0), q_ptr=P, q_heads=4)
    call.update(args)
    with pytest.raises(TritError, match=words):
        Rotary(64).apply(**call)


@pytest.mark.parametrize("n, k, words", [(0, 16, "n is from 1"), (2**31, 16, "n is from 1"), (4, 0, "k is a multiple of 16"),
                                         (4, 24, "k is a multiple of 16"), (4, 2**24 + 16, "k is a multiple of 16")])
def test_fp8_layer_sizes(n, k, words):
    lib = lm.library()
    some = (ctypes.c_uint8 * 64)()
    assert lib.trit_dense_fp8(some, some, n, k, 0) is None
    assert words in lib.trit_cuda_last_error().decode()


def test_fp8_layer_arrays():
    with pytest.raises(TritError, match="not the numbers"):
        Dense.fp8(np.zeros(100, np.uint8), np.zeros(1, np.float32), 4, 32)
    with pytest.raises(TritError, match="not those of the 128 x 128 blocks"):
        Dense.fp8(np.zeros(129 * 160, np.uint8), np.zeros(3, np.float32), 129, 160)


def frequencies(dim, theta, scaling=None, factor=1.0, trained=0, fast=32.0, slow=1.0, low=1.0, high=4.0):
    """The header's formulas, pair by pair."""
    out = []
    for i in range(dim // 2):
        f = theta**(-2.0 * i / dim)
        if scaling == "linear":
            f /= factor
        elif scaling == "ntk":
            f = (theta * factor**(dim / (dim - 2.0)))**(-2.0 * i / dim)
        elif scaling == "bands":
            wave = 2 * math.pi / f
            if wave > trained / low:
                f /= factor
            elif wave >= trained / high:
                part = (trained / wave - low) / (high - low)
                f = (1 - part) * f / factor + part * f
        elif scaling == "yarn":
            # The pair whose frequency turns `n` times over the trained positions: theta^(-2 i / dim) trained = 2 pi n.
            first = math.floor(dim / 2 * math.log(trained / (2 * math.pi * fast), theta))
            last = math.ceil(dim / 2 * math.log(trained / (2 * math.pi * slow), theta))
            first, last = max(first, 0), min(last, dim - 1)
            part = 0.0 if i <= first else 1.0 if i >= last else (i - first) / (last - first)
            f = f * (1 - part) + f / factor * part
        out.append(f)
    return out


@pytest.mark.parametrize("options", [
    {}, dict(scaling="linear", factor=4.0), dict(scaling="ntk", factor=8.0),
    dict(scaling="yarn", factor=16.0, trained=4096), dict(scaling="yarn", factor=40.0, trained=32768, fast=16.0, slow=2.0),
    dict(scaling="bands", factor=8.0, trained=8192), dict(scaling="bands", factor=32.0, trained=1024, low=2.0, high=8.0)])
@pytest.mark.parametrize("dim, theta", [(128, 1e6), (64, 1e4), (36, 5e5)])
def test_frequencies(options, dim, theta):
    got, factor = Rotary(128, rotary_dim=dim, theta=theta, **options).frequencies()
    assert np.allclose(got, frequencies(dim, theta, **options), rtol=1e-12, atol=0)
    want = 0.1 * math.log(options["factor"]) + 1 if options.get("scaling") == "yarn" else 1.0
    assert abs(factor - want) <= want * 2.0**-24


def test_given_frequencies():
    got, factor = Rotary(8, rotary_dim=4, frequencies=[0.5, -0.25], attention_factor=1.25).frequencies()
    assert got == [0.5, -0.25] and factor == 1.25
    assert Rotary(2, scaling="ntk", factor=4.0).frequencies()[0] == [1.0]
