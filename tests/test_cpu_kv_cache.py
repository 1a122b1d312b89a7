"""The 8-bit key/value cache and the Q4_0 layer on a host without a GPU: the
checks that come before any device work."""
import ctypes

import numpy as np
import pytest

from trit_b200 import Dense, KvCache, TritError, lm


@pytest.mark.parametrize("options, words", [
    (dict(kv_heads=0, pages=4), "kv_heads"),
    (dict(kv_heads=2, pages=0), "pages"),
    (dict(kv_heads=2, pages=4, head_dim=96), "head_dim is 64 or 128"),
    (dict(kv_heads=2, pages=4, page_tokens=24), "page_tokens is 16, 32, 64 or 128"),
    (dict(kv_heads=2, pages=4, layers=0), "layers"),
    (dict(kv_heads=2, pages=4, layers=1.5), "layers"),
    (dict(kv_heads=2, pages=4, sequences=0), "sequences"),
    (dict(kv_heads=2, pages=4, max_tokens=0), "max_tokens"),
    (dict(kv_heads=2, pages=4, colour=1), "unknown key colour"),
    (dict(kv_heads=2, pages=4, sequences=1024, max_tokens=1 << 26, page_tokens=16), "2\\^31 or more"),
    (dict(kv_heads=1024, pages=4, layers=4096, page_tokens=128), "4 GB or more"),
])
def test_bad_cache_options(options, words):
    with pytest.raises(TritError, match=words):
        KvCache(**options)


def test_null_arguments():
    lib = lm.library()
    assert lib.trit_cuda_kv_new(None) is None
    assert "kv_heads" in lib.trit_cuda_last_error().decode()
    assert lib.trit_cuda_kv_new(b"[1]") is None
    assert "not a JSON object" in lib.trit_cuda_last_error().decode()
    lib.trit_cuda_kv_free(None)
    out = (ctypes.c_int32 * 1)()
    for call in (lambda: lib.trit_cuda_kv_open(None, 1, out), lambda: lib.trit_cuda_kv_release(None, out, 1),
                 lambda: lib.trit_cuda_kv_length(None, 0), lambda: lib.trit_cuda_kv_compact(None, None)):
        assert call() == -1
        assert "kv is NULL" in lib.trit_cuda_last_error().decode()


def test_q4_0_arguments():
    lib = lm.library()
    assert lib.trit_dense_q4_0(None, 32, 32, 0, 0) is None
    assert "blocks" in lib.trit_cuda_last_error().decode()
    with pytest.raises(TritError, match="Q4_0 blocks of a 4x64"):
        Dense.q4_0(np.zeros(4 * 2 * 18 - 1, np.uint8), 4, 64)
    with pytest.raises(TritError, match="whole blocks of 32"):
        Dense.q4_0(np.zeros(4 * 1 * 18, np.uint8), 4, 48)
    with pytest.raises(TritError, match="whole blocks of 32"):
        Dense.q4_0(np.zeros(0, np.uint8), 0, 32)


@pytest.mark.parametrize("options, words", [
    (b'{"kv": "q4"}', 'kv is "f16", "f32" or "q8"'),
    (b'{"kv": "q8", "page_tokens": 48}', "page_tokens is 16, 32, 64 or 128"),
    (b'{"kv": "q8", "exact": false, "tc_attention": true}', "tc_attention"),
])
def test_bad_cache_options_of_a_model(options, words):
    lib = lm.library()
    assert lib.trit_lm_load(b"/nonexistent/model", options) is None
    assert words in lib.trit_cuda_last_error().decode()
