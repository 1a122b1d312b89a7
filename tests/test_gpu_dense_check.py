"""Dense.check: a product whose waits ran out is reported after it has ended. The failure is made on the host, in the status
word that a kernel would set."""
import ctypes

import numpy as np
import pytest

from trit_b200 import Dense, TritError

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


class Attributes(ctypes.Structure):
    _fields_ = [("type", ctypes.c_int), ("device", ctypes.c_int), ("device_pointer", ctypes.c_void_p), ("host_pointer", ctypes.c_void_p),
                ("reserved", ctypes.c_long * 8)]


def memory_of(address):
    """(CUDA's type of memory at an address: 1 host, 2 device; 0 none)."""
    at = Attributes()
    with open("/proc/self/maps") as f:
        path = next(line.split()[-1] for line in f if "libcudart.so" in line)
    return at.type if ctypes.CDLL(path).cudaPointerGetAttributes(ctypes.byref(at), ctypes.c_void_p(address)) == 0 else 0


def words(address, n):
    return np.frombuffer(ctypes.string_at(address, 8 * n), np.uint64).tolist()


def fp8():
    return Dense.fp8(np.full((256, 128), 0x38, np.uint8), np.ones((2, 1), np.float32), 256, 128)


def status_word(dense):
    """The one word of host memory that a layer's object points at (the handle holds the object in its second word)."""
    found = [w for w in words(words(dense._handle, 2)[1], 36) if w > 4096 and w % 4 == 0 and memory_of(w) == 1]
    assert len(found) == 1
    return ctypes.c_int.from_address(found[0])


def call(dense, rows=5):
    x, out = torch.ones(rows, dense.k, device="cuda"), torch.zeros(rows, dense.n, device="cuda")
    torch.cuda.synchronize()
    dense.forward_device(x.data_ptr(), rows, out.data_ptr())
    torch.cuda.synchronize()
    return out


def test_nothing_to_report():
    for dense in (fp8(), Dense.q8_0(np.zeros(256 * 4 * 34, np.uint8), 256, 128), Dense.q4_0(np.zeros(256 * 4 * 18, np.uint8), 256, 128),
                  Dense.q8_0(np.zeros(256 * 4 * 34, np.uint8), 256, 128, table=True)):
        dense.check()
        call(dense, 70)
        dense.check()


def test_reported_once():
    dense = fp8()
    word = status_word(dense)
    assert word.value == 0 and float(call(dense)[0, 0]) == 128.0
    word.value = 1
    with pytest.raises(TritError, match="gave up waiting"):
        dense.check()
    dense.check()
    assert word.value == 0 and float(call(dense)[0, 0]) == 128.0


def test_reported_by_the_next_call():
    dense = fp8()
    word = status_word(dense)
    word.value = 1
    with pytest.raises(TritError, match="gave up waiting"):
        call(dense)
    dense.check()
    assert float(call(dense)[0, 0]) == 128.0
