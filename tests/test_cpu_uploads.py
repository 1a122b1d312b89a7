"""Copies and fills that kernels of non-blocking streams read behind: such a stream does not wait for the default one, on
which a plain cudaMemcpy of pageable memory (it may return before its last bytes are there) and a cudaMemset run."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "trit_b200", "csrc")
FILES = sorted(f for kind in ("*.cu", "*.cpp", "*.cuh", "*.h") for f in glob.glob(os.path.join(CSRC, kind)))


@pytest.mark.parametrize("path", FILES, ids=[os.path.basename(f) for f in FILES])
def test_uploads_are_in_their_streams_order(path):
    text = re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)
    plain = [m.group(0) for m in re.finditer(r"\bcudaMemcpy\s*\([^;]*;", text) if "DeviceToHost" not in m.group(0)]
    assert not plain, plain
    # A fill on the default stream is waited for before anything else can run.
    for m in re.finditer(r"\bcudaMemset\s*\(", text):
        behind = text[m.start():].split("}", 1)[0]
        assert "cudaDeviceSynchronize" in behind, behind
