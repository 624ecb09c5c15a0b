"""The paged attention's count of a batch's work, run on the CPU against the same count in Python."""
import ctypes as C
import subprocess
from pathlib import Path

import numpy as np
import pytest

from minfer_b200 import build


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    so = tmp_path_factory.mktemp("paged_counts") / "counts.so"
    cmd = [build.nvcc(), *build.NVCC_FLAGS, "-shared", "-o", str(so), str(Path(__file__).parent / "paged_counts.cu")]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    lib = C.CDLL(str(so))
    lib.head_work.restype = C.c_longlong
    return lib


def head_work(RT, KT, n, first, G, window):
    """One unit for each item of at most RT rows, and one for each KT-key tile that its rows see (at least one)."""
    rows = n * G
    items = -(-rows // RT)
    step = RT if items <= 1 else min(-(-(-(-rows // items)) // 8) * 8, RT)
    r = np.arange(0, rows, step, dtype=np.int64)
    last = (np.minimum(r + step, rows) - 1) // G
    hi = np.maximum(first + last + 1, 0)
    lo = np.minimum(np.maximum(first + r // G - window + 1, 0), hi) if window else 0 * hi
    return int((1 + np.maximum((hi + KT - 1) // KT - lo // KT, 1)).sum())


SHAPES = [(16, 64), (32, 64), (64, 64), (16, 128), (32, 128)]


@pytest.mark.parametrize("RT,KT", SHAPES)
@pytest.mark.parametrize("n,first,G,window", [(1, 0, 1, 0), (1, 8191, 8, 0), (5, 100, 8, 0), (333, 0, 3, 0), (333, 5667, 8, 1024), (40, -17, 4, 0), (7, -9, 2, 5),
                                              (4096, 126976, 8, 0), (65, 4031, 2, 1)])
def test_ordinary(lib, RT, KT, n, first, G, window):
    assert lib.head_work(RT, KT, n, first, G, window) == head_work(RT, KT, n, first, G, window)


@pytest.mark.parametrize("RT,KT", SHAPES)
@pytest.mark.parametrize("n,first,G", [(1_600_000, 0, 8), (400_000, 2 ** 31 - 256 - 400_000, 4)])
def test_more_work_than_32_bits_hold(lib, RT, KT, n, first, G):
    want = head_work(RT, KT, n, first, G, 0)
    assert want > 2 ** 31 - 1
    assert lib.head_work(RT, KT, n, first, G, 0) == want
