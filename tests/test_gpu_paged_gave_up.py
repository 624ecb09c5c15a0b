"""Paged attention where a wait gave up: rows without all their parts stay unwritten, and no others do. The joining
kernels get parts that the test made, some of them marked as the attention kernels mark what they did not finish."""
import ctypes as C
import math
import subprocess
from pathlib import Path

import pytest
import torch

from minfer_b200 import build

pytestmark = pytest.mark.gpu
SENTINEL = 77.0
GAVE_UP = -1.0  # PAGED_GAVE_UP


@pytest.fixture(scope="module")
def lib(gpu, tmp_path_factory):
    so = tmp_path_factory.mktemp("paged_join") / "join.so"
    cmd = [build.nvcc(), *build.NVCC_FLAGS, "-shared", "-o", str(so), str(Path(__file__).parent / "paged_join.cu"), "-lcuda"]
    r = subprocess.run(cmd, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return C.CDLL(str(so))


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def address(t):
    return C.c_void_p(t.data_ptr())


def divided(lens, grid):
    """(sequence, first CTA, last CTA) of every item that a cut divides, for one row tile of one head each: an item is
    one unit and its 128-key tiles, the units are cut into equal ranges, and CTAs share its tiles."""
    tiles = [max(1, math.ceil(n / 128)) for n in lens]
    share = math.ceil(sum(1 + t for t in tiles) / grid)
    start, items = 0, []
    for b, t in enumerate(tiles):
        first, last = (start + 1) // share, (start + t) // share
        if last > first:
            items.append((b, first, last))
        start += 1 + t
    return items


@pytest.mark.parametrize("grid", [2, 7, 40])
def test_parts_of_divided_items(lib, grid):
    lens = [5000, 3, 900, 128, 20000, 129, 64, 7000]
    n, G = len(lens), 4
    g = torch.Generator(device="cuda")
    g.manual_seed(grid)
    o = torch.randn(2 * grid, 16, 64, generator=g, device="cuda")
    ml = torch.rand(2 * grid, 16, 2, generator=g, device="cuda") + 0.5
    q_start, kv_lens = ints(list(range(n + 1))), ints(lens)

    def join(ml):
        out = torch.full((n, G, 64), SENTINEL, dtype=torch.bfloat16, device="cuda")
        part = torch.cat([o.flatten(), ml.flatten()])
        assert lib.join_few(address(out), address(part), address(q_start), address(kv_lens), n, n, 1, G, grid) == 0
        return out

    items = divided(lens, grid)
    good = join(ml)
    written = [b for b, _, _ in items]
    assert items and (good[written] != SENTINEL).all() and (good[[b for b in range(n) if b not in written]] == SENTINEL).all()
    for cta in range(grid):
        marked = ml.clone()
        marked[2 * cta:2 * cta + 2, :, 0] = 0
        marked[2 * cta:2 * cta + 2, :, 1] = GAVE_UP
        out = join(marked)
        for b, first, last in items:
            want = torch.full_like(good[b], SENTINEL) if first <= cta <= last else good[b]
            assert torch.equal(out[b], want), (cta, b)


def test_parts_of_split_chunks(lib):
    n, G, hkv, split = 70, 4, 2, 5
    g = torch.Generator(device="cuda")
    g.manual_seed(1)
    o = torch.randn(split, n * hkv * G, 64, generator=g, device="cuda")
    ml = torch.rand(split, n * hkv * G, 2, generator=g, device="cuda") + 0.5
    q_start, kv_lens = ints([0, n]), ints([900])

    def join(ml):
        out = torch.full((n * hkv * G, 64), SENTINEL, dtype=torch.bfloat16, device="cuda")
        assert lib.join_chunks(address(out), address(o), address(ml), address(q_start), address(kv_lens), 1, n, hkv, G, split) == 0
        return out

    good = join(ml)
    assert (good != SENTINEL).all()
    gone = torch.rand(split, n * hkv * G, generator=g, device="cuda") < 0.05
    marked = ml.clone()
    marked[gone] = torch.tensor([0.0, GAVE_UP], device="cuda")
    out = join(marked)
    gone = gone.any(0)
    assert (out[gone] == SENTINEL).all() and torch.equal(out[~gone], good[~gone])
