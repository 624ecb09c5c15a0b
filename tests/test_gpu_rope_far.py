"""Rotary append at far positions, against angles in exact arithmetic."""
import math
from fractions import Fraction

import pytest
import torch

from minfer_b200 import ops
import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(gpu):
    return gpu


def turns(pos, f):
    """pos * f less the nearest whole number, rounded once."""
    t = pos * Fraction(f)
    return float(t - round(t))


@pytest.mark.parametrize("interleaved", [False, True], ids=["half", "pairs"])
@pytest.mark.parametrize("far", [2 ** 31 - 1, 10 ** 9])
def test_far_angles_are_exact(far, interleaved):
    """Vectors (1, 0) at positions where the first pair has turned nearly a whole number of times: its sine is small,
    so any error of the angle beyond its rounding to a float shows.

    With t the angle in turns: t is rounded to a float (2 pi |t| 2^-24 in the angle), sine and cosine are good to one
    unit in the last place (2^-23), the products and their sum round three times (2^-24 each of the result)."""
    f = ops.rope_freqs(128, 1e6)[0]
    pos = sorted(range(far - 20000, far + 1), key=lambda p: abs(turns(p, f[0].item())))[:8]
    b = ref.Batch([(8, 40)], 2, 1, 128, 16, torch.float32, seed=1)
    first = slice(0, 128, 2) if interleaved else slice(0, 64)
    second = slice(1, 128, 2) if interleaved else slice(64, 128)
    qkv = torch.zeros(8, 4, 128, device="cuda")
    qkv[:, :, first] = 1
    q = torch.empty(8, 2, 128, device="cuda")
    ops.paged_rope_append(q, *b.args()[:3], qkv.view(8, -1), b.q_start, b.lens, f.cuda(), interleaved=interleaved,
                          positions=torch.tensor(pos, dtype=torch.int32, device="cuda"))
    t = torch.tensor([[turns(p, x) for x in f.tolist()] for p in pos], dtype=torch.float64, device="cuda")[:, None]
    c, s = torch.cos(2 * math.pi * t), torch.sin(2 * math.pi * t)
    at = torch.arange(32, 40, device="cuda")
    k = b.k[b.table[0, at // 16].long(), :, at % 16]
    for x in (q, k):
        for got, want, other in ((x[..., first], c, s), (x[..., second], s, c)):
            bound = 2 * math.pi * t.abs() * 2.0 ** -24 * other.abs() + (2.0 ** -23 + 3 * 2.0 ** -24) * want.abs() + 1e-15
            assert ((got.double() - want).abs() <= bound).all()
