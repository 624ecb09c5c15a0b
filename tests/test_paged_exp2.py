"""The polynomial of the chunk kernel's exponential (paged_fa.cuh): its stated error is what its coefficients give."""
import re
from pathlib import Path

import numpy as np

SOURCE = (Path(__file__).resolve().parent.parent / "minfer_b200" / "csrc" / "paged_fa.cuh").read_text()


def test_stated_error_of_the_exponential():
    body = SOURCE[SOURCE.index("float2 pf_exp2_fma"):]
    body = body[:body.index("\n}\n")]
    c = [np.float32(x) for x in re.findall(r"q = pf_(?:two\(|fma2\(q, r, pf_two\()([0-9.e+-]+)f,", body)]
    assert len(c) == 6
    exact, rounded = (2.0 ** -float(x) for x in re.search(r"2\^-([0-9.]+) in\n// exact arithmetic, 2\^-([0-9.]+) with every step rounded", SOURCE).groups())
    r = np.linspace(-0.5, 0.5, 1 << 21).astype(np.float32)
    x, want = r.astype(np.float64), np.exp2(r.astype(np.float64))
    q64, q32 = np.full_like(x, c[0]), np.full_like(r, c[0])
    for k in c[1:]:
        q64 = q64 * x + float(k)
        q32 = (q32.astype(np.float64) * x + float(k)).astype(np.float32)  # one rounding: 48 bits of product fit
    assert np.abs(q64 / want - 1).max() <= exact
    assert np.abs(q32 / want - 1).max() <= rounded
