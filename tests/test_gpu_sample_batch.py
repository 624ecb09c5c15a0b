"""mf_sample_batch against the Sampler's rules in 64 bits: every filter, ties, NaN, infinities, borders, types, strides."""
import math

import numpy as np
import pytest
import torch

from minfer_b200 import ops
from minfer_b200._lib import MinferError

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(gpu):
    return gpu


def rule(x, r, temp, top_k, top_p, min_p):
    """(id, probability) of one row: the candidates sorted by value and index, cut by each filter in turn, in 64 bits."""
    x = np.where(np.isnan(x), -np.inf, x.astype(np.float64))
    if x.max() == -np.inf:
        return -1, 0.0
    ids = np.argsort(-x, kind="stable")
    v = x[ids]
    if not temp > 0:
        return int(ids[0]), 1.0
    z = np.where(v == v[0], 0.0, v - v[0])
    n = top_k if 0 < top_k < len(v) else len(v)
    if top_p < 1:
        c = np.cumsum(np.exp(z[:n]))
        n = min(n, 1 + int(np.searchsorted(c, max(top_p, 0.0) * c[-1], side="left")))
    if min_p > 0:
        n = min(n, max(1, int((v >= v[0] + math.log(min(min_p, 1.0))).sum())))
    w = np.exp(z[:n] / temp)
    c = np.cumsum(w)
    at = min(int(np.searchsorted(c, r * c[-1], side="left")), n - 1)
    return int(ids[at]), float(w[at] / c[-1])


def run(logits, r, temp, top_k, top_p, min_p, probs=True):
    n = logits.shape[0]
    f = lambda v, t=torch.float32: torch.as_tensor(v, dtype=t, device="cuda").expand(n).contiguous()  # noqa: E731
    ids = torch.full((n,), -7, dtype=torch.int32, device="cuda")
    p = torch.full((n,), -7.0, device="cuda") if probs else None
    a = (f(r), f(temp), f(top_k, torch.int32), f(top_p), f(min_p))
    ops.sample_batch(ids, logits, *a, probs=p)
    return ids.tolist(), p.tolist() if probs else None, [x.tolist() for x in a]


def check(logits, r, temp, top_k, top_p, min_p):
    ids, p, a = run(logits, r, temp, top_k, top_p, min_p)
    rows = logits.float().cpu().numpy()
    for i, row in enumerate(rows):
        want, prob = rule(row, *(x[i] for x in a))
        assert ids[i] == want, (i, ids[i], want, [x[i] for x in a])
        # a float of a quotient of sums that are exact to 2^-45 of the largest weight per candidate
        assert abs(p[i] - prob) <= 2.0 ** -23 * prob + 1e-12


FILTERS = [(1.0, 0, 1.0, 0.0), (0.7, 20, 0.9, 0.0), (1.0, 1, 1.0, 0.0), (1.5, 0, 0.5, 0.0), (0.3, 50, 1.0, 0.1), (2.0, 0, 1.0, 1.0),
           (1.0, 3, 0.0, 0.0), (0.0, 5, 0.5, 0.0), (5.0, 1000, 0.99, 1e-4), (1e-3, 0, 1.0, 0.0), (100.0, 0, 0.999999, 0.0)]


@pytest.mark.parametrize("temp,top_k,top_p,min_p", FILTERS)
@pytest.mark.parametrize("vocab", [1, 2, 31, 1024, 5000, 32003, 151936])
def test_filters(vocab, temp, top_k, top_p, min_p):
    g = torch.Generator(device="cuda")
    g.manual_seed(vocab + top_k)
    n = 6
    x = torch.randn(n, vocab, generator=g, device="cuda") * torch.tensor([0.01, 1.0, 3.0, 10.0, 2.0, 0.5], device="cuda")[:, None]
    r = torch.rand(n, generator=g, device="cuda")
    r[0], r[1] = 0.0, 0.99999994
    check(x, r, temp, top_k, top_p, min_p)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("temp,top_k,top_p,min_p", FILTERS)
def test_16_bit_logits_tie_often(dtype, temp, top_k, top_p, min_p):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x = (torch.randn(8, 40001, generator=g, device="cuda") * 2).to(dtype)
    check(x, torch.rand(8, generator=g, device="cuda"), temp, top_k, top_p, min_p)


@pytest.mark.parametrize("vocab", [1, 65, 1000, 4097, 20000, 262144])
def test_equal_logits(vocab):
    """All candidates equal: the filters count, the draw picks by index; borders fall on whole numbers."""
    x = torch.full((7, vocab), 1.25, device="cuda")
    r = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.99999994, 1e-7, 0.125], device="cuda")
    for top_k in (0, 1, vocab // 2 + 1):
        for top_p in (0.0, 0.5, 0.25, 1.0):
            check(x, r, 0.8, top_k, top_p, 0.0)
    x[:, vocab // 3:] = 1.0  # two values
    check(x, r, 0.8, 0, 0.5, 0.0)
    check(x, r, 3.0, vocab - 1, 1.0, 0.9)


def test_special_values():
    inf, nan = math.inf, math.nan
    x = torch.zeros(9, 300, device="cuda")
    x[0] = -inf
    x[1] = nan
    x[2] = -inf
    x[2, 17] = -1e30
    x[3, 5] = inf
    x[3, 9] = inf
    x[4, ::2] = nan
    x[5] = torch.finfo(torch.float32).min
    x[6] = -0.0
    x[6, 100] = 0.0
    x[7, 4] = torch.finfo(torch.float32).max
    x[8] = torch.finfo(torch.float32).tiny * torch.arange(300, device="cuda") * 1e-3
    for temp in (0.0, 1.0):
        for top_k, top_p, min_p in ((0, 1.0, 0.0), (3, 0.9, 0.0), (0, 0.7, 0.2), (299, 1.0, 0.0)):
            check(x, 0.6, temp, top_k, top_p, min_p)


def test_rows_are_independent():
    """Each row with its own parameters, against rows one at a time; strided and unaligned rows; without probs."""
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    n, vocab = 40, 9973
    wide = torch.randn(n, vocab + 13, generator=g, device="cuda") * 3
    x = wide[:, 3:3 + vocab]
    pick = lambda *v: torch.tensor(v, device="cuda")[torch.randint(0, len(v), (n,), generator=g, device="cuda")]  # noqa: E731
    r, temp, top_k = torch.rand(n, generator=g, device="cuda"), pick(0.0, 0.5, 1.0, 2.0), pick(0, -1, 1, 7, 100, 20000)
    top_p, min_p = pick(0.3, 0.9, 1.0, 1.5), pick(0.0, 0.02, 0.3)
    check(x, r, temp, top_k, top_p, min_p)
    ids, _, _ = run(x, r, temp, top_k, top_p, min_p, probs=False)
    for i in (0, 7, 39):
        one, _, _ = run(x[i:i + 1], r[i:i + 1], temp[i:i + 1], top_k[i:i + 1], top_p[i:i + 1], min_p[i:i + 1])
        assert one[0] == ids[i]


def test_bad_parameters_have_a_meaning():
    x = torch.tensor([[1.0, 3.0, 2.0]], device="cuda")
    assert run(x, 0.5, -1.0, 0, 1.0, 0.0)[0] == [1]  # no positive temperature: the first maximum
    assert run(x, 0.5, math.nan, 0, 1.0, 0.0)[0] == [1]
    assert run(x, 2.0, 1.0, 0, 1.0, 0.0)[0] == run(x, 0.99999994, 1.0, 0, 1.0, 0.0)[0]
    assert run(x, -1.0, 1.0, 0, 1.0, 0.0)[0] == [1]
    assert run(x, 0.9, 1.0, 0, -3.0, 0.0)[0] == [1]
    assert run(x, 0.9, 1.0, 0, 1.0, 7.0)[0] == [1]
    with pytest.raises(ValueError):
        ops.sample_batch(torch.zeros(1, dtype=torch.int64, device="cuda"), x, *[torch.zeros(1, device="cuda")] * 5)


def test_no_rows():
    ids = torch.empty(0, dtype=torch.int32, device="cuda")
    f = torch.empty(0, device="cuda")
    ops.sample_batch(ids, torch.empty(0, 100, device="cuda"), f, f, ids, f, f, probs=f)
    with pytest.raises(MinferError):  # rows that overlap
        x = torch.zeros(1, 9, device="cuda").expand(3, -1)
        ops.sample_batch(torch.zeros(3, dtype=torch.int32, device="cuda"), x, *[torch.zeros(3, device="cuda")] * 2, torch.zeros(3, dtype=torch.int32, device="cuda"),
                         *[torch.zeros(3, device="cuda")] * 2)


def test_crowded_bins():
    """Thousands of candidates within a sixteenth of the border: the descent that does not fit one block."""
    g = torch.Generator(device="cuda")
    g.manual_seed(6)
    x = 5 + torch.rand(4, 30000, generator=g, device="cuda") * 0.05
    x[1, :9000] = x[1, 0]
    x[2] = x[2].to(torch.bfloat16).float()
    x[3, ::3] -= 40
    r = torch.rand(4, generator=g, device="cuda")
    for temp, top_k, top_p, min_p in ((1.0, 0, 0.5, 0.0), (0.01, 0, 0.999, 0.0), (1.0, 12000, 1.0, 0.0), (2.0, 12000, 0.7, 0.97), (1.0, 0, 1.0, 0.98), (0.3, 29999, 0.3, 0.0)):
        check(x, r, temp, top_k, top_p, min_p)


def test_draws_follow_the_distribution():
    """The draw is the quantile of the cumulative distribution: a sweep of r walks the candidates in order."""
    x = torch.tensor([0.1, 2.0, -1.0, 1.0, 2.0, 0.5], device="cuda").expand(4096, 6).contiguous()
    check(x, torch.arange(4096, device="cuda") / 4096, 0.9, 5, 0.97, 0.01)


def test_graph_and_stream():
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x = torch.randn(5, 50000, generator=g, device="cuda") * 3
    r = torch.rand(5, generator=g, device="cuda")
    f = lambda v, t=torch.float32: torch.full((5,), v, dtype=t, device="cuda")  # noqa: E731
    temp, top_k, top_p, min_p, ids = f(0.8), f(40, torch.int32), f(0.95), f(0.0), f(-7, torch.int32)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ops.sample_batch(ids, x, r, temp, top_k, top_p, min_p)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        ops.sample_batch(ids, x, r, temp, top_k, top_p, min_p)
    for _ in range(3):
        x.normal_(0, 3)
        r.uniform_(0, 0.999)
        graph.replay()
        torch.cuda.synchronize()
        for i, row in enumerate(x.cpu().numpy()):
            assert ids[i].item() == rule(row, r[i].item(), temp[i].item(), 40, top_p[i].item(), 0.0)[0]
