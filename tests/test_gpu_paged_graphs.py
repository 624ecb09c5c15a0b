"""Captured steps of batches that mix chunks and single tokens (several kernels that start before the one before them
has ended): replays with new lengths, tables and inputs, two at once, against the same calls one at a time."""
import pytest
import torch

from minfer_b200 import ops
import paged_ref as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def _device(gpu):
    return gpu


class Step:
    """Two layers of a step over one batch, with buffers of its own."""

    def __init__(self, b, seed, **kw):
        self.b, self.kw, self.seed = b, kw, seed
        self.table, self.lens = b.table.clone(), b.lens.clone()
        self.caches = [(b.k.clone(), b.v.clone()) for _ in range(2)]
        self.qkv = [torch.zeros(b.total, (b.hq + 2 * b.hkv) * b.d, device="cuda") for _ in range(2)]
        self.q = torch.zeros(b.total, b.hq, b.d, dtype=b.dtype, device="cuda")
        self.outs = [torch.zeros_like(self.q) for _ in range(2)]
        n = ops.paged_attention_workspace_bytes(b.total, b.hq, b.hkv, b.d, b.dtype)
        self.ws = torch.empty(n, dtype=torch.uint8, device="cuda")
        self.f = ops.rope_freqs(b.d, 1e6)[0].cuda()

    def new_inputs(self, turn):
        g = torch.Generator(device="cuda")
        g.manual_seed(100 * self.seed + turn)
        for x in self.qkv:
            x.normal_(generator=g)
        self.lens.copy_((self.b.lens - turn % 3).clamp(min=0))
        self.table.copy_(self.b.table)
        if turn % 2:
            self.table[0, 0] = -1  # a page that is given away

    def run(self, between=lambda: None):
        b = self.b
        for (k, v), qkv, out in zip(self.caches, self.qkv, self.outs):
            ops.paged_rope_append(self.q, k, v, self.table, qkv, b.q_start, self.lens, self.f)
            between()
            ops.paged_attention(out, self.q, k, v, self.table, b.q_start, self.lens, workspace=self.ws, **self.kw)
            between()

    def state(self):
        return [x.nan_to_num(9.0).clone() for x in (*self.outs, *self.caches[0], *self.caches[1])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16], ids=["f32", "f16", "bf16"])
@pytest.mark.parametrize("hint", [False, True], ids=["", "hints"])
def test_mixed_batches_replayed_two_at_once(dtype, hint):
    batches = [[(70, 900), (1, 2500), (1, 33), (130, 130), (0, 0), (3, 700)], [(1, 4000), (40, 41), (1, 1), (200, 3000), (2, 900)]]
    pairs = []
    for seed, seqs in enumerate(batches):
        kw = dict(max_new=max(n for n, _ in seqs), max_len=max(n for _, n in seqs)) if hint else {}
        captured, plain = (Step(ref.Batch(seqs, 8, 2, 128, 16, dtype, seed=seed), seed, **kw) for _ in range(2))
        stream = torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            captured.run()
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            captured.run()
        pairs.append((captured, plain, stream, graph))
    for turn in range(6):
        for captured, plain, _, _ in pairs:
            captured.new_inputs(turn)
            plain.new_inputs(turn)
            captured.caches = [(k.copy_(plain.b.k), v.copy_(plain.b.v)) for k, v in captured.caches]
            plain.caches = [(k.copy_(plain.b.k), v.copy_(plain.b.v)) for k, v in plain.caches]
        torch.cuda.synchronize()
        for _ in range(3):  # the same step again and again, the two graphs beside each other
            for _, _, stream, graph in pairs:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for captured, plain, _, _ in pairs:
            plain.run(torch.cuda.synchronize)
            for got, want in zip(captured.state(), plain.state()):
                assert torch.equal(got, want)
    assert ops.paged_status() == 0
