"""The paged operators from their definitions, in 64 bits: a plain loop over sequences (test infrastructure)."""
import math

import torch


class Batch:
    """A ragged batch over a paged cache on `device`. `seqs`: (new tokens, length with them) of each sequence. Every
    page row that holds no position of a sequence is NaN, so are the unused pages. `gap` rows in front of the first
    sequence and behind the last belong to nobody."""

    def __init__(self, seqs, hq, hkv, d, page, dtype, device="cuda", seed=0, nhd=False, gap=(0, 0), spare=2):
        g = torch.Generator(device=device)
        g.manual_seed(seed)
        self.seqs, self.hq, self.hkv, self.d, self.page, self.dtype, self.device = seqs, hq, hkv, d, page, dtype, device
        need = [max(0, -(-length // page)) for _, length in seqs]
        self.n_pages = sum(need) + spare
        ids = torch.randperm(self.n_pages, generator=g, device=device).tolist()
        self.max_pages = max(max(need), 1) + 1
        table = torch.full((len(seqs), self.max_pages), 1 << 30, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            for i in range(n):
                table[b, i] = ids[at]
                at += 1
        self.table = table.to(device)
        shape = (self.n_pages, page, hkv, d) if nhd else (self.n_pages, hkv, page, d)
        make = lambda: torch.full(shape, math.nan, dtype=dtype, device=device)  # noqa: E731
        k, v = make(), make()
        self.k, self.v = (k.transpose(1, 2), v.transpose(1, 2)) if nhd else (k, v)
        for b, (_, length) in enumerate(seqs):
            for i in range(need[b]):
                n = min(page, length - i * page)
                for p in (self.k, self.v):
                    p[table[b, i], :, :n] = torch.randn(hkv, n, d, generator=g, device=device).to(dtype)
        start = [gap[0]]
        for n, _ in seqs:
            start.append(start[-1] + n)
        self.total = start[-1] + gap[1]
        self.start = start
        self.q_start = torch.tensor(start, dtype=torch.int32, device=device)
        self.lens = torch.tensor([length for _, length in seqs], dtype=torch.int32, device=device)
        self.gen = g

    def q(self):
        return torch.randn(self.total, self.hq, self.d, generator=self.gen, device=self.device).to(self.dtype)

    def args(self):
        return self.k, self.v, self.table, self.q_start, self.lens


def attention(b, q, window=0, scale=None):
    """(o, bound) in 64 bits; bound: the largest error that the arithmetic allows, element by element.

    With u the rounding unit of a type (half of eps): the output's rounding is u_T |o|; p is rounded to the pages'
    type (16-bit kernels), u_T sum p|v|, which also bounds the effect on the sum of p; a score is a sum of d products
    in fp32, off by at most (d + 3) 2^-24 scale sum|q||k| (accumulation, scaling, base 2), which moves every p by that
    relative amount, twice (p and the sum); the exponential is off by 2^-21; n accumulated terms add at most
    (n + 8) 2^-24 of sum p|v|, twice (o and the sum), and a few rescalings."""
    scale = 1 / math.sqrt(b.d) if scale is None else scale
    out = torch.zeros(b.total, b.hq, b.d, dtype=torch.float64, device=b.device)
    bound = torch.zeros_like(out)
    u = torch.finfo(b.dtype).eps / 2
    up = 0.0 if b.dtype == torch.float32 else u
    f = 2.0 ** -24
    table = b.table.tolist()
    for s, (n, length) in enumerate(b.seqs):
        if n == 0:
            continue
        pos = torch.arange(length - n, length, device=b.device)
        key = torch.arange(max(length, 0), device=b.device)
        page_ok = torch.tensor([0 <= table[s][i] < b.n_pages for i in range(b.max_pages)], device=b.device)
        pages = torch.tensor([p if 0 <= p < b.n_pages else 0 for p in table[s]], device=b.device)
        k = b.k[pages[key // b.page], :, key % b.page].double().transpose(0, 1)  # [hkv, len, d]
        v = b.v[pages[key // b.page], :, key % b.page].double().transpose(0, 1)
        see = (key <= pos[:, None]) & page_ok[key // b.page]
        if window:
            see &= key > pos[:, None] - window
        dead = ~see.any(0)
        k, v = torch.where(dead[None, :, None], 0.0, k), torch.where(dead[None, :, None], 0.0, v)
        rows = slice(b.start[s], b.start[s] + n)
        for h in range(b.hq):
            kh, vh = k[h * b.hkv // b.hq], v[h * b.hkv // b.hq]
            qh = q[rows, h].double()
            w = (qh @ kh.T * scale).masked_fill(~see, -math.inf)
            m = w.amax(-1, keepdim=True) if len(key) else torch.full((n, 1), -math.inf, dtype=torch.float64, device=b.device)
            p = torch.exp(w - torch.where(m == -math.inf, 0.0, m))
            p = p / p.sum(-1, keepdim=True).clamp(min=1e-300)
            out[rows, h] = p @ vh
            a = p @ vh.abs()
            delta = ((qh.abs() @ kh.abs().T) * see).amax(-1, keepdim=True) * abs(scale) * (b.d + 3) * f if len(key) else 0.0
            bound[rows, h] = u * out[rows, h].abs() + a * (2 * up + 2 * delta + 2.0 ** -20 + 2 * (len(key) + 8) * f) + 1e-30
            if b.dtype == torch.float16:
                bound[rows, h] += 2.0 ** -25  # subnormal outputs
    return out, bound


def rope(b, qkv, freqs, interleaved=False, mscale=1.0, qw=None, kw=None, eps=1e-6, positions=None):
    """(q_out, k_pages, v_pages) in 64 bits, NaN where nothing is written."""
    hq, hkv, d = b.hq, b.hkv, b.d
    r = 2 * len(freqs)
    q_out = torch.full((b.total, hq, d), math.nan, dtype=torch.float64, device=b.device)
    kp, vp = (torch.full(tuple(b.k.shape), math.nan, dtype=torch.float64, device=b.device) for _ in range(2))
    j = torch.arange(r // 2, device=b.device)
    lo, hi = (2 * j, 2 * j + 1) if interleaved else (j, j + r // 2)
    table = b.table.tolist()
    for s, (n, length) in enumerate(b.seqs):
        for i in range(n):
            t, pos = b.start[s] + i, length - n + i
            x = qkv[t].double().view(hq + 2 * hkv, d).clone()
            for heads, w in ((slice(0, hq), qw), (slice(hq, hq + hkv), kw)):
                if w is not None:
                    x[heads] = x[heads] / torch.sqrt((x[heads] ** 2).mean(-1, keepdim=True) + eps) * w.double()
            at = int(positions[t]) if positions is not None else pos
            ang = 2 * math.pi * torch.fmod(at * freqs, 1.0)
            y = x[:hq + hkv].clone()
            y[:, lo] = mscale * (x[:hq + hkv, lo] * torch.cos(ang) - x[:hq + hkv, hi] * torch.sin(ang))
            y[:, hi] = mscale * (x[:hq + hkv, hi] * torch.cos(ang) + x[:hq + hkv, lo] * torch.sin(ang))
            q_out[t] = y[:hq]
            if 0 <= pos < b.max_pages * b.page and 0 <= table[s][pos // b.page] < b.n_pages:
                kp[table[s][pos // b.page], :, pos % b.page] = y[hq:]
                vp[table[s][pos // b.page], :, pos % b.page] = x[hq + hkv:]
    return q_out, kp, vp
