"""The operators of one step of a batch of sequences over a paged KV cache: what is measured, and their plain forms.

`paged_rope_append` (Q/K norm, rotary positions, append), `paged_attention` (new tokens over the cached ones) and
`sample_batch` (one id per row of logits). `run` computes them in elementary torch operations, or through
`minfer_b200.ops` where `own` is set.
"""
import math
import random

import numpy as np
import torch

own = False

_T = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------- cases

def listed():
    rope = dict(op="rope", norm=True, mix=1)
    attn = dict(op="attn", d=128, window=0, mix=1)
    return [
        # one sequence's next token, the shape of the 8B model
        dict(rope, name="rope_decode_1", seqs=1, tokens=1, ctx=4096, hq=32, hkv=8, d=128, d_rot=128, page=16, x="f32",
             t="bf16", interleaved=False, scaling="none"),
        # a decode batch, half of the head rotated in the interleaved layout
        dict(rope, name="rope_decode_64_il", seqs=64, tokens=1, ctx=8192, hq=64, hkv=8, d=128, d_rot=64, page=64, x="f16",
             t="f16", interleaved=True, scaling="linear", norm=False),
        # prompt chunks far into a stretched context, the heads of the 32B model
        dict(rope, name="rope_chunk_long", seqs=3, tokens=2048, ctx=131072, hq=64, hkv=8, d=128, d_rot=128, page=64, x="f32",
             t="bf16", interleaved=False, scaling="yarn"),
        # one sequence decoding at the benchmark's context: the smallest call, latency counts
        dict(attn, name="attn_decode_1", seqs=1, tokens=1, ctx=4096, hq=32, hkv=8, page=16, t="bf16", ragged=False),
        # a decode batch of sequences of very different lengths
        dict(attn, name="attn_decode_32_ragged", seqs=32, tokens=1, ctx=32768, hq=64, hkv=8, page=64, t="bf16", ragged=True),
        # small heads without sharing, short sequences
        dict(attn, name="attn_decode_64_d64", seqs=64, tokens=1, ctx=2048, hq=16, hkv=16, d=64, page=32, t="f16", ragged=True),
        # a whole prompt at once
        dict(attn, name="attn_prompt_4096", seqs=1, tokens=4096, ctx=4096, hq=32, hkv=8, page=64, t="bf16", ragged=False),
        # a chunk of a prompt late in a long context
        dict(attn, name="attn_chunk_512", seqs=1, tokens=512, ctx=29184, hq=64, hkv=8, page=64, t="bf16", ragged=False),
        # chunks and single tokens in one batch, pages that are no power of two, a sliding window
        dict(attn, name="attn_mixed_window", seqs=12, tokens=333, ctx=6000, hq=32, hkv=4, page=24, t="f16", ragged=True,
             window=1024),
        # the cache as the reference keeps it, in 32 bits
        dict(attn, name="attn_f32", seqs=4, tokens=65, ctx=4096, hq=16, hkv=8, page=16, t="f32", ragged=True),
        # one row of the vocabulary, the sampled decode of one sequence
        dict(op="sample", name="sample_1", rows=1, vocab=151936, t="f32"),
        # a serving batch, each row with its own parameters
        dict(op="sample", name="sample_64", rows=64, vocab=151936, t="f32"),
    ]


def _spread(rng, lo, hi):
    """A whole number in [lo, hi], spread evenly over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "attn", "attn", "sample"])
    mix = rng.randrange(1 << 20)
    if op == "sample":
        vocab = rng.choice([151936, _spread(rng, 1000, 200000)])
        return dict(op=op, rows=min(_spread(rng, 1, 128), 64 * 151936 // vocab), vocab=vocab, t=rng.choice(["f32", "f32", "bf16", "f16"]))
    hq, hkv = rng.choice([(16, 8), (32, 8), (32, 4), (64, 8), (4, 2), (16, 2), (12, 4), (8, 8), (20, 4)])
    d = rng.choice([128, 128, 64])
    page = rng.choice([16, 32, 64, 128, 8, 24, 48, 80])
    if op == "rope":
        t = rng.choice(["bf16", "bf16", "f16", "f32"])
        return dict(op=op, seqs=_spread(rng, 1, 48), tokens=rng.choice([1, _spread(rng, 2, 128)]), ctx=_spread(rng, 256, 100000),
                    hq=hq, hkv=hkv, d=d, d_rot=rng.choice([d, d, d // 2, d - 16]), page=page, x=rng.choice(["f32", t]), t=t,
                    interleaved=rng.random() < 0.4, scaling=rng.choice(["none", "linear", "ntk", "yarn"]), norm=rng.random() < 0.6, mix=mix)
    case = dict(op=op, hq=hq, hkv=hkv, d=d, page=page, mix=mix, window=rng.choice([0, 0, 0, _spread(rng, 16, 4096)]), ragged=rng.random() < 0.7)
    if rng.random() < 0.5:  # single tokens, or a few of each sequence
        t = rng.choice(["bf16", "bf16", "f16", "f32"])
        seqs = _spread(rng, 1, 64)
        return dict(case, seqs=seqs, tokens=rng.choice([1, 1, 1, rng.randrange(2, 6)]), t=t,
                    ctx=_spread(rng, 16, min(32768, 262144 // seqs)))
    t = rng.choice(["bf16", "bf16", "f16", "f32"])
    seqs = _spread(rng, 1, 4)
    tokens = _spread(rng, 16, (256 if t == "f32" else 2048) // seqs)
    return dict(case, seqs=seqs, tokens=tokens, t=t, ctx=tokens + _spread(rng, 1, (2048 if t == "f32" else 8192) // seqs))


def _lengths(case):
    """(new tokens, length with them) of each sequence of the batch: plain numbers that a scheduler has. A ragged batch
    mixes chunks, single tokens and lengths from one key on; its first sequence is the longest."""
    r = random.Random(case["mix"])
    new, lens = [], []
    for b in range(case["seqs"]):
        n, length = case["tokens"], case["ctx"]
        if case.get("ragged", True) and b:
            n = r.choice([1, r.randint(1, n)])
            length = r.randint(n, length)
        new.append(n)
        lens.append(length)
    return new, lens


# ---------------------------------------------------------------- state

def _freqs(d_rot, base, scaling, factor=4.0, orig=32768):
    """Turns per position of each pair, in 64 bits, and the magnitude: as published for each kind of scaling."""
    j = torch.arange(d_rot // 2, dtype=torch.float64)
    if scaling == "ntk":
        base = base * factor ** (d_rot / (d_rot - 2))
    f = base ** (-2.0 * j / d_rot)
    mag = 1.0
    if scaling == "linear":
        f = f / factor
    elif scaling == "yarn":
        at = [d_rot * math.log(orig / (turns * 2 * math.pi)) / (2 * math.log(base)) for turns in (32.0, 1.0)]
        lo, hi = max(math.floor(at[0]), 0), min(math.ceil(at[1]), d_rot - 1)
        ramp = ((j - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        f = f / factor * ramp + f * (1 - ramp)
        mag = 0.1 * math.log(factor) + 1.0
    return f / (2 * math.pi), mag


def _batch(case, gen):
    new, lens = _lengths(case)
    page, seqs = case["page"], case["seqs"]
    need = [-(-n // page) for n in lens]
    start = [0]
    for n in new:
        start.append(start[-1] + n)
    n_pages = sum(need) + 3  # pages in any order, a few of them free
    ids = torch.randperm(n_pages, generator=gen, device="cuda").to(torch.int32)
    width = max(need)
    at = torch.tensor(need, device="cuda").cumsum(0) - torch.tensor(need, device="cuda")
    col = torch.arange(width, device="cuda")
    table = ids[(at[:, None] + col).clamp(max=n_pages - 1)]
    table = torch.where(col < torch.tensor(need, device="cuda")[:, None], table, torch.zeros_like(table)).contiguous()
    return dict(case=case, n_pages=n_pages, total=start[-1], max_new=max(new), max_len=max(lens), page_table=table,
                q_start=torch.tensor(start, dtype=torch.int32, device="cuda"),
                kv_lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), seqs=seqs)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    normal = lambda *shape, t=torch.float32: torch.randn(*shape, generator=gen, device="cuda", dtype=t)  # noqa: E731
    if case["op"] == "sample":
        rows, vocab = case["rows"], case["vocab"]
        # a wide body and a few likely tokens, as a model's logits have
        logits = normal(rows, vocab) * 2.5
        likely = torch.randint(0, vocab, (rows, 24), generator=gen, device="cuda")
        logits.scatter_add_(1, likely, torch.rand(rows, 24, generator=gen, device="cuda") * 9)
        pick = lambda *values: torch.tensor(values, device="cuda")[torch.randint(0, len(values), (rows,), generator=gen, device="cuda")]  # noqa: E731
        return dict(case=case, logits=logits.to(_T[case["t"]]), draws=torch.rand(rows, generator=gen, device="cuda"),
                    temp=pick(0.0, 0.6, 0.7, 1.0, 1.0, 1.5), top_k=pick(0, 20, 50, 1000).to(torch.int32), top_p=pick(0.8, 0.9, 0.95, 1.0),
                    min_p=pick(0.0, 0.0, 0.05, 0.1), ids=torch.zeros(rows, dtype=torch.int32, device="cuda"), probs=torch.zeros(rows, device="cuda"))
    s = _batch(case, gen)
    t, hq, hkv, d = _T[case["t"]], case["hq"], case["hkv"], case["d"]
    s["k_pages"] = normal(s["n_pages"], hkv, case["page"], d, t=t)
    s["v_pages"] = normal(s["n_pages"], hkv, case["page"], d, t=t)
    if case["op"] == "rope":
        s["qkv"] = (normal(s["total"], (hq + 2 * hkv) * d) * 1.5).to(_T[case["x"]])
        f, s["mscale"] = _freqs(case["d_rot"], 1e6, case["scaling"])
        s["freqs"] = f.cuda()
        s["q_norm_w"], s["k_norm_w"] = ((1 + 0.2 * normal(d), 1 + 0.2 * normal(d)) if case["norm"] else (None, None))
        s["q_out"] = torch.zeros(s["total"], hq, d, dtype=t, device="cuda")
    else:
        s["q"] = normal(s["total"], hq, d).to(t)
        s["out"] = torch.zeros(s["total"], hq, d, dtype=t, device="cuda")
    return s


# ---------------------------------------------------------------- plain forms

_EPS = 1e-6


def _owner(s):
    """Sequence and position of every new token."""
    tok = torch.arange(s["total"], device="cuda")
    seq = torch.searchsorted(s["q_start"][1:].long().contiguous(), tok, right=True)
    return seq, (s["kv_lens"].long() - s["q_start"][1:].long())[seq] + tok


def _plain_rope(s):
    c = s["case"]
    hq, hkv, d, r = c["hq"], c["hkv"], c["d"], c["d_rot"]
    x = s["qkv"].float().view(-1, hq + 2 * hkv, d)
    q, k, v = x[:, :hq], x[:, hq:hq + hkv], x[:, hq + hkv:]
    if c["norm"]:
        q = q * torch.rsqrt(q.square().mean(-1, keepdim=True) + _EPS) * s["q_norm_w"]
        k = k * torch.rsqrt(k.square().mean(-1, keepdim=True) + _EPS) * s["k_norm_w"]
    seq, pos = _owner(s)
    turns = pos.double()[:, None] * s["freqs"]  # 64 bits: far positions
    angle = 2 * math.pi * (turns - torch.round(turns))
    cos, sin = (s["mscale"] * torch.cos(angle)).float()[:, None], (s["mscale"] * torch.sin(angle)).float()[:, None]

    def turn(y):
        a, b = (y[..., 0:r:2], y[..., 1:r:2]) if c["interleaved"] else (y[..., :r // 2], y[..., r // 2:r])
        a, b = a * cos - b * sin, b * cos + a * sin
        rot = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([rot, y[..., r:]], -1)

    t = s["k_pages"].dtype
    slot, row = s["page_table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["k_pages"][slot, :, row] = turn(k).to(t)
    s["v_pages"][slot, :, row] = v.to(t)
    return turn(q).to(t), s["k_pages"], s["v_pages"]


def _plain_attn(s):
    c = s["case"]
    hq, hkv, d, b, n = c["hq"], c["hkv"], c["d"], s["seqs"], s["max_new"]
    g = hq // hkv
    start, lens = s["q_start"][:-1].long(), s["kv_lens"].long()
    new = s["q_start"][1:].long() - start
    i = torch.arange(n, device="cuda")
    q = s["q"].float()[(start[:, None] + i).clamp(max=s["total"] - 1)]  # [b, n, hq, d], each sequence padded to the longest
    q = q.view(b, n, hkv, g, d).permute(0, 2, 1, 3, 4).reshape(b, hkv, n * g, d)
    pages = s["page_table"].long()
    keys = lambda x: x[pages].float().permute(0, 2, 1, 3, 4).reshape(b, hkv, -1, d)  # noqa: E731
    k, v = keys(s["k_pages"]), keys(s["v_pages"])
    at = torch.arange(k.shape[2], device="cuda")
    pos = (lens - new)[:, None] + i
    see = at <= pos[..., None]  # [b, n, keys]
    if c["window"]:
        see &= at > pos[..., None] - c["window"]
    w = (q @ k.transpose(-1, -2)) * (1 / math.sqrt(d))
    w.masked_fill_(~see.repeat_interleave(g, 1)[:, None], -math.inf)
    w = torch.exp(w - w.amax(-1, keepdim=True).clamp(min=-1e30))
    o = (w @ v) / w.sum(-1, keepdim=True).clamp(min=1e-30)
    o = o.view(b, hkv, n, g, d).permute(0, 2, 1, 3, 4).reshape(b, n, hq, d)
    seq, _ = _owner(s)
    return o[seq, torch.arange(s["total"], device="cuda") - start[seq]].to(s["q"].dtype)


def _plain_sample(s):
    x = s["logits"].float()
    rows, vocab = x.shape
    v, ids = torch.sort(x, dim=-1, descending=True, stable=True)  # equal values: the lower index first
    v = v.double()  # sums over the vocabulary, borders of the filters
    top, temp = v[:, :1], s["temp"].double()[:, None]
    rank = torch.arange(vocab, device="cuda")
    k = torch.where((s["top_k"] <= 0) | (s["top_k"] > vocab), vocab, s["top_k"])[:, None]
    top_p, min_p = s["top_p"].double()[:, None], s["min_p"].double()[:, None]
    w = torch.where(rank < k, torch.exp(v - top), 0.0)
    before = (w.cumsum(-1) < top_p * w.sum(-1, keepdim=True)).sum(-1, keepdim=True)
    kept = torch.where(top_p < 1, torch.minimum(before + 1, k), k)
    keep = (rank < kept) & ((v >= top + torch.log(min_p)) | (min_p <= 0))
    w = torch.where(keep, torch.exp((v - top) / torch.where(temp > 0, temp, 1.0)), 0.0)
    total = w.sum(-1, keepdim=True)
    at = (w.cumsum(-1) < s["draws"].double()[:, None] * total).sum(-1, keepdim=True)
    at = torch.minimum(at, keep.sum(-1, keepdim=True) - 1)
    at = torch.where(temp > 0, at, 0)
    prob = torch.where(temp > 0, w.gather(1, at) / total, 1.0)
    return ids.gather(1, at)[:, 0].to(torch.int32), prob[:, 0].float()


def run(state):
    c = state["case"]
    if own:
        from minfer_b200 import ops

        if c["op"] == "rope":
            ops.paged_rope_append(state["q_out"], state["k_pages"], state["v_pages"], state["page_table"], state["qkv"], state["q_start"],
                                  state["kv_lens"], state["freqs"], interleaved=c["interleaved"], mscale=state["mscale"],
                                  q_norm_w=state["q_norm_w"], k_norm_w=state["k_norm_w"], eps=_EPS)
            return state["q_out"], state["k_pages"], state["v_pages"]
        if c["op"] == "attn":
            ops.paged_attention(state["out"], state["q"], state["k_pages"], state["v_pages"], state["page_table"], state["q_start"],
                                state["kv_lens"], window=c["window"], max_new=state["max_new"], max_len=state["max_len"])
            return state["out"]
        ops.sample_batch(state["ids"], state["logits"], state["draws"], state["temp"], state["top_k"], state["top_p"], state["min_p"],
                         probs=state["probs"])
        return state["ids"], state["probs"]
    if c["op"] == "rope":
        return _plain_rope(state)
    return _plain_attn(state) if c["op"] == "attn" else _plain_sample(state)


# ---------------------------------------------------------------- work

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2}
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * size[case["t"]] + 28), "flops": 2 * case["rows"] * case["vocab"]}
    new, lens = _lengths(case)
    hq, hkv, d, t = case["hq"], case["hkv"], case["d"], size[case["t"]]
    if case["op"] == "rope":
        n = sum(new) * (hq + 2 * hkv) * d
        return {"bytes": n * (size[case["x"]] + t), "flops": 6 * n}
    keys = pairs = 0
    for n, length in zip(new, lens):
        first = length - n  # position of the first new token
        w = case["window"] or length
        keys += length - max(0, first - w + 1)
        full = min(n, max(0, w - first - 1))  # tokens whose window still reaches the first key
        pairs += full * first + full * (full + 1) // 2 + (n - full) * w
    return {"bytes": keys * 2 * hkv * d * t + 2 * sum(new) * hq * d * t, "flops": 4 * d * hq * pairs}


# ---------------------------------------------------------------- 64 bits

def _exact_sample(s):
    """Row by row on the host: the candidates in order, cut by each filter in turn. An id is a whole number; its
    probability is what 64 bits say."""
    probs = []
    rows = zip(s["logits"].double().cpu().numpy(), *(s[k].cpu().double().tolist() for k in ("draws", "temp", "top_k", "top_p", "min_p")))
    for x, r, temp, top_k, top_p, min_p in rows:
        x = -np.sort(-x)
        if temp == 0:
            probs.append(1.0)
            continue
        if 0 < top_k < x.size:
            x = x[:int(top_k)]
        if top_p < 1:
            c = np.cumsum(np.exp(x - x[0]))
            x = x[:1 + int(np.searchsorted(c, top_p * c[-1], side="left"))]
        if min_p > 0:
            x = x[np.exp(x - x[0]) >= min_p]
        p = np.exp((x - x[0]) / temp)
        c = np.cumsum(p)
        at = min(int(np.searchsorted(c, r * c[-1], side="left")), x.size - 1)
        probs.append(float(p[at] / c[-1]))
    return None, torch.tensor(probs, dtype=torch.float64)


def exact(case, seed):
    """The definitions, one sequence at a time, in 64 bits."""
    s = prepare(case, seed)
    if case["op"] == "sample":
        return _exact_sample(s)
    new, lens = _lengths(case)
    hq, hkv, d, page = case["hq"], case["hkv"], case["d"], case["page"]
    outs, first = [], 0
    if case["op"] == "rope":
        kp, vp, r = s["k_pages"].double(), s["v_pages"].double(), case["d_rot"]
        j = torch.arange(r // 2, device="cuda")
        a, b = (2 * j, 2 * j + 1) if case["interleaved"] else (j, j + r // 2)
    for q_n, length, table in zip(new, lens, s["page_table"].long()):
        tok = slice(first, first + q_n)
        first += q_n
        pos = torch.arange(length - q_n, length, device="cuda")
        if case["op"] == "rope":
            x = s["qkv"][tok].double().view(q_n, hq + 2 * hkv, d).clone()
            if case["norm"]:
                for heads, w in ((slice(0, hq), s["q_norm_w"]), (slice(hq, hq + hkv), s["k_norm_w"])):
                    x[:, heads] *= w.double() / torch.sqrt((x[:, heads] ** 2).mean(-1, keepdim=True) + _EPS)
            z = torch.polar(torch.tensor(s["mscale"], dtype=torch.float64, device="cuda"),
                            2 * math.pi * torch.fmod(pos.double()[:, None] * s["freqs"], 1.0))[:, None]
            y = x[:, :hq + hkv]
            z = torch.complex(y[..., a], y[..., b]) * z
            y[..., a], y[..., b] = z.real, z.imag
            outs.append(y[:, :hq].clone())
            kp[table[pos // page], :, pos % page] = y[:, hq:]
            vp[table[pos // page], :, pos % page] = x[:, hq + hkv:]
            continue
        used = table[: -(-length // page)]
        k, v = (p[used].double().transpose(0, 1).reshape(hkv, -1, d)[:, :length] for p in (s["k_pages"], s["v_pages"]))
        key = torch.arange(length, device="cuda")
        back = pos[:, None] - key
        hidden = (back < 0) | (back >= (case["window"] or length + 1))
        o = torch.empty(q_n, hq, d, dtype=torch.float64, device="cuda")
        for h in range(hq):
            sc = s["q"][tok, h].double() @ k[h * hkv // hq].T / math.sqrt(d)
            o[:, h] = torch.softmax(sc.masked_fill(hidden, -math.inf), -1) @ v[h * hkv // hq]
        outs.append(o)
    return (torch.cat(outs), kp, vp) if case["op"] == "rope" else torch.cat(outs)
