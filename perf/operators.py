"""Cases and plain forms of the decoder operators: the norm and rotation of
queries and keys (with the cache append), attention over a paged cache, and
sampling.

``run`` computes a case with elementary torch operations, or, with ``own``
set, with the framework's kernels (``rten_hip``).  Sizes are generic decoder
sizes and this repository's BERT sizes (12 heads of 64, 30,522 tokens).
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

DEV = "cuda"
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _rotary(name, seqs, q, ctx, hq, hk, d, rot, cache, page, inter=False, norm=True, lens=1):
    """One norm + rotation + append over `seqs` sequences: new tokens per
    sequence in q = (lo, hi), cached tokens before them in ctx = (lo, hi)."""
    c = {"op": "rotary", "seqs": seqs, "q_lo": q[0], "q_hi": q[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1], "hq": hq,
         "hk": hk, "d": d, "rot": rot, "cache": cache, "page": page, "inter": inter, "norm": norm, "lens": lens}
    return dict(c, name=name) if name else c


def _attention(name, seqs, q, ctx, hq, hk, d, cache, page, window=0, sinks=0, lens=1):
    c = {"op": "attention", "seqs": seqs, "q_lo": q[0], "q_hi": q[1], "ctx_lo": ctx[0], "ctx_hi": ctx[1], "hq": hq,
         "hk": hk, "d": d, "cache": cache, "page": page, "window": window, "sinks": sinks, "lens": lens}
    return dict(c, name=name) if name else c


def _sample(name, rows, vocab, temperature, top_k, top_p, min_p, sharp):
    """sharp: the logits' standard deviation (4 and more: a sure model)."""
    c = {"op": "sample", "rows": rows, "vocab": vocab, "temperature": temperature, "top_k": top_k, "top_p": top_p,
         "min_p": min_p, "sharp": sharp}
    return dict(c, name=name) if name else c


def listed():
    return [
        # One sequence answering: the smallest step, all latency.
        _rotary("rotary 1 token", 1, (1, 1), (900, 900), 32, 8, 128, 128, "f16", 16),
        # A few ragged prompts of a model with 12 heads of 64, interleaved
        # pairs, half of each head rotated, float32 cache.
        _rotary("rotary ragged prompts", 7, (31, 701), (0, 300), 12, 12, 64, 32, "f32", 16, inter=True, lens=3),
        # A long prompt taken in one piece.
        _rotary("rotary 8192 tokens", 1, (8192, 8192), (0, 0), 32, 8, 128, 128, "bf16", 64),
        # One sequence answering on a float32 cache of odd length.
        _attention("attention 1 token", 1, (1, 1), (777, 777), 12, 12, 64, "f32", 16),
        # A serving batch: one new token for each of 64 ragged sequences.
        _attention("attention batch of 64", 64, (1, 1), (60, 6000), 32, 8, 128, "f16", 16, lens=5),
        # One long conversation: a token over 131,072 cached ones in float32.
        _attention("attention long", 1, (1, 1), (131071, 131071), 32, 8, 128, "f32", 64),
        # Long conversations of a model with a window of 4096 and 4 sinks.
        _attention("attention window", 32, (1, 1), (5000, 32000), 64, 8, 64, "bf16", 32, 4096, 4, lens=7),
        # A mixed step: answering sequences next to prompt chunks.
        _attention("attention mixed chunks", 9, (1, 600), (0, 6000), 32, 8, 128, "f16", 16, lens=11),
        # A long prompt attended in one piece on a float32 cache.
        _attention("attention 8192 tokens", 1, (8192, 8192), (0, 0), 32, 8, 128, "f32", 64),
        # One row of this repository's BERT vocabulary, all filters on.
        _sample("sample 1 row", 1, 30522, 0.8, 50, 0.95, 0.02, 3.0),
        # A serving batch with top-p over a large odd vocabulary.
        _sample("sample 64 rows top-p", 64, 100003, 0.7, 0, 0.9, 0.0, 2.5),
        # The largest: 256 rows, temperature only (no filter).
        _sample("sample 256 rows", 256, 131072, 1.0, 0, 1.0, 0.0, 2.0),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "attention", "attention", "sample"])
    cache, page = rng.choice(list(TYPES)), rng.choice([8, 16, 16, 24, 32, 64, 128])
    lens = rng.randrange(1, 1 << 20)
    hk = rng.choice([1, 2, 4, 8, 8, 12])
    hq = hk * rng.choice([1, 2, 3, 4, 7, 8])
    d = rng.choice([64, 64, 80, 96, 128, 128, 128, 192, 256])
    if op == "sample":
        vocab = _log_int(rng, 1000, 131072)
        rows = _log_int(rng, 1, max(1, min(256, (256 * 131072) // vocab)))
        top_k = rng.choice([0, 0, 1, _log_int(rng, 2, 200), _log_int(rng, 2, vocab)])
        return _sample(None, rows, vocab, rng.choice([0.0, 1.0, round(rng.uniform(0.3, 1.6), 2)]), top_k,
                       rng.choice([1.0, round(rng.uniform(0.3, 0.99), 3)]),
                       rng.choice([0.0, 0.0, round(rng.uniform(0.001, 0.2), 3)]), round(rng.uniform(0.5, 4.0), 2))
    if op == "rotary":
        tokens = _log_int(rng, 1, 8192)
        while tokens * (hq + 2 * hk) * d > 8192 * 48 * 128:
            tokens = max(1, tokens // 2)
        seqs = _log_int(rng, 1, min(64, tokens))
        hi = max(1, tokens // seqs)
        return _rotary(None, seqs, (max(1, hi // 8), hi), (0, _log_int(rng, 1, 4000)), hq, hk, d,
                       rng.choice([d, d, d // 16 * 8]), cache, page, rng.random() < 0.3, rng.random() < 0.8, lens)
    window = rng.choice([0, 0, 0, _log_int(rng, 16, 4096)])
    sinks = rng.choice([0, 4, rng.randrange(1, 100)]) if window else 0
    if rng.random() < 0.5:  # single tokens
        seqs = _log_int(rng, 1, 128)
        hi = _log_int(rng, 16, 131072)
        while seqs * hi * hk * d > 131072 * 8 * 128:
            hi = max(1, hi // 2)
        return _attention(None, seqs, (1, 1), (hi // 8, hi), hq, hk, d, cache, page, window, sinks, lens)
    seqs = _log_int(rng, 1, 16)
    q = _log_int(rng, 2, 4096)
    ctx = _log_int(rng, 1, 8192)
    while seqs * q * (q + ctx) * hq > 8192 * 8192 * 16 or seqs * (q + ctx) * hk * d > 131072 * 8 * 128:
        q, ctx = max(2, q // 2), max(1, ctx // 2)
    return _attention(None, seqs, (max(1, q // 5), q), (0, ctx), hq, hk, d, cache, page, window, sinks, lens)


def _lengths(case):
    """(new tokens, all cached tokens with them) of each sequence: plain
    lists that follow from the case alone."""
    r = random.Random(case["lens"])
    q = [_log_int(r, case["q_lo"], case["q_hi"]) for _ in range(case["seqs"])]
    ctx = [r.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["seqs"])]
    return q, [a + b for a, b in zip(q, ctx)]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    s = dict(case)
    if case["op"] == "sample":
        # Zipf-like: a few likely tokens over a long tail of unlikely ones.
        s["logits"] = normal(case["rows"], case["vocab"]) * case["sharp"]
        s["uniforms"] = torch.rand(case["rows"], generator=g, device=DEV)
        return s
    q_lens, kv_lens = _lengths(case)
    page, hq, hk, d = case["page"], case["hq"], case["hk"], case["d"]
    pages = [-(-n // page) for n in kv_lens]
    total, width = sum(pages), max(pages) + 1
    n_pages = total + 3
    order = torch.randperm(n_pages, generator=g, device=DEV).to(torch.int32)
    # Sequence i owns the next pages[i] of the shuffled pages; -1: no page.
    first = torch.tensor([sum(pages[:i]) for i in range(len(pages))], device=DEV)
    at = torch.arange(width, device=DEV)
    owned = at[None, :] < torch.tensor(pages, device=DEV)[:, None]
    s["page_table"] = torch.where(owned, order[(first[:, None] + at).clamp(max=n_pages - 1)], -1).to(torch.int32)
    s["kv_lens"] = torch.tensor(kv_lens, dtype=torch.int32, device=DEV)
    s["q_starts"] = torch.tensor([sum(q_lens[:i]) for i in range(len(q_lens) + 1)], dtype=torch.int32, device=DEV)
    s["tokens"], s["q_max"], s["kv_max"] = sum(q_lens), max(q_lens), max(kv_lens)
    s["single"] = s["q_max"] == 1  # one new token for every sequence: the step's own shape
    kind = TYPES[case["cache"]]
    shape = (n_pages, page, hk, d)
    if case["op"] == "rotary":
        # The fused projection's output: q, k and v side by side in a row.
        qkv = normal(s["tokens"], hq + 2 * hk, d)
        s["q"], s["k"], s["v"] = qkv[:, :hq], qkv[:, hq:hq + hk], qkv[:, hq + hk:]
        s["k_cache"], s["v_cache"] = torch.zeros(shape, dtype=kind, device=DEV), torch.zeros(shape, dtype=kind, device=DEV)
        s["q_scale"] = 1 + 0.2 * normal(d) if case["norm"] else None
        s["k_scale"] = 1 + 0.2 * normal(d) if case["norm"] else None
        half = case["rot"] // 2
        s["inv_freq"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64, device=DEV) / half)).float()
        return s
    # Queries and keys after their norms: unit variance with some channels
    # that are louder, as trained scales give.
    loud = 1 + 2 * (torch.rand(d, generator=g, device=DEV) < 0.05).float()
    s["q"] = normal(s["tokens"], hq, d) * loud
    s["k_cache"] = torch.empty(shape, dtype=kind, device=DEV)
    s["v_cache"] = torch.empty(shape, dtype=kind, device=DEV)
    s["k_cache"].copy_(normal(*shape).mul_(loud))
    s["v_cache"].copy_(normal(*shape).mul_(0.5))
    s["scale"] = 1 / math.sqrt(d)
    return s


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    return {"rotary": _rotary_plain, "attention": _attention_plain, "sample": _sample_plain}[state["op"]](state)


def _run_own(s):
    if _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    import rten_hip

    if s["op"] == "sample":
        tokens, logprobs = rten_hip.sample(s["logits"], s["uniforms"], temperature=s["temperature"], top_k=s["top_k"],
                                           top_p=s["top_p"], min_p=s["min_p"])
        return {"tokens": tokens, "logprobs": logprobs}
    starts = None if s["single"] else s["q_starts"]
    if s["op"] == "rotary":
        q = rten_hip.qk_norm_rotary_append(s["q"], s["k"], s["v"], s["inv_freq"], s["k_cache"], s["v_cache"],
                                           s["page_table"], s["kv_lens"], starts, q_scale=s["q_scale"],
                                           k_scale=s["k_scale"], epsilon=1e-6, interleaved=s["inter"])
        return {"q": q, "k_cache": s["k_cache"], "v_cache": s["v_cache"]}
    return {"out": rten_hip.paged_attention(s["q"], s["k_cache"], s["v_cache"], s["page_table"], s["kv_lens"], starts,
                                            scale=s["scale"], window=s["window"], sinks=s["sinks"])}


_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rten-fork_amd")


def _places(s):
    """Sequence, number within it and position in its cache of every token."""
    t = torch.arange(s["tokens"], device=DEV)
    starts = s["q_starts"].long()
    seq = torch.searchsorted(starts[1:], t, right=True)
    nth = t - starts[seq]
    pos = s["kv_lens"].long()[seq] - (starts[seq + 1] - starts[seq]) + nth
    return seq, nth, pos


def _rotary_plain(s):
    seq, _, pos = _places(s)
    half = s["rot"] // 2
    angle = pos.double()[:, None] * s["inv_freq"].double()
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def rows(x, scale):
        if scale is not None:
            x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + 1e-6) * scale
        r, rest = x[..., :2 * half], x[..., 2 * half:]
        if s["inter"]:
            a, b = r[..., 0::2], r[..., 1::2]
            r = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = r[..., :half], r[..., half:]
            r = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((r, rest), -1)

    page = s["page_table"].long()[seq, pos // s["page"]]
    s["k_cache"][page, pos % s["page"]] = rows(s["k"], s["k_scale"]).to(s["k_cache"].dtype)
    s["v_cache"][page, pos % s["page"]] = s["v"].to(s["v_cache"].dtype)
    return {"q": rows(s["q"], s["q_scale"]), "k_cache": s["k_cache"], "v_cache": s["v_cache"]}


def _attention_plain(s):
    seq, nth, _ = _places(s)
    n, q_max, hk, d = s["seqs"], s["q_max"], s["hk"], s["d"]
    group = s["hq"] // hk
    starts, kv = s["q_starts"].long(), s["kv_lens"].long()
    # Queries padded to [sequence, kv head, token x group, d].
    at = (starts[:-1, None] + torch.arange(q_max, device=DEV)).clamp(max=s["tokens"] - 1)
    q = s["q"][at].view(n, q_max, hk, group, d).permute(0, 2, 1, 3, 4).reshape(n, hk, q_max * group, d)
    pages = s["page_table"][:, :-(-s["kv_max"] // s["page"])].long().clamp(min=0)
    k = s["k_cache"][pages].flatten(1, 2).float().permute(0, 2, 3, 1)
    v = s["v_cache"][pages].flatten(1, 2).float().permute(0, 2, 1, 3)
    j = torch.arange(k.shape[-1], device=DEV)
    pos = (kv - starts[1:] + starts[:-1])[:, None] + torch.arange(q_max, device=DEV)
    seen = j <= pos[..., None]
    if s["window"]:
        seen &= (j > pos[..., None] - s["window"]) | (j < s["sinks"])
    seen = seen & (j < kv[:, None, None])
    seen = seen[:, None, :, None].expand(n, 1, q_max, group, j.numel()).reshape(n, 1, q_max * group, -1)
    x = torch.matmul(q * s["scale"], k).masked_fill_(~seen, -math.inf)
    x = torch.exp_(x.sub_(x.amax(-1, keepdim=True).clamp(min=-3e38)))
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x, v) / torch.where(total > 0, total, 1)
    o = o.view(n, hk, q_max, group, d).permute(0, 2, 1, 3, 4)[seq, nth]
    return {"out": o.reshape(s["tokens"], s["hq"], d)}


def _sample_plain(s):
    logits, rows, vocab = s["logits"], s["rows"], s["vocab"]
    best = logits.argmax(-1)
    if s["temperature"] <= 0:
        return {"tokens": best.int(), "logprobs": torch.zeros(rows, device=DEV)}
    x = logits.double()
    mass = torch.exp((x - x.amax(-1, keepdim=True)) / float(np.float32(s["temperature"])))
    if s["top_k"] or s["top_p"] < 1 or s["min_p"] > 0:
        order = torch.sort(logits, dim=-1, descending=True, stable=True).indices
        ranked = mass.gather(-1, order)
        rank = torch.arange(vocab, device=DEV)
        if s["top_k"]:
            ranked = torch.where(rank < s["top_k"], ranked, 0)
        before = ranked.cumsum(-1) - ranked
        if s["top_p"] < 1:
            p = float(np.float32(s["top_p"]))
            ranked = torch.where((before < p * ranked.sum(-1, keepdim=True)) | (rank == 0), ranked, 0)
        if s["min_p"] > 0:
            ranked = torch.where(ranked >= float(np.float32(s["min_p"])), ranked, 0)
        mass = torch.zeros_like(mass).scatter_(-1, order, ranked)
    upto = mass.cumsum(-1)
    total = upto[:, -1:]
    token = torch.searchsorted(upto, s["uniforms"].double()[:, None] * total, right=True).clamp(max=vocab - 1)
    return {"tokens": token[:, 0].int(), "logprobs": torch.log(mass.gather(-1, token) / total)[:, 0].float()}


# ---------------------------------------------------------------------------
# What a pass cannot do without
# ---------------------------------------------------------------------------

def _seen_pairs(case):
    """(visible query-key pairs, keys that some query of their sequence sees)
    summed over the sequences."""
    pairs = keys = 0
    w, sinks = case["window"], case["sinks"]
    for q, kv in zip(*_lengths(case)):
        first = kv - q
        if not w:
            pairs += q * (2 * first + q + 1) // 2
            keys += kv
        else:
            pos = np.arange(first, kv)
            low = np.maximum(0, pos - w + 1)
            pairs += int((pos + 1 - low + np.minimum(low, sinks)).sum())
            keys += kv - int(low[0]) + min(int(low[0]), sinks)
    return pairs, keys


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": 4 * n + 12 * case["rows"], "flops": 4 * n}
    size, d = (4 if case["cache"] == "f32" else 2), case["d"]
    tokens = sum(_lengths(case)[0])
    if case["op"] == "rotary":
        return {"bytes": tokens * d * (8 * case["hq"] + case["hk"] * (8 + 2 * size)),
                "flops": tokens * (case["hq"] + case["hk"]) * (3 * case["rot"] + (4 * d if case["norm"] else 0))}
    pairs, keys = _seen_pairs(case)
    return {"bytes": 2 * keys * case["hk"] * d * size + 8 * tokens * case["hq"] * d, "flops": 4 * pairs * case["hq"] * d}


# ---------------------------------------------------------------------------
# The definitions in 64 bits
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _rotary_exact, "attention": _attention_exact, "sample": _sample_exact}[case["op"]](s)


def _rotary_exact(s):
    q_lens, kv_lens = _lengths(s)
    pos = torch.tensor([kv - q + i for q, kv in zip(q_lens, kv_lens) for i in range(q)], dtype=torch.float64, device=DEV)
    seq = torch.tensor([n for n, q in enumerate(q_lens) for _ in range(q)], device=DEV)
    turn = torch.polar(torch.ones(1, dtype=torch.float64, device=DEV), pos[:, None] * s["inv_freq"].double())[:, None]
    half = s["rot"] // 2

    def rows(x, scale):
        x = x.double()
        if scale is not None:
            x = x / torch.sqrt(x.square().mean(-1, keepdim=True) + 1e-6) * scale.double()
        lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if s["inter"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(x[..., lo].contiguous(), x[..., hi].contiguous()) * turn
        x = x.clone()
        x[..., lo], x[..., hi] = z.real, z.imag
        return x

    at = s["page_table"].long()[seq, pos.long() // s["page"]] * s["page"] + pos.long() % s["page"]
    caches = []
    for cache, x in ((s["k_cache"], rows(s["k"], s["k_scale"])), (s["v_cache"], s["v"].double())):
        flat = cache.double().flatten(0, 1)
        flat[at] = x
        caches.append(flat.view(cache.shape))
    return {"q": rows(s["q"], s["q_scale"]), "k_cache": caches[0], "v_cache": caches[1]}


def _attention_exact(s):
    out, first = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), 0
    group = s["hq"] // s["hk"]
    for n, (q_len, kv_len) in enumerate(zip(*_lengths(s))):
        pages = s["page_table"][n, :-(-kv_len // s["page"])].long()
        pos = torch.arange(kv_len - q_len, kv_len, device=DEV)[:, None]
        j = torch.arange(kv_len, device=DEV)
        hidden = j > pos
        if s["window"]:
            hidden = hidden | ((j <= pos - s["window"]) & (j >= s["sinks"]))
        for h in range(s["hk"]):
            k = s["k_cache"][pages, :, h].double().flatten(0, 1)[:kv_len]
            v = s["v_cache"][pages, :, h].double().flatten(0, 1)[:kv_len]
            for e in range(h * group, (h + 1) * group):
                x = s["q"][first:first + q_len, e].double() @ k.t().contiguous() * s["scale"]
                out[first:first + q_len, e] = torch.softmax(x.masked_fill_(hidden, -math.inf), -1) @ v
        first += q_len
    return {"out": out}


def _sample_exact(s):
    logits, uniforms = s["logits"].cpu().numpy().astype(np.float64), s["uniforms"].cpu().numpy().astype(np.float64)
    tokens, logprobs = [], []
    for x, u in zip(logits, uniforms):
        if s["temperature"] <= 0:
            tokens.append(int(np.flatnonzero(x == x.max())[0]))
            logprobs.append(0.0)
            continue
        p = np.exp((x - x.max()) / float(np.float32(s["temperature"])))
        p /= p.sum()
        kept = np.ones(p.size, bool)
        if s["top_k"] or s["top_p"] < 1 or s["min_p"] > 0:
            order = np.lexsort((np.arange(p.size), -x))
            if s["top_k"]:
                order = order[:s["top_k"]]
            if s["top_p"] < 1:
                mass = np.concatenate(([0.0], np.cumsum(p[order])))
                order = order[:max(1, int(np.sum(mass[:-1] < float(np.float32(s["top_p"])) * mass[-1])))]
            if s["min_p"] > 0:
                order = order[p[order] >= float(np.float32(s["min_p"])) * p.max()]
            kept[:] = False
            kept[order] = True
        at = np.flatnonzero(kept)
        mass = np.cumsum(p[at])
        n = min(int(np.searchsorted(mass, u * mass[-1], side="right")), at.size - 1)
        tokens.append(int(at[n]))
        logprobs.append(math.log(p[at[n]] / mass[-1]))
    return {"tokens": torch.tensor(tokens, dtype=torch.int32), "logprobs": torch.tensor(logprobs, dtype=torch.float64)}
