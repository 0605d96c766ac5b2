"""GPU tests of the decoder operators (qk_norm_rotary, its append to a paged
cache, paged_attention, sample) against plain 64-bit forms on the CPU.

Tolerances count roundings.  u = 2^-24 is half a step of float32 relative to
the value; a 16-bit cache adds half a step of its type where a value is stored.
"""
import math

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
TYPES = ["float32", "float16", "bfloat16"]


@pytest.fixture(scope="module")
def rh():
    import torch

    if not torch.cuda.is_available():
        pytest.skip("no GPU")
    import rten_hip

    rten_hip.default_context()
    return rten_hip


def dtype(name):
    import torch

    return getattr(torch, name)


class Paged:
    """Sequences with shuffled pages: page tables on the host and the device."""

    def __init__(self, q_lens, kv_lens, page, seed=0, extra=2, width=0):
        import torch

        self.q_lens, self.kv_lens, self.page = list(q_lens), list(kv_lens), page
        pages = [-(-n // page) for n in kv_lens]
        self.n_pages = sum(pages) + extra
        order = np.random.default_rng(seed).permutation(self.n_pages)
        width = max(width, max(pages, default=0))
        self.table = np.full((len(pages), width), -1, np.int32)
        at = 0
        for i, n in enumerate(pages):
            self.table[i, :n] = order[at:at + n]
            at += n
        self.starts = np.concatenate(([0], np.cumsum(q_lens))).astype(np.int32)
        self.tokens = int(self.starts[-1])
        self.d_table = torch.from_numpy(self.table).cuda()
        self.d_kv = torch.tensor(self.kv_lens, dtype=torch.int32).cuda()
        self.d_starts = torch.from_numpy(self.starts).cuda()

    def place(self, s, j):
        """(page, slot) of token j of sequence s; page -1: none."""
        p = j // self.page
        return (int(self.table[s, p]) if p < self.table.shape[1] else -1), j % self.page


# ---------------------------------------------------------------------------
# Norm, rotation, append
# ---------------------------------------------------------------------------

def rotary_ref(x, pos, inv_freq, scale, eps, interleaved):
    """x [tokens, heads, dim] float64."""
    x = x.astype(np.float64)
    if scale is not None:
        x = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps) * scale.astype(np.float64)
    half = len(inv_freq)
    a = pos.astype(np.float64)[:, None] * inv_freq.astype(np.float64)
    c, s = np.cos(a)[:, None], np.sin(a)[:, None]
    y = x.copy()
    lo, hi = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y[..., lo], y[..., hi] = x[..., lo] * c - x[..., hi] * s, x[..., hi] * c + x[..., lo] * s
    return y


def rotary_close(got, want, what):
    # The norm: at most 8 + 5 roundings in the sum of squares (half of that in
    # its root), 2 for the root and the quotient, 2 products: under 11 u.  The
    # turn: cos and sin within 3 u, two roundings each of two terms, each term
    # at most the pair's length: 8 u of that length, which the row's largest
    # pair bounds by sqrt(2) of the largest value.
    tol = 24 * U * np.abs(want).max(-1, keepdims=True) + 1e-40
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:3], np.abs(got - want).max())


@pytest.mark.parametrize("tokens,hq,hk,dim,rot,inter,norm", [
    (1, 1, 1, 8, 8, False, True), (3, 5, 1, 64, 64, False, True), (2, 12, 12, 64, 32, True, True),
    (5, 7, 7, 80, 40, False, True), (4, 4, 2, 96, 96, True, False), (9, 32, 8, 128, 128, False, True),
    (600, 8, 2, 128, 64, False, True), (2, 3, 3, 192, 0, False, True), (3, 2, 1, 256, 256, True, True),
    (1, 3, 2, 24, 16, False, False), (0, 3, 2, 64, 64, False, True),
])
def test_rotary(rh, tokens, hq, hk, dim, rot, inter, norm):
    import torch

    g = torch.Generator().manual_seed(tokens * 1000 + dim)
    qkv = torch.randn(tokens, hq + hk, dim, generator=g)
    pos = torch.randint(0, 1_000_000, (tokens,), generator=g, dtype=torch.int32)
    half = rot // 2
    freq = (10000.0 ** (-torch.arange(half).double() / max(half, 1))).float()
    w = [1 + 0.3 * torch.randn(dim, generator=g) for _ in range(2)] if norm else [None, None]
    d = qkv.cuda()
    q, k = d[:, :hq], d[:, hq:]
    qo, ko = rh.qk_norm_rotary(q, k, pos.cuda(), freq.cuda() if rot else None, *[x.cuda() if norm else None for x in w],
                               epsilon=1e-5, interleaved=inter)
    torch.cuda.synchronize()
    assert torch.equal(d.cpu(), qkv)
    for got, x, s in ((qo, qkv[:, :hq], w[0]), (ko, qkv[:, hq:], w[1])):
        assert got.shape == x.shape
        if tokens:
            rotary_close(got.cpu().numpy(), rotary_ref(x.numpy(), pos.numpy(), freq.numpy(),
                                                       s.numpy() if norm else None, 1e-5, inter), "rows")
    # In place, on the parts of the same buffer: the same bits.
    q2, k2 = rh.qk_norm_rotary(q, k, pos.cuda(), freq.cuda() if rot else None, *[x.cuda() if norm else None for x in w],
                               epsilon=1e-5, interleaved=inter, q_out=q, k_out=k)
    assert q2.data_ptr() == q.data_ptr() and torch.equal(q2, qo) and torch.equal(k2, ko)


def test_rotary_far_positions_and_edge_rows(rh):
    """Positions up to 2^31 - 1 and below 0; rows of zeros; a NaN stays in its
    row."""
    import torch

    pos = torch.tensor([0, 1, 2 ** 20 + 7, 2 ** 31 - 1, -5, 3, 4], dtype=torch.int32)
    x = torch.randn(7, 2, 64, generator=torch.Generator().manual_seed(3))
    x[5, 0] = 0
    x[6, 1, 9] = math.nan
    freq = (10000.0 ** (-torch.arange(32).double() / 32)).float()
    w = torch.ones(64)
    q, k = rh.qk_norm_rotary(x.cuda(), x.cuda(), pos.cuda(), freq.cuda(), w.cuda(), None)
    want = rotary_ref(x.numpy(), pos.numpy(), freq.numpy(), w.numpy(), 1e-6, False)
    got = q.cpu().numpy()
    # The angle itself, up to 2^31, is rounded to 64 bits: 2^-22 at the most.
    far = np.abs(got[3] - want[3]).max() <= (2.0 ** -22 + 24 * U) * np.abs(want[3]).max()
    assert far
    keep = [0, 1, 2, 4, 5]
    rotary_close(got[keep], want[keep], "q")
    assert not got[5, 0].any() and np.isnan(got[6, 1]).all() and np.isfinite(got[6, 0]).all()
    assert np.isfinite(k.cpu().numpy()[:6]).all()


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("page,heads_first", [(1, False), (5, True), (16, False), (64, True)])
@pytest.mark.parametrize("q_lens,kv_lens", [
    ([1, 1, 1], [1, 40, 129]), ([0, 7, 0, 0, 70, 1], [5, 7, 0, 9, 100, 1]), ([130] * 3, [130, 200, 131]),
])
def test_append(rh, cache_type, page, heads_first, q_lens, kv_lens):
    import torch

    hq, hk, dim = 6, 2, 64
    s = Paged(q_lens, kv_lens, page, seed=page, width=3)
    g = torch.Generator().manual_seed(7)
    pad = 5
    qkv = torch.randn(s.tokens + pad, hq + 2 * hk, dim, generator=g)
    freq = (1000.0 ** (-torch.arange(32).double() / 32)).float()
    w = 1 + 0.3 * torch.randn(2, dim, generator=g)
    shape = (s.n_pages, hk, page, dim) if heads_first else (s.n_pages, page, hk, dim)
    caches = [torch.full(shape, 7.0, dtype=dtype(cache_type)) for _ in range(2)]
    kc, vc = (c.cuda().transpose(1, 2) if heads_first else c.cuda() for c in caches)
    d = qkv.cuda()
    out = torch.full((s.tokens + pad, hq, dim), 9.0).cuda()
    single = all(n == 1 for n in q_lens)
    if single:
        d, out, pad = d[:s.tokens], out[:s.tokens], 0
    got = rh.qk_norm_rotary_append(d[:, :hq], d[:, hq:hq + hk], d[:, hq + hk:], freq.cuda(), kc, vc, s.d_table, s.d_kv,
                                   None if single else s.d_starts, q_scale=w[0].cuda(), k_scale=w[1].cuda(), out=out)
    assert got is out
    pos = np.concatenate([np.arange(kv - q, kv) for q, kv in zip(q_lens, kv_lens)])
    seq = np.repeat(np.arange(len(q_lens)), q_lens)
    x = qkv.numpy()[:s.tokens]
    rotary_close(out.cpu().numpy()[:s.tokens],
                 rotary_ref(x[:, :hq], pos, freq.numpy(), w[0].numpy(), 1e-6, False), "q")
    assert (out.cpu().numpy()[s.tokens:] == 9).all()
    want_k = rotary_ref(x[:, hq:hq + hk], pos, freq.numpy(), w[1].numpy(), 1e-6, False)
    k, v = kc.cpu().float().numpy(), vc.cpu().float().numpy()
    step = 0 if cache_type == "float32" else torch.finfo(dtype(cache_type)).eps / 2
    written = np.zeros(k.shape[:2], bool)
    for t in range(s.tokens):
        p, o = s.place(seq[t], int(pos[t]))
        written[p, o] = True
        top = np.abs(want_k[t]).max(-1, keepdims=True)
        # (float16 has steps of 2^-24 below 2^-14.)
        assert (np.abs(k[p, o] - want_k[t]) <= 24 * U * top + step * (1 + 24 * U) * np.abs(want_k[t]) + 2.0 ** -25).all()
        assert np.array_equal(v[p, o], qkv[t, hq + hk:].to(dtype(cache_type)).float().numpy())
    assert (k[~written] == 7).all() and (v[~written] == 7).all()


def test_append_positions_and_missing_pages(rh):
    """Given positions turn the rows without moving them; a token whose page
    is -1, out of the cache or past the table is written nowhere."""
    import torch

    s = Paged([3, 2, 2], [3, 18, 40], 16)
    s.d_table[0, 0], s.d_table[1, 1], s.d_table[2, 2] = -1, s.n_pages, 2 ** 30
    x = torch.randn(7, 3, 64, generator=torch.Generator().manual_seed(1))
    freq = torch.ones(4)
    pos = torch.tensor([5, -1, 2, 9, 9, 1, 0], dtype=torch.int32)
    kc = torch.full((s.n_pages, 16, 1, 64), 7.0).cuda()
    vc = kc.clone()
    d = x.cuda()
    out = rh.qk_norm_rotary_append(d[:, :1], d[:, 1:2], d[:, 2:], freq.cuda(), kc, vc, s.d_table[:, :2], s.d_kv,
                                   s.d_starts, positions=pos.cuda())
    rotary_close(out.cpu().numpy(), rotary_ref(x[:, :1].numpy(), pos.numpy(), freq.numpy(), None, 0, False), "q")
    # Sequence 2's tokens 38, 39 lie past a table of two pages.
    assert (kc == 7).all() and (vc == 7).all()
    s = Paged([2], [2], 16)
    out = rh.qk_norm_rotary_append(d[:2, :1], d[:2, 1:2], d[:2, 2:], freq.cuda(), kc, vc, s.d_table, s.d_kv, s.d_starts,
                                   positions=pos[:2].cuda())
    want = rotary_ref(x[:2, 1:2].numpy(), pos[:2].numpy(), freq.numpy(), None, 0, False)
    rotary_close(kc[int(s.table[0, 0]), :2].cpu().numpy(), want, "k")


# ---------------------------------------------------------------------------
# Attention
# ---------------------------------------------------------------------------

def attention_ref(q, k, v, s, scale, window, sinks, q_lens=None):
    """(out, tolerance) [tokens, hq, dim] in float64; q, k, v numpy float32 (of
    the cache's values)."""
    tokens, hq, dim = q.shape
    group = hq // k.shape[2]
    out, tol = np.zeros((tokens, hq, dim)), np.zeros((tokens, hq, 1))
    for i, (ql, kv) in enumerate(zip(q_lens or s.q_lens, s.kv_lens)):
        places = [s.place(i, j) for j in range(kv)]
        here = np.array([p >= 0 for p, _ in places], bool)
        pj, oj = np.array([max(p, 0) for p, _ in places], int), np.array([o for _, o in places], int)
        j = np.arange(kv)
        for t in range(ql):
            pos = kv - ql + t
            seen = here & (j <= pos)
            if window:
                seen &= (j > pos - window) | (j < sinks)
            at = np.flatnonzero(seen)
            if not len(at):
                continue
            for h in range(hq):
                kk, vv = k[pj[at], oj[at], h // group].astype(np.float64), v[pj[at], oj[at], h // group].astype(np.float64)
                x = q[s.starts[i] + t, h].astype(np.float64)
                a = kk @ x * scale
                e = np.exp(a - a.max())
                out[s.starts[i] + t, h] = (e / e.sum()) @ vv
                # A score: q's product with the scale is rounded, each of its
                # dim products is off by up to 3 2^-23 (two terms of 11 bits
                # for either factor, their smallest product left out) or a
                # rounding, and their sum by dim / 8 more (a matrix
                # instruction adds 4 or more products at once), all relative
                # to sum |q k|; the exponent is rounded to u of the score, its
                # power to 2 u.  A relative error d of the weights moves the
                # result by at most 2 d max |v|.
                d = (6 + 2 + dim / 8) * U * (np.abs(kk) @ np.abs(x)).max() * scale + 4 * U * np.abs(a).max() + 8 * U
                # The sums over the keys: n / 16 steps in a row at the most,
                # the split of p and v 6 u more, joins and quotients 16 u.
                tol[s.starts[i] + t, h] = (2 * d + (len(at) / 16 + 24) * U) * np.abs(vv).max()
    return out, tol


def run_attention(rh, s, hq, hk, dim, cache_type, window=0, sinks=0, scale=None, seed=0, heads_first=False, single=False,
                  tweak=None, loud=1.0):
    import torch

    g = torch.Generator().manual_seed(seed)
    q = torch.randn(s.tokens, hq, dim, generator=g) * loud
    k = torch.randn(s.n_pages, s.page, hk, dim, generator=g).to(dtype(cache_type))
    v = (torch.randn(s.n_pages, s.page, hk, dim, generator=g) + 0.3).to(dtype(cache_type))
    if tweak:
        tweak(q, k, v)
    kd, vd = k.cuda(), v.cuda()
    if heads_first:
        kd, vd = (x.transpose(1, 2).contiguous().transpose(1, 2) for x in (kd, vd))
    out = rh.paged_attention(q.cuda(), kd, vd, s.d_table, s.d_kv, None if single else s.d_starts, scale=scale,
                             window=window, sinks=sinks)
    scale = 1 / math.sqrt(dim) if scale is None else scale
    return out.cpu().numpy(), q.numpy(), k.float().numpy(), v.float().numpy(), scale


def attention_close(got, want, tol, what=""):
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, np.argwhere(bad)[:4], np.nanmax(np.abs(got - want)), tol.max())


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hq,hk,dim", [(1, 1, 64), (4, 4, 8), (8, 2, 128), (16, 1, 128), (3, 1, 80), (6, 2, 256), (7, 1, 96)])
@pytest.mark.parametrize("kv_lens,page", [([1, 0, 63, 64, 65], 16), ([130, 1, 700], 7), ([2, 257], 64), ([5], 1)])
def test_attention_single_tokens(rh, cache_type, hq, hk, dim, kv_lens, page):
    s = Paged([1] * len(kv_lens), kv_lens, page, seed=page)
    got, q, k, v, scale = run_attention(rh, s, hq, hk, dim, cache_type, single=True, heads_first=page == 7)
    want, tol = attention_ref(q, k, v, s, scale, 0, 0)
    attention_close(got, want, tol)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hq,hk,dim", [(2, 2, 64), (8, 2, 128), (5, 1, 96), (2, 1, 256), (20, 1, 40)])
@pytest.mark.parametrize("q_lens,kv_lens,page", [
    ([70], [70], 16), ([0, 33, 1, 0, 5], [7, 90, 200, 0, 5], 5), ([129, 2], [300, 64], 64),
])
def test_attention_chunks(rh, cache_type, hq, hk, dim, q_lens, kv_lens, page):
    s = Paged(q_lens, kv_lens, page, seed=page)
    got, q, k, v, scale = run_attention(rh, s, hq, hk, dim, cache_type, heads_first=page == 5)
    want, tol = attention_ref(q, k, v, s, scale, 0, 0)
    attention_close(got, want, tol)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("dim", [16, 24, 56, 72, 104, 136, 152, 200, 248])
def test_attention_odd_head_dims(rh, cache_type, dim):
    for q_lens, kv_lens in (([1, 1], [70, 9]), ([30, 1], [100, 9])):
        s = Paged(q_lens, kv_lens, 16)
        got, q, k, v, scale = run_attention(rh, s, 4, 2, dim, cache_type)
        want, tol = attention_ref(q, k, v, s, scale, 0, 0)
        attention_close(got, want, tol)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 3), (17, 0), (64, 4), (100, 70), (1000, 4), (2 ** 31 - 1, 2 ** 31 - 1)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1, 1], [500, 64, 3]), ([40, 3], [333, 70])])
def test_attention_window(rh, cache_type, window, sinks, q_lens, kv_lens):
    s = Paged(q_lens, kv_lens, 16)
    got, q, k, v, scale = run_attention(rh, s, 8, 2, 64, cache_type, window, sinks)
    want, tol = attention_ref(q, k, v, s, scale, window, sinks)
    attention_close(got, want, tol)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("q_len", [1, 60])
def test_attention_long_splits(rh, cache_type, q_len):
    """One long sequence next to short ones: its keys are cut into stretches."""
    s = Paged([q_len, 1, 2], [5000, 3, 130], 16)
    got, q, k, v, scale = run_attention(rh, s, 4, 1, 128, cache_type, loud=3.0)
    want, tol = attention_ref(q, k, v, s, scale, 0, 0)
    attention_close(got, want, tol)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [100, 300]), ([1, 50], [100, 300])])
def test_attention_ignores_what_no_query_sees(rh, cache_type, q_lens, kv_lens):
    """NaN and infinity in free pages, behind the last token of a page, before
    the window, and under table entries that are no page."""
    import torch

    s = Paged(q_lens, kv_lens, 16)
    window, sinks = 64, 2
    s.d_table[1, 16] = -1  # tokens 256 .. 271 of sequence 1
    s.table[1, 16] = -1
    seen = np.zeros((s.n_pages, 16), bool)
    for i, (ql, kv) in enumerate(zip(q_lens, kv_lens)):
        for j in range(kv):
            p, o = s.place(i, j)
            if p >= 0 and (j > kv - ql - window or j < sinks):
                seen[p, o] = True

    def tweak(q, k, v):
        hidden = torch.from_numpy(~seen)
        k[hidden] = math.nan
        v[hidden] = math.inf
        v[torch.from_numpy(~seen) & (torch.arange(16) % 2 == 0)] = math.nan

    got, q, k, v, scale = run_attention(rh, s, 8, 2, 64, cache_type, window, sinks, tweak=tweak)
    with np.errstate(invalid="ignore"):
        want, tol = attention_ref(q, k, v, s, scale, window, sinks)
    assert np.isfinite(want).all()
    attention_close(got, want, tol)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hq", [2, 8])
def test_attention_later_tokens_do_not_reach_earlier_rows(rh, cache_type, hq):
    """A NaN or infinity in a key or value of the chunk reaches the rows that
    see it and no other."""
    import torch

    for q_len, kv in ((5, 50), (40, 90)):
        s = Paged([q_len], [kv], 16)
        at = kv - 3
        p, o = s.place(0, at)
        for bad_k, bad_v in ((0.0, math.inf), (math.nan, 0.5), (math.inf, -math.inf), (0.0, math.nan)):
            def tweak(q, k, v):
                k[p, o, 0, 5] = bad_k
                v[p, o, 0, 7] = bad_v

            got, q, k, v, scale = run_attention(rh, s, hq, 1, 64, cache_type, tweak=tweak)
            n = q_len - 3  # rows before the token
            s2 = Paged([n], [at], 16)
            s2.table, s2.n_pages = s.table, s.n_pages
            want, tol = attention_ref(q[:n], k, v, s2, scale, 0, 0)
            attention_close(got[:n], want, tol, (q_len, bad_k, bad_v))
            if not math.isfinite(bad_v):
                assert not np.isfinite(got[n:]).all()


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [90, 200]), ([30, 1], [90, 200])])
@pytest.mark.parametrize("qs,ks,vs", [(1e-3, 1e3, 1e-4), (50.0, 1.0, 1.0), (0.0, 1.0, 1.0), (1e-20, 1e-3, 1e-6), (1.0, 0.0, 0.0)])
def test_attention_ranges(rh, cache_type, q_lens, kv_lens, qs, ks, vs):
    """Loud, faint and zero operands, uneven from token to token."""
    import torch

    s = Paged(q_lens, kv_lens, 16)

    def tweak(q, k, v):
        uneven = torch.exp2(torch.randint(-6, 7, k.shape[:3], generator=torch.Generator().manual_seed(2)).float())[..., None]
        q *= qs
        k.copy_(k.float() * ks)
        v.copy_(v.float() * vs * uneven)

    got, q, k, v, scale = run_attention(rh, s, 4, 2, 64, cache_type, tweak=tweak)
    want, tol = attention_ref(q, k, v, s, scale, 0, 0)
    attention_close(got, want, tol)


@pytest.mark.parametrize("q_lens,kv_lens", [([1, 1], [1000, 90]), ([200, 1], [1000, 90])])
def test_attention_float32_huge_and_tiny(rh, q_lens, kv_lens):
    """A float32 cache far outside the range of 16 bits."""
    s = Paged(q_lens, kv_lens, 16)

    def tweak(q, k, v):
        q *= 1e-25
        k *= 1e25
        v *= 1e30
        v[::2] *= 2.0 ** -20

    got, q, k, v, scale = run_attention(rh, s, 2, 2, 64, "float32", tweak=tweak)
    want, tol = attention_ref(q, k, v, s, scale, 0, 0)
    attention_close(got, want, tol)


def test_attention_empty_rows_and_padding(rh):
    """Sequences without cached tokens or whose pages are all missing give
    zeros; padding rows stay; more new than cached tokens: the early ones see
    nothing."""
    import torch

    s = Paged([3, 2, 4], [0, 40, 2], 16)
    s.d_table[1] = -1
    s.table[1] = -1
    q = torch.randn(14, 4, 64)
    kv = torch.randn(s.n_pages, 16, 2, 64)
    out = torch.full((14, 4, 64), 5.0).cuda()
    got = rh.paged_attention(q.cuda(), kv.cuda(), kv.cuda(), s.d_table, s.d_kv, s.d_starts, out=out).cpu().numpy()
    assert (got[:5] == 0).all() and (got[5:7] == 0).all() and (got[9:] == 5).all()
    want, tol = attention_ref(q[:9].numpy(), kv.numpy(), kv.numpy(), s, 1 / 8, 0, 0)
    attention_close(got[:9], want, tol)
    # No sequences, no tokens, no pages.
    none = torch.empty(0, dtype=torch.int32).cuda()
    rh.paged_attention(q.cuda(), kv.cuda(), kv.cuda(), s.d_table[:0], none, torch.zeros(1, dtype=torch.int32).cuda(), out=out)
    assert (out.cpu().numpy() == got).all()
    assert rh.paged_attention(q[:0].cuda(), kv.cuda(), kv.cuda(), s.d_table[:0], none).shape == (0, 4, 64)
    empty = kv[:0].cuda()
    assert (rh.paged_attention(q[:3].cuda(), empty, empty, s.d_table[:, :0], s.d_kv).cpu() == 0).all()


def test_attention_strides_in_place_and_wild_metadata(rh):
    """q as part of a wider buffer, the result in its place; q_starts and
    tables that make no sense stay inside the buffers."""
    import torch

    s = Paged([20, 1, 9], [60, 33, 9], 16)
    g = torch.Generator().manual_seed(5)
    wide = torch.randn(s.tokens, 3, 8, 64, generator=g)
    kv = torch.randn(2, s.n_pages, 16, 2, 64, generator=g)
    d, c = wide.cuda(), kv.cuda()
    q = d[:, 1]
    got = rh.paged_attention(q, c[0], c[1], s.d_table, s.d_kv, s.d_starts, out=q)
    assert got.data_ptr() == q.data_ptr()
    want, tol = attention_ref(wide[:, 1].numpy(), kv[0].numpy(), kv[1].numpy(), s, 1 / 8, 0, 0)
    attention_close(got.cpu().numpy(), want, tol)
    assert torch.equal(d[:, 0].cpu(), wide[:, 0]) and torch.equal(d[:, 2].cpu(), wide[:, 2])
    for starts, lens in (([5, -3, 99, 7], [60, 33, 9]), ([0, 20, 21, 30], [2 ** 31 - 1, -4, 10 ** 6])):
        rh.paged_attention(q, c[0], c[1], s.d_table * 1000 - 7, torch.tensor(lens, dtype=torch.int32).cuda(),
                           torch.tensor(starts, dtype=torch.int32).cuda())
        rh.qk_norm_rotary_append(q, q[:, :2], q[:, 2:4], None, c[0], c[1], s.d_table * 1000 - 7,
                                 torch.tensor(lens, dtype=torch.int32).cuda(),
                                 torch.tensor(starts, dtype=torch.int32).cuda())
    torch.cuda.synchronize()


def test_attention_many_sequences(rh):
    """More sequences than a workgroup has threads."""
    lens = [(7 * i) % 90 for i in range(700)]
    q_lens = [1 if i % 5 else (i // 5) % 4 for i in range(700)]
    s = Paged(q_lens, [max(a, b) for a, b in zip(lens, q_lens)], 16)
    got, q, k, v, scale = run_attention(rh, s, 2, 1, 64, "float16")
    want, tol = attention_ref(q, k, v, s, scale, 0, 0)
    attention_close(got, want, tol)


# ---------------------------------------------------------------------------
# Sampling
# ---------------------------------------------------------------------------

def sample_ref(x, u, t, k, p, mp):
    """(token, log of its share, whether u is next to a border) of one row."""
    x = x.astype(np.float64)
    x[np.isnan(x)] = -np.inf
    if not len(x) or x.max() == -np.inf:
        return -1, -np.inf, False
    if not t > 0:
        return int(np.argmax(x)), 0.0, False
    if x.max() == np.inf:
        m = (x == np.inf).astype(np.float64)
    else:
        m = np.exp((x - x.max()) / t)
        m[m < 2.0 ** -47] = 0
    order = np.lexsort((np.arange(len(x)), -x))
    if k > 0:
        order = order[:k]
    if p < 1:
        before = np.cumsum(m[order]) - m[order]
        order = order[:max(1, int((before < max(p, 0.0) * m[order].sum()).sum()))]
    if mp > 0:
        order = order[m[order] >= min(mp, 1.0)]
    kept = np.sort(order)
    c = np.cumsum(m[kept])
    at = min(max(u, 0.0), 0.99999994) * c[-1]
    i = int(np.searchsorted(c, at, side="right"))
    # A border is a share F of the whole.  Weights that are off by up to 2^-31.5
    # of themselves move it by F (1 - F) 2 2^-31.5 <= 2^-32.5; the rounding to
    # whole multiples of 2^-46 (50,001 tokens; twice that for up to 131,072) by
    # half of one for each token on the smaller side, 2^-32 at most: in all
    # less than 2^-31.2.  This is 2^-30.97.
    near = np.abs(c - at).min() < 2.0 ** -21 * 1e-3 * c[-1]
    return int(kept[i]), math.log(m[kept[i]] / c[-1]), near and at > 0


def check_samples(rh, logits, u, **f):
    import torch

    def dev(v):
        return torch.from_numpy(v).cuda() if isinstance(v, np.ndarray) else v

    tokens, logprobs = rh.sample(dev(logits), dev(u), **{n: dev(v) for n, v in f.items()})
    tokens, logprobs = tokens.cpu().numpy(), logprobs.cpu().numpy()
    for r in range(len(u)):
        def at(n, d):
            v = f.get(n, d)
            return v[r].item() if isinstance(v, np.ndarray) else (np.float32(v).item() if n != "top_k" else v)

        want, lp, near = sample_ref(logits[r].copy(), float(u[r]), at("temperature", 1.0), at("top_k", 0),
                                    at("top_p", 1.0), at("min_p", 0.0))
        if near and tokens[r] != want:
            continue
        assert tokens[r] == want, (r, tokens[r], want, {n: at(n, 0) for n in f})
        # (The share is rounded once, its log once.)
        assert logprobs[r] == lp or abs(logprobs[r] - lp) <= 2 * U * max(1.0, abs(lp)) + 1e-9, (r, logprobs[r], lp)
    return tokens


FILTERS = [dict(), dict(top_k=1), dict(top_k=40), dict(top_p=0.9), dict(min_p=0.05), dict(top_k=40, top_p=0.9),
           dict(top_k=500, top_p=0.5, min_p=0.01), dict(temperature=0.0), dict(temperature=0.3, top_p=0.99),
           dict(temperature=3.0, top_k=10 ** 6), dict(top_p=0.0), dict(min_p=1.0), dict(min_p=7.0, top_k=3)]


@pytest.mark.parametrize("f", FILTERS, ids=str)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (2, 255), (5, 2048), (4, 2049), (2, 50001), (70, 5000)])
def test_sample(rh, f, rows, vocab):
    g = np.random.default_rng(rows * vocab)
    check_samples(rh, (g.standard_normal((rows, vocab)) * 3).astype(np.float32), g.random(rows, dtype=np.float32), **f)


@pytest.mark.parametrize("f", FILTERS, ids=str)
def test_sample_ties(rh, f):
    """Equal logits, in groups and everywhere, -0 and 0: the lowest index
    first."""
    g = np.random.default_rng(1)
    x = g.integers(-3, 4, (24, 5000)).astype(np.float32)
    x[8:16] = 1.5
    x[16:] = np.where(g.random((8, 5000)) < 0.5, np.float32(0), np.float32(-0.0))
    check_samples(rh, x, np.linspace(0, 0.999, 24, dtype=np.float32), **f)


def test_sample_filters_of_each_row(rh):
    g = np.random.default_rng(2)
    rows = 64
    x = (g.standard_normal((rows, 9000)) * 2).astype(np.float32)
    f = dict(temperature=g.choice([0.0, 0.5, 1.0, 1.7, np.nan, -1.0], rows).astype(np.float32),
             top_k=g.choice([-1, 0, 1, 7, 300, 8999, 9000, 2 ** 31 - 1], rows).astype(np.int32),
             top_p=g.choice([-1.0, 0.0, 0.1, 0.6, 0.95, 1.0, 2.0], rows).astype(np.float32),
             min_p=g.choice([-1.0, 0.0, 0.02, 0.5, 1.0], rows).astype(np.float32))
    check_samples(rh, x, g.random(rows, dtype=np.float32), **f)


@pytest.mark.parametrize("f", [dict(), dict(top_k=3), dict(top_p=0.7), dict(top_k=5, top_p=0.5, min_p=0.1), dict(temperature=0.0)], ids=str)
def test_sample_special_values(rh, f):
    """-inf and the type's lowest value as masks, NaN, +inf, rows of nothing
    else, and random numbers at and outside their range's ends."""
    g = np.random.default_rng(3)
    low = np.finfo(np.float32).min
    x = (g.standard_normal((14, 3000)) * 2).astype(np.float32)
    x[0, 1:] = -np.inf
    x[1] = -np.inf
    x[2] = np.nan
    x[3, ::2] = np.nan
    x[4, 10], x[4, 2000] = np.inf, np.inf
    x[5] = low
    x[6, 100:] = low
    x[7, :2999] = -np.inf
    x[8] = np.inf
    x[9] = -1e30
    x[10, 5] = 3e38
    x[11] = np.float32(1e-45) * g.integers(0, 3, 3000).astype(np.float32)
    u = g.random(14, dtype=np.float32)
    tokens = check_samples(rh, x, u, **f)
    assert tokens[1] == -1 and tokens[2] == -1 and tokens[7] == 2999
    for v in (0.0, 0.99999994, 1.0, 5.0, -3.0):
        check_samples(rh, x, np.full(14, v, np.float32), **f)
    nan = rh.sample(*[__import__("torch").from_numpy(a).cuda() for a in (x, np.full(14, np.nan, np.float32))], **f)[0]
    zero = rh.sample(*[__import__("torch").from_numpy(a).cuda() for a in (x, np.zeros(14, np.float32))], **f)[0]
    assert __import__("torch").equal(nan, zero)


def test_sample_strided_rows_and_repeats(rh):
    """Rows of a wider buffer, one row for all (stride 0), and the same call
    again: the same tokens."""
    import torch

    g = np.random.default_rng(4)
    wide = (g.standard_normal((6, 7001)) * 2).astype(np.float32)
    u = g.random(6, dtype=np.float32)
    d, du = torch.from_numpy(wide).cuda(), torch.from_numpy(u).cuda()
    a = [rh.sample(d[:, 1:6900], du, top_k=50, top_p=0.9) for _ in range(3)]
    b = rh.sample(d[:, 1:6900].contiguous(), du, top_k=50, top_p=0.9)
    for x in a:
        assert torch.equal(x[0], b[0]) and torch.equal(x[1], b[1])
    e = rh.sample(d[2:3].expand(6, 7001), du, top_p=0.8)
    want = [sample_ref(wide[2].copy(), float(v), 1.0, 0, float(np.float32(0.8)), 0.0)[0] for v in u]
    assert e[0].tolist() == want
    assert rh.sample(d[:0], du[:0])[0].shape == (0,)


@pytest.mark.parametrize("f", [dict(top_k=129), dict(top_k=5000, top_p=0.9), dict(top_k=3, top_p=0.3), dict(top_p=0.97, min_p=0.001),
                               dict(min_p=0.05), dict(temperature=30.0, top_p=0.8), dict(temperature=0.01, top_p=0.9),
                               dict(temperature=30.0, top_k=20000, top_p=0.5, min_p=0.5), dict()], ids=str)
@pytest.mark.parametrize("vocab", [16384, 16385, 32768, 32769, 131072])
def test_sample_large_vocabularies(rh, f, vocab):
    """At the ends of what one workgroup holds and past them: loud, faint,
    sorted, equal and nearly equal rows."""
    g = np.random.default_rng(vocab)
    x = (g.standard_normal((8, vocab)) * 2.5).astype(np.float32)
    x[1] *= np.float32(0.01)
    x[2] = np.sort(x[2])
    x[3] = -np.sort(x[3])
    x[4] = np.round(x[4])
    x[5] = np.float32(-1e30)
    x[6] = np.where(g.random(vocab) < 0.999, np.finfo(np.float32).min, x[6])
    x[7, g.integers(0, vocab, 3)] = np.inf
    check_samples(rh, x, g.random(8, dtype=np.float32), **f)


# ---------------------------------------------------------------------------
# Together
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("cache_type,page,window", [("float32", 16, 0), ("float16", 24, 0), ("bfloat16", 8, 40)])
def test_decoder_run(rh, cache_type, page, window):
    """Prompts in one step, then token by token, through two layers: every
    operator against its plain form on what the step gave it, the caches at the
    end against all tokens' rows."""
    import copy

    import torch

    prompts, steps, hq, hk, dim, vocab, layers = [70, 5, 33, 1], 5, 4, 2, 64, 1000, 2
    final = [n + steps for n in prompts]
    pages = Paged(prompts, final, page, seed=3)
    g = torch.Generator().manual_seed(11)

    def weights(*shape):
        return (torch.randn(*shape, generator=g) / math.sqrt(shape[0])).cuda()

    width = hq * dim
    embedding, head = weights(vocab, width) * math.sqrt(vocab), weights(width, vocab) * 3
    w_in = [weights(width, (hq + 2 * hk) * dim) for _ in range(layers)]
    w_out = [weights(width, width) for _ in range(layers)]
    scales = [(1 + 0.2 * torch.randn(2, dim, generator=g)).cuda() for _ in range(layers)]
    freq = (10000.0 ** (-torch.arange(dim // 2).double() / (dim // 2))).float().cuda()
    caches = [[torch.zeros(pages.n_pages, page, hk, dim, dtype=dtype(cache_type)).cuda() for _ in range(2)] for _ in range(layers)]
    rows = [[[] for _ in prompts] for _ in range(layers)]  # k as it came, of each layer and sequence
    tokens = torch.randint(0, vocab, (sum(prompts),), generator=g).cuda()
    f = dict(temperature=0.9, top_k=60, top_p=0.95)
    for step in range(steps + 1):
        s = copy.copy(pages)
        s.q_lens = prompts if step == 0 else [1] * len(prompts)
        s.kv_lens = [n + step for n in prompts]
        s.starts = np.concatenate(([0], np.cumsum(s.q_lens)))
        s.d_kv = torch.tensor(s.kv_lens, dtype=torch.int32).cuda()
        starts = torch.from_numpy(s.starts.astype(np.int32)).cuda() if step == 0 else None
        pos = np.concatenate([np.arange(kv - q, kv) for q, kv in zip(s.q_lens, s.kv_lens)])
        x = embedding[tokens]
        for i in range(layers):
            qkv = (x @ w_in[i]).view(-1, hq + 2 * hk, dim)
            q, k, v = qkv.split([hq, hk, hk], 1)
            kc, vc = caches[i]
            turned = rh.qk_norm_rotary_append(q, k, v, freq, kc, vc, s.d_table, s.d_kv, starts, q_scale=scales[i][0],
                                              k_scale=scales[i][1])
            rotary_close(turned.cpu().numpy(), rotary_ref(q.cpu().numpy(), pos, freq.cpu().numpy(),
                                                          scales[i][0].cpu().numpy(), 1e-6, False), "q")
            o = rh.paged_attention(turned, kc, vc, s.d_table, s.d_kv, starts, window=window, sinks=2 if window else 0)
            want, tol = attention_ref(turned.cpu().numpy(), kc.cpu().float().numpy(), vc.cpu().float().numpy(), s,
                                      1 / math.sqrt(dim), window, 2)
            attention_close(o.cpu().numpy(), want, tol, (step, i))
            for n in range(len(prompts)):
                rows[i][n].append(k[int(s.starts[n]):int(s.starts[n + 1])].cpu().numpy())
            x = x + o.reshape(-1, width) @ w_out[i]
        logits = x[torch.from_numpy(s.starts[1:] - 1).cuda()] @ head
        u = np.random.default_rng(step).random(len(prompts), dtype=np.float32)
        tokens = torch.from_numpy(check_samples(rh, logits.cpu().numpy(), u, **f)).cuda().long()
    step16 = 0 if cache_type == "float32" else torch.finfo(dtype(cache_type)).eps / 2
    for i in range(layers):
        k = caches[i][0].cpu().float().numpy()
        for n, kv in enumerate(final):
            want = rotary_ref(np.concatenate(rows[i][n]), np.arange(kv), freq.cpu().numpy(), scales[i][1].cpu().numpy(), 1e-6, False)
            for j in range(kv):
                p, o = pages.place(n, j)
                top = np.abs(want[j]).max(-1, keepdims=True)
                assert (np.abs(k[p, o] - want[j]) <= 24 * U * top + step16 * (1 + 24 * U) * np.abs(want[j]) + 2.0 ** -25).all()


class Step:
    """One token for each of some sequences: append, attention and a draw, on
    buffers that stay."""

    def __init__(self, rh, seed, kv_lens, cache_type="float16"):
        import torch

        self.rh, self.s = rh, Paged([1] * len(kv_lens), [n + 8 for n in kv_lens], 16, seed=seed)
        g = torch.Generator().manual_seed(seed)
        n = len(kv_lens)
        self.kv = torch.tensor(kv_lens, dtype=torch.int32).cuda()
        self.cache = torch.randn(2, self.s.n_pages, 16, 2, 64, generator=g).to(dtype(cache_type)).cuda()
        self.qkv, self.logits, self.u = torch.zeros(n, 12, 64).cuda(), torch.zeros(n, 40000).cuda(), torch.zeros(n).cuda()
        self.freq = torch.ones(32).cuda()
        self.inputs = [(torch.randn(n, 12, 64, generator=g).cuda(), (torch.randn(n, 40000, generator=g) * 3).cuda(),
                        torch.rand(n, generator=g).cuda()) for _ in range(5)]
        self.kv0, self.cache0 = self.kv.clone(), self.cache.clone()

    def reset(self):
        self.kv.copy_(self.kv0)
        self.cache.copy_(self.cache0)

    def feed(self, i):
        for to, x in zip((self.qkv, self.logits, self.u), self.inputs[i]):
            to.copy_(x)
        self.kv.add_(1)

    def run(self, ctx=None):
        q, k, v = self.qkv.split([8, 2, 2], 1)
        a = (self.cache[0], self.cache[1], self.s.d_table, self.kv)
        q = self.rh.qk_norm_rotary_append(q, k, v, self.freq, *a, ctx=ctx)
        o = self.rh.paged_attention(q, *a, ctx=ctx)
        return (q, o, *self.rh.sample(self.logits, self.u, top_p=0.9, ctx=ctx), *self.rh.sample(self.logits[:, :5000], self.u, top_k=50, ctx=ctx))

    def eager(self):
        self.reset()
        want = []
        for i in range(len(self.inputs)):
            self.feed(i)
            want.append([x.clone() for x in self.run()])
        return want, self.cache.clone()


def same(a, b):
    import torch

    return all(torch.equal(x, y) for x, y in zip(a, b))


def test_decoder_step_captured(rh):
    """A captured step, replayed on changing inputs and lengths with eager work
    between, gives the eager steps' bits; so do two graphs, replayed in turn on
    two streams."""
    import torch

    steps = [Step(rh, 1, [5, 900, 64, 3000]), Step(rh, 2, [17, 2, 40])]
    wants = [s.eager() for s in steps]
    graphs, outs = [], []
    for s in steps:
        s.reset()
        s.feed(0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            s.run()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(s.run())
        graphs.append(g)
    for s, (want, cache), g, out in zip(steps, wants, graphs, outs):
        s.reset()
        for i in range(len(want)):
            s.feed(i)
            g.replay()
            assert same(out, want[i]), i
            rh.sample(s.logits, s.u, top_k=7)  # eager work between
            torch.cuda.synchronize()
        assert torch.equal(s.cache, cache)
    streams = [torch.cuda.Stream() for _ in steps]
    for s in steps:
        s.reset()
    for i in range(len(wants[0][0])):
        for s in steps:
            s.feed(i)
        for g, st in zip(graphs, streams):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                g.replay()
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for out, (want, _) in zip(outs, wants):
            assert same(out, want[i]), i


def test_decoder_own_context(rh):
    """A context on a stream of its own, torch's current stream another one;
    two contexts at once."""
    import torch

    steps = [Step(rh, 3, [300, 31]), Step(rh, 4, [16, 4000])]
    wants = [s.eager() for s in steps]
    ctxs, streams = [rh.Context(0) for _ in steps], [torch.cuda.Stream() for _ in steps]
    for c, st in zip(ctxs, streams):
        c.sync_stream(st)
    for s in steps:
        s.reset()
    for i in range(len(wants[0][0])):
        outs = []
        for s in steps:
            s.feed(i)
        for s, c, st in zip(steps, ctxs, streams):
            st.wait_stream(torch.cuda.current_stream())
            outs.append(s.run(c))
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        for out, (want, _) in zip(outs, wants):
            assert same(out, want[i]), i
    torch.cuda.synchronize()
    for c in ctxs:
        c.close()


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("page", [16, 24])
@pytest.mark.parametrize("q_lens", [[1, 1], [40, 3]])
def test_decoder_large_cache(rh, cache_type, page, q_lens):
    """Pages past 2^31 elements and 2^32 bytes of a cache: the bits that a small
    one gives.  Keys and values lie side by side in one buffer."""
    import torch

    hk, dim, kv_lens = 8, 128, [200, 90]
    width = sum(-(-n // page) for n in kv_lens)
    g = torch.Generator().manual_seed(page)
    qkv = torch.randn(sum(q_lens), 16 + 2 * hk, dim, generator=g).cuda()
    start = torch.tensor([0, q_lens[0], sum(q_lens)], dtype=torch.int32).cuda()
    kv = torch.tensor(kv_lens, dtype=torch.int32).cuda()
    old = torch.randn(width, 2, page, hk, dim, generator=g).to(dtype(cache_type))
    got = []
    for n_pages in (width, 2 ** 31 // (page * hk * dim) + 3 * width):
        cache = torch.empty(n_pages, 2, page, hk, dim, dtype=dtype(cache_type), device="cuda")
        cache[n_pages - width:] = old.cuda()
        table = torch.full((2, width), -1, dtype=torch.int32)
        at = 0
        for s, n in enumerate(kv_lens):
            for p in range(-(-n // page)):
                table[s, p] = n_pages - 1 - at
                at += 1
        q, k, v = qkv.split([16, hk, hk], 1)
        a = (cache[:, 0], cache[:, 1], table.cuda(), kv, start)
        q = rh.qk_norm_rotary_append(q, k, v, None, *a)
        o = rh.paged_attention(q, *a)
        got.append((q, o, rh.paged_attention(q, *a), cache[n_pages - width:].clone()))
        del cache, a
    torch.cuda.empty_cache()
    assert same(*got) and torch.equal(got[0][1], got[0][2])
    assert got[0][1].abs().min() > 0


@pytest.mark.parametrize("vocab", [20000, 40000])
def test_sample_filters_of_each_row_large(rh, vocab):
    """As test_sample_filters_of_each_row, for rows of several blocks and rows
    that are cut; then each filter's array alone."""
    g = np.random.default_rng(vocab)
    rows = 40
    x = (g.standard_normal((rows, vocab)) * 2).astype(np.float32)
    x[3], x[4], x[5, 1:] = -np.inf, 2.5, -np.inf
    u = g.random(rows, dtype=np.float32)
    f = dict(temperature=g.choice([0.0, 0.5, 1.0, 1.7, np.nan, -1.0], rows).astype(np.float32),
             top_k=g.choice([-1, 0, 1, 7, 300, 5000, vocab - 1, vocab, 2 ** 31 - 1], rows).astype(np.int32),
             top_p=g.choice([-1.0, 0.0, 0.1, 0.6, 0.95, 1.0, 2.0], rows).astype(np.float32),
             min_p=g.choice([-1.0, 0.0, 0.02, 0.5, 1.0], rows).astype(np.float32))
    check_samples(rh, x, u, **f)
    for n, v in f.items():
        check_samples(rh, x, u, **{n: v})


def test_decoder_workspaces_hold_anything(rh, monkeypatch):
    """Memory that comes back with old contents: the same bits."""
    import torch

    import rten_hip.decoder as D

    s = Step(rh, 9, [5, 900, 64, 3000])
    want, _ = s.eager()
    plain = D._empty
    for byte in (0xff, 0x7f, 0):
        def dirty(like, shape, dtype, ctx, here):
            t = plain(like, shape, dtype, ctx, here)
            t.view(torch.uint8).fill_(byte)
            return t

        monkeypatch.setattr(D, "_empty", dirty)
        s.reset()
        for i in range(3):
            s.feed(i)
            assert same(s.run(), want[i])
            q = s.qkv[:, :8].repeat(40, 1, 1)  # a chunk of 40 tokens, kept as the first run gives it
            starts = torch.tensor([0, 40, 80, 120, 160], dtype=torch.int32).cuda()
            o = rh.paged_attention(q, s.cache[0], s.cache[1], s.s.d_table, s.kv, starts)
            if byte == 0xff and i == 0:
                first, start = o.clone(), q.clone()
            if i == 0:
                assert torch.equal(q, start) and torch.equal(o, first)


@pytest.mark.parametrize("f", [dict(), dict(top_k=7), dict(top_k=700), dict(top_p=0.4), dict(top_k=300, top_p=0.7),
                               dict(min_p=0.5), dict(top_p=0.9, min_p=1.0)], ids=str)
@pytest.mark.parametrize("vocab", [5, 1000, 30522, 40000])
def test_sample_infinite_temperature(rh, f, vocab):
    """All finite logits weigh the same; -infinity, NaN and what lies behind
    the row weigh nothing."""
    import torch

    g = np.random.default_rng(vocab)
    rows = 48
    x = (g.standard_normal((rows, vocab)) * 3).astype(np.float32)
    x[1::4][g.random((rows // 4, vocab)) < 0.6] = -np.inf
    x[2::4][g.random((rows // 4, vocab)) < 0.6] = np.nan
    x[3::4, vocab // 2:] = np.finfo(np.float32).min
    x[:, 1] = 2.0  # (some token is always there)
    u = np.linspace(0, 0.999999, rows).astype(np.float32)
    d, du = torch.from_numpy(x).cuda(), torch.from_numpy(u).cuda()
    arrays = dict(f, temperature=torch.full((rows,), math.inf).cuda())
    a, b = rh.sample(d, du, temperature=math.inf, **f), rh.sample(d, du, **arrays)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    tokens, logprobs = a[0].cpu().numpy(), a[1].cpu().numpy()
    for r in range(rows):
        y = np.where(np.isnan(x[r]), -np.inf, x[r]).astype(np.float64)
        order = np.lexsort((np.arange(vocab), -y))[:np.isfinite(y).sum()]
        order = order[:f.get("top_k", vocab)]
        # (Counts times a 24-bit number are exact.)
        n = len(order)
        order = order[:int((np.arange(n) < float(np.float32(f.get("top_p", 1.0))) * n).sum())]
        kept = np.sort(order)
        assert tokens[r] == kept[int(float(u[r]) * len(kept))], (r, tokens[r])
        want = -math.log(len(kept))
        assert abs(logprobs[r] - want) <= 2 * U * max(1.0, -want), (r, logprobs[r], want)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hq,dim", [(1, 64), (4, 128), (1, 192)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf])
def test_attention_infinite_keys_leave_their_neighbours(rh, cache_type, hq, dim, bad):
    """An infinity in a key whose values are finite: the rows before the token
    are as they are without it, also where the scores of those that see it
    are -infinity and leave nothing that is not finite."""
    for seed in range(4):
        for q_len, kv, back in ((40, 90, 1), (33, 70, 2), (300, 300, 7)):
            s = Paged([q_len], [kv], 16)
            at = kv - back
            p, o = s.place(0, at)

            def tweak(q, k, v):
                k[p, o, 0, 5] = bad

            got, q, k, v, scale = run_attention(rh, s, hq, 1, dim, cache_type, tweak=tweak, seed=seed)
            n = q_len - back  # rows before the token
            s2 = Paged([n], [at], 16)
            s2.table, s2.n_pages = s.table, s.n_pages
            want, tol = attention_ref(q[:n], k, v, s2, scale, 0, 0)
            attention_close(got[:n], want, tol, (seed, q_len, back))


@pytest.mark.parametrize("cache_type", ["float32", "bfloat16"])
@pytest.mark.parametrize("loud", [2.0 ** 13, 2.0 ** 20, 1e12, 1e30])
@pytest.mark.parametrize("q_len,kv,window,sinks,dim", [(40, 90, 0, 0, 64), (200, 700, 0, 0, 128), (60, 150, 20, 3, 64),
                                                       (30, 60, 0, 0, 256)])
def test_attention_loud_keys_leave_their_neighbours(rh, cache_type, loud, q_len, kv, window, sinks, dim):
    """Two keys that are far larger than the others, one that some rows do not
    see yet and one that, with a window, later rows do not see any more."""
    s = Paged([q_len], [kv], 16)

    def tweak(q, k, v):
        for at in [kv - 3] + ([kv - q_len - 10] if window else []):
            p, o = s.place(0, at)
            k[p, o] *= loud

    got, q, k, v, scale = run_attention(rh, s, 2, 1, dim, cache_type, window, sinks, tweak=tweak)
    want, tol = attention_ref(q, k, v, s, scale, window, sinks)
    attention_close(got, want, tol)


@pytest.mark.parametrize("cache_type", ["float32", "bfloat16"])
@pytest.mark.parametrize("loud", [2.0 ** 9, 2.0 ** 11, 2.0 ** 14, 2.0 ** 20, 1e12, 1e30])
@pytest.mark.parametrize("q_len,kv,window,sinks,dim", [(40, 90, 0, 0, 64), (200, 700, 0, 0, 128), (60, 150, 20, 3, 64),
                                                       (30, 60, 0, 0, 256), (300, 300, 0, 0, 96)])
def test_attention_loud_values_leave_their_neighbours(rh, cache_type, loud, q_len, kv, window, sinks, dim):
    """Values far larger than the others: of a token that some rows do not see
    yet, of a whole tile of such tokens, and, with a window, of tokens that
    later rows do not see any more."""
    s = Paged([q_len], [kv], 16)
    for where in ([kv - 3], range(kv - 20, kv), range(kv - q_len - 10, kv - q_len - 8) if window else [2]):
        def tweak(q, k, v):
            for at in where:
                p, o = s.place(0, at)
                v[p, o] *= loud

        got, q, k, v, scale = run_attention(rh, s, 2, 1, dim, cache_type, window, sinks, tweak=tweak)
        want, tol = attention_ref(q, k, v, s, scale, window, sinks)
        attention_close(got, want, tol, (loud, where))


@pytest.mark.parametrize("cache_type", ["float32", "bfloat16"])
@pytest.mark.parametrize("spread", [6, 30, 90])
def test_attention_values_of_all_sizes(rh, cache_type, spread):
    """Keys' values from 2^-spread to 2^spread, some all zero, in two sequences
    of which one is cut."""
    import torch

    s = Paged([50, 20], [1500, 70], 16)

    def tweak(q, k, v):
        g = torch.Generator().manual_seed(spread)
        v *= torch.exp2(torch.randint(-spread, spread + 1, v.shape[:3], generator=g).float())[..., None].to(v.dtype)
        v[torch.rand(v.shape[:3], generator=g) < 0.1] = 0

    got, q, k, v, scale = run_attention(rh, s, 4, 2, 64, cache_type, tweak=tweak)
    want, tol = attention_ref(q, k, v, s, scale, 0, 0)
    attention_close(got, want, tol)


@pytest.mark.parametrize("cache_type", TYPES)
@pytest.mark.parametrize("hq,hk,dim,q_len", [(8, 1, 64, 1), (2, 1, 64, 40), (3, 1, 128, 70), (1, 1, 256, 33)])
@pytest.mark.parametrize("base", [2.0 ** 21, 2.0 ** 24, 2.0 ** 25, 2.0 ** 26, 2.0 ** 27, -2.0 ** 26, -2.0 ** 27])
def test_attention_scores_of_few_bits_behind_the_point(rh, cache_type, hq, hk, dim, q_len, base):
    """Scores so large that whole numbers are rounded, rising by one step of
    float32 from one stretch of keys to the next, all sums exact."""
    import torch

    kv = 200
    s = Paged([q_len], [kv], 16)
    # scale log2 e is 1: the weights are powers of two.
    scale = np.float32(math.log(2))
    assert scale * np.float32(1.44269504088896340736) == 1
    step = 2.0 ** max(0, int(math.log2(abs(base))) - 23)
    root = 2.0 ** 12
    rise = np.arange(kv) // 30

    def tweak(q, k, v):
        q.zero_()
        q[..., 0], q[..., 1] = abs(base) / root, step
        k.zero_()
        for j in range(kv):
            p, o = s.place(0, j)
            k[p, o, :, 0], k[p, o, :, 1] = math.copysign(root, base), float(rise[j])

    got, q, k, v, _ = run_attention(rh, s, hq, hk, dim, cache_type, tweak=tweak, scale=float(scale))
    vv = np.stack([v[s.place(0, j)] for j in range(kv)])[:, 0].astype(np.float64)
    for t in range(q_len):
        n = kv - q_len + t + 1
        w = np.exp2((rise[:n] - rise[n - 1]) * step)
        want = (w / w.sum()) @ vv[:n]
        # (The sums over the keys, the split of p and v, the powers and the
        # quotient: as attention_ref counts them.)
        assert (np.abs(got[t] - want) <= (n / 16 + 40) * U * np.abs(vv[:n]).max()).all(), t


@pytest.mark.parametrize("q_len", [1, 40])
def test_attention_joins_values_near_the_end_of_the_range(rh, q_len):
    """A float32 cache's values at 2^-12 of the largest number, in a sequence
    that is cut into stretches."""
    s = Paged([q_len], [2000], 16)

    def tweak(q, k, v):
        v *= 3e35 / 4

    got, q, k, v, scale = run_attention(rh, s, 2, 1, 64, "float32", tweak=tweak)
    want, tol = attention_ref(q, k, v, s, scale, 0, 0)
    attention_close(got, want, tol)


def test_decoder_threads(rh):
    """Two threads, each with its stream as torch's current one and without a
    context of its own: the bits of the eager steps."""
    import threading

    import torch

    steps = [Step(rh, 5, [300, 31]), Step(rh, 6, [16, 4000])]
    wants = [s.eager()[0] for s in steps]
    torch.cuda.synchronize()
    turn, failed = threading.Barrier(2, timeout=60), []

    def work(s, want):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(10):
                    s.reset()
                    for i in range(len(want)):
                        s.feed(i)
                        turn.wait()
                        if not same(s.run(), want[i]):
                            failed.append(i)
                torch.cuda.current_stream().synchronize()
        except Exception as e:
            failed.append(e)
            turn.abort()

    threads = [threading.Thread(target=work, args=a) for a in zip(steps, wants)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(100)
    assert not failed, failed


@pytest.mark.parametrize("inter", [False, True])
def test_rotary_turns_are_rounded_once(rh, inter):
    """Pairs (1, 0) turn into cos and sin, off by half a step of float32."""
    import torch

    pos = torch.cat([torch.arange(300), torch.randint(0, 1_000_000, (300,), generator=torch.Generator().manual_seed(1))]).int()
    half = 64
    freq = (10000.0 ** (-torch.arange(half).double() / half)).float()
    x = torch.zeros(len(pos), 1, 2 * half)
    x[..., 0::2] = 1
    if not inter:
        x = torch.cat((torch.ones(len(pos), 1, half), torch.zeros(len(pos), 1, half)), -1)
    got = rh.qk_norm_rotary(x.cuda(), x.cuda(), pos.cuda(), freq.cuda(), interleaved=inter)[0].cpu().numpy()[:, 0]
    a = pos.numpy().astype(np.float64)[:, None] * freq.numpy().astype(np.float64)
    for part, want in ((slice(0, None, 2) if inter else slice(0, half), np.cos(a)),
                       (slice(1, None, 2) if inter else slice(half, None), np.sin(a))):
        # (2^-36 of the series left out beside half a step, 2^-25 at least of a
        # number above 1/2; smaller cosines and sines come from smaller x.)
        step = np.spacing(np.abs(want).astype(np.float32)).astype(np.float64)
        assert (np.abs(got[:, part] - want) <= step * (0.5 + 2.0 ** -10)).all()


def test_thread_ends_before_its_work(rh):
    """A thread's context goes with it; what it queued is still done."""
    import threading

    import torch

    x, w = torch.randn(2048, 2048).cuda(), torch.randn(2048, 2048).cuda()
    want, got = rh.matmul(x, w), []

    def work():
        got.append([rh.matmul(x, w) for _ in range(20)][-1])

    for _ in range(3):
        t = threading.Thread(target=work)
        t.start()
        t.join(60)
    torch.cuda.synchronize()
    assert len(got) == 3 and all(torch.equal(y, want) for y in got)
