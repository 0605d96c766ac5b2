"""Refusals and sizes of the decoder operators' C entry points (no GPU): every
check comes before the context is looked at, so a call with a null context
returns the check's error, or "Missing context" where all checks pass."""
import ctypes as C
import math
import os
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
PKG = os.path.join(ROOT, "rten-fork_amd")

TYPE, SHAPES, MISSING, VALUE, UNSUPPORTED = 1, 3, 4, 5, 6
BASE = 1 << 20  # an address that is never read: buffers of the calls lie 1 GiB apart
GIB = 1 << 30


@pytest.fixture(scope="module")
def d():
    if not os.path.exists(os.path.join(PKG, "librten_hip.so")):
        subprocess.check_call(["make", "-s", "-j8", "-C", PKG])
    import rten_hip
    from rten_hip import decoder

    decoder.message = lambda: rten_hip.lib().rtenhip_last_error_message().decode()
    return decoder


def call(d, name, *args):
    import rten_hip

    f = getattr(rten_hip.lib(), name)
    f.argtypes, f.restype = d._SIGNATURES[name], C.c_int
    return f(*args), d.message()


def tensor(d, n, *shape, strides=None, at=0):
    if strides is None:
        strides = [math.prod(shape[i + 1:]) for i in range(len(shape))]
    return d.Tensor(BASE + n * GIB + at, len(shape), tuple(shape), tuple(strides))


def cache(d, dtype=0, page=16, pages=10, heads=2, dim=64, **kw):
    st = (page * heads * dim, heads * dim, dim)
    f = dict(k=BASE + 20 * GIB, v=BASE + 30 * GIB, dtype=dtype, page_size=page, n_pages=pages, n_heads=heads, head_dim=dim,
             k_strides=st, v_strides=st)
    f.update(kw)
    return d.KVCache(**f)


def seqs(d, n=3, pages=4, starts=True, **kw):
    f = dict(page_table=BASE + 40 * GIB, table_stride=pages, kv_lens=BASE + 41 * GIB,
             q_starts=BASE + 42 * GIB if starts else None, n_seqs=n, max_pages=pages)
    f.update(kw)
    return d.Sequences(**f)


def rotary(d, **kw):
    f = dict(q_scale=None, k_scale=None, inv_freq=BASE + 50 * GIB, positions=BASE + 51 * GIB, epsilon=1e-6, rotary_dim=64,
             interleaved=0)
    f.update(kw)
    return d.Rotary(**f)


def attention(d, q=None, c=None, s=None, scale=0.1, window=0, sinks=0, ws=BASE + 60 * GIB, ws_bytes=1 << 40, out=None):
    q, c, s = q or tensor(d, 0, 5, 4, 64), c or cache(d), s or seqs(d)
    out = out or tensor(d, 1, 5, 4, 64)
    return call(d, "rtenhip_paged_attention_f32", None, C.byref(q), C.byref(c), C.byref(s), scale, window, sinks, ws,
                ws_bytes, C.byref(out))


def workspace(d, q, c, s):
    n = C.c_size_t()
    st, msg = call(d, "rtenhip_paged_attention_workspace", C.byref(q), C.byref(c), C.byref(s), C.byref(n))
    assert st == 0, msg
    return n.value


def test_attention_accepts(d):
    ok = (MISSING, "Missing context")
    assert attention(d) == ok
    for dtype in (0, 1, 2):
        assert attention(d, c=cache(d, dtype)) == ok
    assert attention(d, window=2 ** 31 - 1, sinks=2 ** 31 - 1) == ok
    assert attention(d, s=seqs(d, 5, starts=False)) == ok
    q = tensor(d, 0, 5, 4, 64, strides=[1000, 100, 1])
    assert attention(d, q=q, out=q) == ok
    # Heads before slots; a page shared by all (stride 0) is read only.
    assert attention(d, c=cache(d, k_strides=(2048, 64, 1024))) == ok
    assert attention(d, c=cache(d, k_strides=(0, 128, 64))) == ok
    # Side by side in the same rows.
    assert attention(d, q=tensor(d, 0, 5, 4, 64, strides=[512, 64, 1]),
                     out=tensor(d, 0, 5, 4, 64, strides=[512, 64, 1], at=1024)) == ok


@pytest.mark.parametrize("code,text,kw", [
    (SHAPES, "Expected [tokens, heads, head_dim]", dict(q=(5, 256))),
    (SHAPES, "multiple of the cache's", dict(q=(5, 3, 64))),
    (SHAPES, "cache's head_dim", dict(q=(5, 4, 128))),
    (SHAPES, "shape of q", dict(out=(5, 2, 64))),
    (VALUE, "Invalid input size", dict(q=(5, 0, 64))),
    (UNSUPPORTED, "Too many query rows", dict(q=(1 << 29, 4, 64))),
    (TYPE, "Cache must be", dict(c=dict(dtype=3))),
    (VALUE, "Invalid cache size", dict(c=dict(page=0))),
    (VALUE, "Invalid cache size", dict(c=dict(page=65537))),
    (VALUE, "Invalid cache size", dict(c=dict(heads=0))),
    (VALUE, "Invalid cache size", dict(c=dict(pages=-1))),
    (UNSUPPORTED, "head_dim", dict(c=dict(dim=60))),
    (UNSUPPORTED, "head_dim", dict(c=dict(dim=264))),
    (MISSING, "Missing cache", dict(c=dict(k=None))),
    (UNSUPPORTED, "16 bytes", dict(c=dict(v=BASE + 8))),
    (UNSUPPORTED, "16 bytes", dict(c=dict(k_strides=(2048, 130, 64)))),
    (UNSUPPORTED, "16 bytes", dict(c=dict(dtype=1, k_strides=(2048, 132, 64)))),
    (UNSUPPORTED, "Unsupported cache strides", dict(c=dict(k_strides=(-2048, 128, 64)))),
    (VALUE, "Invalid sequences", dict(s=dict(n=-1))),
    (VALUE, "Invalid sequences", dict(s=dict(max_pages=-1))),
    (SHAPES, "one row per sequence", dict(s=dict(starts=False))),
    (MISSING, "Missing sequences", dict(s=dict(kv_lens=None))),
    (MISSING, "Missing sequences", dict(s=dict(page_table=None))),
    (UNSUPPORTED, "on 4 bytes", dict(s=dict(kv_lens=BASE + 2))),
    (VALUE, "window and sinks", dict(window=-1)),
    (VALUE, "window and sinks", dict(sinks=-1)),
    (VALUE, "scale must be finite", dict(scale=math.nan)),
    (VALUE, "scale must be finite", dict(scale=math.inf)),
    (VALUE, "Workspace is too small", dict(s=dict(pages=5), ws_bytes=100)),
    (VALUE, "Workspace is too small", dict(s=dict(pages=5), ws=None)),
    (UNSUPPORTED, "Workspace must be on 16", dict(ws=BASE + 8)),
])
def test_attention_refuses(d, code, text, kw):
    kw = dict(kw)
    for n, make in (("q", lambda v: tensor(d, 0, *v)), ("out", lambda v: tensor(d, 1, *v)), ("c", lambda v: cache(d, **v)),
                    ("s", lambda v: seqs(d, **v))):
        if n in kw:
            kw[n] = make(kw[n])
    st, msg = attention(d, **kw)
    assert st == code and text in msg, (st, msg)


def test_attention_refuses_views(d):
    for bad in (dict(strides=[256, 64, 2]), dict(strides=[258, 64, 1]), dict(strides=[256, 66, 1]), dict(at=4),
                dict(strides=[-256, 64, 1])):
        st, msg = attention(d, q=tensor(d, 0, 5, 4, 64, **bad))
        assert st == UNSUPPORTED and "Head rows" in msg, (bad, msg)
    st, msg = attention(d, out=tensor(d, 1, 5, 4, 64, strides=[0, 64, 1]))
    assert st == VALUE and "must not overlap" in msg
    st, msg = attention(d, out=tensor(d, 1, 5, 4, 64, strides=[128, 64, 1]))
    assert st == VALUE and "must not overlap" in msg
    st, msg = attention(d, out=tensor(d, 0, 5, 4, 64, at=16))
    assert st == VALUE and "share memory" in msg
    st, msg = attention(d, q=tensor(d, 0, 5, 4, 64, strides=[512, 64, 1]),
                        out=tensor(d, 0, 5, 4, 64, strides=[512, 64, 1], at=512))
    assert st == VALUE and "share memory" in msg


def test_attention_workspace(d):
    # Nothing can be cut where no sequence has more than one tile of keys.
    assert workspace(d, tensor(d, 0, 5, 4, 64), cache(d), seqs(d, pages=4)) == 0
    n = workspace(d, tensor(d, 0, 5, 4, 64), cache(d), seqs(d, pages=5))
    assert n > 0 and attention(d, s=seqs(d, pages=5), ws_bytes=n) == (MISSING, "Missing context")
    assert attention(d, s=seqs(d, pages=5), ws_bytes=n - 1)[0] == VALUE
    assert workspace(d, tensor(d, 0, 0, 4, 64), cache(d), seqs(d, 3, pages=5)) < n


def rot(d, q=None, k=None, r=None, qo=None, ko=None):
    q, k, r = q or tensor(d, 0, 5, 4, 64), k or tensor(d, 1, 5, 2, 64), r or rotary(d)
    qo, ko = qo or tensor(d, 2, 5, 4, 64), ko or tensor(d, 3, 5, 2, 64)
    return call(d, "rtenhip_qk_norm_rotary_f32", None, *map(C.byref, (q, k, r, qo, ko)))


def test_rotary(d):
    ok = (MISSING, "Missing context")
    q, k = tensor(d, 0, 5, 4, 64, strides=[512, 64, 1]), tensor(d, 0, 5, 2, 64, strides=[512, 64, 1], at=1024)
    assert rot(d) == ok and rot(d, q=q, k=k) == ok and rot(d, q=q, k=k, qo=q, ko=k) == ok
    assert rot(d, r=rotary(d, rotary_dim=0, inv_freq=None, positions=None)) == ok
    for code, text, kw in (
            (SHAPES, "Expected [tokens", dict(q=tensor(d, 0, 5, 256))),
            (SHAPES, "same tokens and head_dim", dict(k=tensor(d, 1, 4, 2, 64))),
            (SHAPES, "same tokens and head_dim", dict(ko=tensor(d, 3, 5, 4, 64))),
            (UNSUPPORTED, "head_dim", dict(q=tensor(d, 0, 5, 4, 4), k=tensor(d, 1, 5, 4, 4))),
            (UNSUPPORTED, "head_dim", dict(q=tensor(d, 0, 5, 4, 512))),
            (UNSUPPORTED, "rotary_dim", dict(r=rotary(d, rotary_dim=72))),
            (UNSUPPORTED, "rotary_dim", dict(r=rotary(d, rotary_dim=12))),
            (VALUE, "epsilon", dict(r=rotary(d, epsilon=-1e-6))),
            (VALUE, "epsilon", dict(r=rotary(d, epsilon=math.nan))),
            (MISSING, "inv_freq", dict(r=rotary(d, inv_freq=None))),
            (MISSING, "positions", dict(r=rotary(d, positions=None))),
            (UNSUPPORTED, "on 4 bytes", dict(r=rotary(d, q_scale=BASE + 2))),
            (UNSUPPORTED, "Head rows", dict(q=tensor(d, 0, 5, 4, 64, at=4))),
            (VALUE, "must not overlap", dict(qo=tensor(d, 2, 5, 4, 64, strides=[0, 64, 1]))),
            (VALUE, "must not overlap", dict(ko=tensor(d, 2, 5, 2, 64, strides=[128, 0, 1]))),
            (VALUE, "share memory", dict(qo=tensor(d, 1, 5, 4, 64))),
            (VALUE, "share memory", dict(ko=tensor(d, 0, 5, 2, 64))),
            (VALUE, "share memory", dict(ko=tensor(d, 2, 5, 2, 64, at=64)))):
        st, msg = rot(d, **kw)
        assert st == code and text in msg, (kw, st, msg)


def test_append(d):
    def app(q=None, k=None, v=None, r=None, c=None, s=None, out=None):
        q, k, v = q or tensor(d, 0, 5, 4, 64), k or tensor(d, 1, 5, 2, 64), v or tensor(d, 2, 5, 2, 64)
        return call(d, "rtenhip_qk_norm_rotary_append_f32", None, C.byref(q), C.byref(k), C.byref(v),
                    C.byref(r or rotary(d, positions=None)), C.byref(c or cache(d)), C.byref(s or seqs(d)),
                    C.byref(out or tensor(d, 3, 5, 4, 64)))

    assert app() == (MISSING, "Missing context")
    for code, text, kw in (
            (SHAPES, "v must have the shape of k", dict(v=tensor(d, 2, 5, 4, 64))),
            (SHAPES, "Cache heads", dict(c=cache(d, heads=4))),
            (SHAPES, "Cache heads", dict(c=cache(d, dim=128))),
            (SHAPES, "one row per sequence", dict(s=seqs(d, starts=False))),
            (VALUE, "Cache rows must not overlap", dict(c=cache(d, k_strides=(0, 128, 64)))),
            (VALUE, "Cache rows must not overlap", dict(c=cache(d, v_strides=(1024, 128, 64)))),
            (VALUE, "share memory", dict(out=tensor(d, 1, 5, 4, 64))),
            (VALUE, "share memory", dict(out=tensor(d, 2, 5, 4, 64, at=256)))):
        st, msg = app(**kw)
        assert st == code and text in msg, (kw, st, msg)


def test_more_workgroups_than_a_launch_has(d):
    """A launch has fewer than 2^32 threads."""
    n = (1 << 24) - 1
    assert rot(d, q=tensor(d, 0, n, 1, 8), k=tensor(d, 100, n, 1, 8), qo=tensor(d, 200, n, 1, 8), ko=tensor(d, 300, n, 1, 8),
               r=rotary(d, rotary_dim=8)) == (MISSING, "Missing context")
    n += 1
    assert rot(d, q=tensor(d, 0, n, 1, 8), k=tensor(d, 100, n, 1, 8), qo=tensor(d, 200, n, 1, 8), ko=tensor(d, 300, n, 1, 8),
               r=rotary(d, rotary_dim=8)) == (UNSUPPORTED, "Too many tokens")
    c, s = cache(d, heads=64, dim=8), seqs(d, 1 << 18, pages=1, starts=False)
    st, msg = attention(d, q=tensor(d, 0, 1 << 18, 64, 8), c=c, s=s, out=tensor(d, 100, 1 << 18, 64, 8))
    assert st == UNSUPPORTED and "Too many query rows" in msg
    s = seqs(d, (1 << 18) - 1, pages=1, starts=False)
    assert attention(d, q=tensor(d, 0, (1 << 18) - 1, 64, 8), c=c, s=s,
                     out=tensor(d, 100, (1 << 18) - 1, 64, 8)) == (MISSING, "Missing context")


def test_sample(d):
    def samp(x=None, f=None, u=BASE + 5 * GIB, ws=BASE + 6 * GIB, n=1 << 40, tokens=BASE + 7 * GIB, lp=None):
        return call(d, "rtenhip_sample_f32", None, C.byref(x or tensor(d, 0, 3, 1000)),
                    C.byref(f or d.Sampling(1.0, 1.0, 0.0, 0)), u, ws, n, tokens, lp)

    ok = (MISSING, "Missing context")
    assert samp() == ok
    assert samp(x=tensor(d, 0, 3, 1 << 24)) == ok
    assert samp(x=tensor(d, 0, 3, 1000, strides=[0, 1])) == ok
    assert samp(x=tensor(d, 0, 0, 1000), u=None, ws=None, tokens=None)[0] == 0
    need = C.c_size_t()
    assert call(d, "rtenhip_sample_workspace", 3, 1000, C.byref(need))[0] == 0 and need.value > 0
    assert samp(n=need.value) == ok and samp(n=need.value - 1) == (VALUE, "Workspace is too small")
    for code, text, kw in (
            (SHAPES, "Expected [rows, vocab]", dict(x=tensor(d, 0, 3, 10, 10))),
            (VALUE, "Invalid logits size", dict(x=tensor(d, 0, 3, 0))),
            (UNSUPPORTED, "Vocabulary", dict(x=tensor(d, 0, 3, (1 << 24) + 1))),
            (UNSUPPORTED, "Too many rows", dict(x=tensor(d, 0, (1 << 20) + 1, 10))),
            (UNSUPPORTED, "unit stride", dict(x=tensor(d, 0, 3, 1000, strides=[2000, 2]))),
            (UNSUPPORTED, "unit stride", dict(x=tensor(d, 0, 3, 1000, strides=[-1000, 1]))),
            (UNSUPPORTED, "on 4 bytes", dict(u=BASE + 1)),
            (UNSUPPORTED, "on 4 bytes", dict(f=d.Sampling(1.0, 1.0, 0.0, 0, temperatures=BASE + 2))),
            (UNSUPPORTED, "Workspace must be on 16", dict(ws=BASE + 4)),
            (VALUE, "Workspace is too small", dict(ws=None)),
            (MISSING, "Missing input", dict(u=None)), (MISSING, "Missing input", dict(tokens=None))):
        st, msg = samp(**kw)
        assert st == code and text in msg, (kw, st, msg)


@pytest.mark.parametrize("rows,vocab", [(1, 1), (4096, 1000), (100, 32768), (1000, 32769), (2, 131072), (1, 1 << 24)])
def test_sample_workspace(d, rows, vocab):
    """16 bytes for each 1024 tokens of a row; from 32,769 tokens on what
    gathers its candidates too, no more than 27 KB for each row and stretch."""
    need = C.c_size_t()
    assert call(d, "rtenhip_sample_workspace", rows, vocab, C.byref(need))[0] == 0
    blocks = -(-vocab // 1024)
    small = rows * blocks * 16 + 10 * 256
    stretches = min(64, -(-blocks // 4), max(1, 1024 // rows))
    assert need.value <= (small if vocab <= 32768 else small + rows * (stretches * 27000 + 10000))
    assert need.value >= rows * blocks * 16


def test_null_descriptors(d):
    n = C.c_size_t()
    assert call(d, "rtenhip_paged_attention_workspace", None, None, None, C.byref(n))[0] == MISSING
    assert call(d, "rtenhip_paged_attention_workspace", None, None, None, None)[0] == MISSING
    assert call(d, "rtenhip_paged_attention_f32", None, None, None, None, 1.0, 0, 0, None, 0, None)[0] == MISSING
    assert call(d, "rtenhip_qk_norm_rotary_f32", *[None] * 6)[0] == MISSING
    assert call(d, "rtenhip_qk_norm_rotary_append_f32", *[None] * 8)[0] == MISSING
    assert call(d, "rtenhip_sample_f32", *[None] * 5, 0, None, None)[0] == MISSING
    assert call(d, "rtenhip_sample_workspace", 1, 1, None)[0] == MISSING


def test_python_binding_refuses_before_the_library(d):
    """Types, devices and sizes that the descriptors do not carry."""
    torch = pytest.importorskip("torch")
    from rten_hip import OpError

    class Ctx:  # no GPU here: the checks only compare the device's number
        device, ptr = 0, None

    x = torch.zeros(3, 2, 64)
    with pytest.raises(OpError, match="must be on the context's GPU"):
        d._rows(x, Ctx, "q")
    with pytest.raises(OpError, match="expected float32"):
        d._rows(x.half(), Ctx, "q")
    with pytest.raises(OpError, match="expected int32"):
        d._vector(torch.zeros(3, dtype=torch.int64), 3, Ctx, torch.int32, "kv_lens")
    c = torch.zeros(4, 16, 2, 64)
    for k, v, msg in ((c, c[:2], "same shape"), (c[0], c[0], "same shape"), (c.double(), c.double(), "must be float32"),
                      (c, c, "GPU")):
        with pytest.raises(OpError, match=msg):
            d._cache(k, v, Ctx)


class NoGPU:
    """A context of the CPU: a call gets as far as the library's own check of it."""
    device, ptr, stream = -1, None, None


@pytest.fixture
def on_cpu(d, monkeypatch):
    monkeypatch.setattr(d, "_context", lambda ctx: (NoGPU, True))
    return d


@pytest.mark.parametrize("each", ["temperature", "top_k", "top_p", "min_p"])
def test_sample_no_rows(on_cpu, each):
    """Filters of each of no rows."""
    torch = pytest.importorskip("torch")
    none = torch.empty(0, dtype=torch.int32 if each == "top_k" else torch.float32)
    tokens, logprobs = on_cpu.sample(torch.zeros(0, 10), torch.zeros(0), **{each: none})
    assert tokens.shape == logprobs.shape == (0,)


def test_numbers_past_float32(on_cpu):
    """They reach the library as infinities, or are refused as it refuses them."""
    torch = pytest.importorskip("torch")
    from rten_hip import OpError

    for kw in (dict(temperature=1e39), dict(top_p=1e300), dict(min_p=-1e39), dict(temperature=-math.inf, min_p=1e39)):
        with pytest.raises(OpError, match="Missing context"):
            on_cpu.sample(torch.zeros(2, 10), torch.zeros(2), **kw)
    x = torch.zeros(2, 1, 64)
    for epsilon, text in ((1e39, "epsilon"), (-1e-9, "epsilon"), (math.inf, "Missing context")):
        with pytest.raises(OpError, match=text):
            on_cpu.qk_norm_rotary(x, x, torch.zeros(2, dtype=torch.int32), None, epsilon=epsilon)
    n = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(OpError, match="scale must be finite"):
        on_cpu.paged_attention(x, torch.zeros(3, 16, 1, 64), torch.zeros(3, 16, 1, 64), n[:, None], n, scale=1e39)


def test_default_context_of_each_thread(monkeypatch):
    """Two threads on two streams: each one's calls stay on its own, however
    they interleave."""
    import threading

    import rten_hip

    here = threading.local()

    class Recorder:  # a context that notes the stream it was set to last
        def __init__(self, device):
            self.device, self.stream = device, None

        def sync_stream(self):
            self.stream = here.stream

    monkeypatch.setattr(rten_hip, "Context", Recorder)
    if hasattr(rten_hip, "_default_ctx"):
        monkeypatch.setattr(rten_hip, "_default_ctx", None)
    turn, seen = threading.Barrier(2, timeout=20), {}

    def work(name):
        here.stream = name
        ctx = rten_hip.default_context()
        turn.wait()  # both have set their stream
        seen[name] = (ctx, ctx.stream, rten_hip.default_context())

    threads = [threading.Thread(target=work, args=(n,)) for n in "ab"]
    for t in threads:
        t.start()
    for t in threads:
        t.join(30)
    for name in "ab":
        ctx, stream, again = seen[name]
        assert stream == name and again is ctx
    assert seen["a"][0] is not seen["b"][0]


def test_packed_descriptors_have_the_structures_layouts(d):
    """The bytes that the binding passes, field by field."""
    def same(kind, packed, **fields):
        s = kind.from_buffer_copy(packed)
        assert C.sizeof(kind) == len(packed)
        for name, want in fields.items():
            got = getattr(s, name)
            assert (tuple(got) if hasattr(got, "__len__") else got) == want, name

    same(d.Tensor, d._ROWS.pack(7, 3, 1, 2, 3, 6, 5, 4), data=7, ndim=3, shape=(1, 2, 3, 0, 0, 0, 0, 0),
         strides=(6, 5, 4, 0, 0, 0, 0, 0))
    same(d.Tensor, d._MATRIX.pack(7, 2, 1, 2, 6, 5), data=7, ndim=2, shape=(1, 2) + (0,) * 6, strides=(6, 5) + (0,) * 6)
    same(d.KVCache, d._CACHE.pack(1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13), k=1, v=2, dtype=3, page_size=4, n_pages=5,
         n_heads=6, head_dim=7, k_strides=(8, 9, 10), v_strides=(11, 12, 13))
    same(d.Sequences, d._SEQUENCES.pack(1, 2, 3, 4, 5, 6), page_table=1, table_stride=2, kv_lens=3, q_starts=4, n_seqs=5,
         max_pages=6)
    same(d.Rotary, d._ROTARY.pack(1, 2, 3, 4, 0.5, 6, 7), q_scale=1, k_scale=2, inv_freq=3, positions=4, epsilon=0.5,
         rotary_dim=6, interleaved=7)
    same(d.Sampling, d._SAMPLING.pack(0.5, 0.25, 0.125, 4, 5, 6, 7, 8), temperature=0.5, top_p=0.25, min_p=0.125, top_k=4,
         temperatures=5, top_ps=6, min_ps=7, top_ks=8)
