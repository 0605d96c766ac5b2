"""Operators of a decoder that answers token by token (the "decoder operators"
of include/rten_hip.h): the norm and rotation of queries and keys, attention
over a paged cache, and sampling.

A cache is a pair of device tensors ``[pages, page size, heads, head_dim]``
(float32, float16 or bfloat16, any order of the first three dimensions in
memory, e.g. a transposed ``[pages, heads, page size, head_dim]``).  Sequence s
owns the pages in row s of ``page_table`` (int32, -1 = none) and has
``kv_lens[s]`` tokens there.  The rows of a call are the new tokens of its
sequences, one after the other: ``q_starts[s]`` .. ``q_starts[s + 1]`` - 1 for
sequence s; without ``q_starts`` row s is the one new token of sequence s.
Rows from ``q_starts[-1]`` on are padding and left as they are.  ``kv_lens``
counts the new tokens: append before attending.  All calls only queue work on
the context's stream and can be captured.  Without ``ctx`` that is the calling
thread's own context on torch's current stream; a context that is given is used
by one thread at a time.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct

from . import OpError, Tensor, _torch, check, default_context, lib  # noqa: F401  (Tensor: the row descriptors' layout)


class KVCache(C.Structure):
    """rtenhip_kv_cache."""
    _fields_ = [("k", C.c_void_p), ("v", C.c_void_p), ("dtype", C.c_int32), ("page_size", C.c_int32),
                ("n_pages", C.c_int64), ("n_heads", C.c_int32), ("head_dim", C.c_int32),
                ("k_strides", C.c_int64 * 3), ("v_strides", C.c_int64 * 3)]


class Sequences(C.Structure):
    """rtenhip_sequences."""
    _fields_ = [("page_table", C.c_void_p), ("table_stride", C.c_int64), ("kv_lens", C.c_void_p),
                ("q_starts", C.c_void_p), ("n_seqs", C.c_int32), ("max_pages", C.c_int32)]


class Rotary(C.Structure):
    """rtenhip_rotary."""
    _fields_ = [("q_scale", C.c_void_p), ("k_scale", C.c_void_p), ("inv_freq", C.c_void_p),
                ("positions", C.c_void_p), ("epsilon", C.c_float), ("rotary_dim", C.c_int32),
                ("interleaved", C.c_int32)]


class Sampling(C.Structure):
    """rtenhip_sampling."""
    _fields_ = [("temperature", C.c_float), ("top_p", C.c_float), ("min_p", C.c_float), ("top_k", C.c_int32),
                ("temperatures", C.c_void_p), ("top_ps", C.c_void_p), ("min_ps", C.c_void_p),
                ("top_ks", C.c_void_p)]


_P = C.c_void_p
_SIGNATURES = {
    "rtenhip_qk_norm_rotary_f32": [_P] * 6,
    "rtenhip_qk_norm_rotary_append_f32": [_P] * 8,
    "rtenhip_paged_attention_workspace": [_P] * 4,
    "rtenhip_paged_attention_f32": [_P, _P, _P, _P, C.c_float, C.c_int32, C.c_int32, _P, C.c_size_t, _P],
    "rtenhip_sample_workspace": [C.c_int64, C.c_int64, _P],
    "rtenhip_sample_f32": [_P, _P, _P, _P, _P, C.c_size_t, _P, _P],
}
_functions = {}

# A call's descriptors as bytes in the structures' layouts: packing one takes
# a third of filling a ctypes structure, and a step of a decoder makes hundreds
# of calls that the GPU is done with in a few microseconds each.
_ROWS = struct.Struct("Pi4x3q40x3q40x")
_MATRIX = struct.Struct("Pi4x2q48x2q48x")
_CACHE = struct.Struct("PPiiqii3q3q")
_SEQUENCES = struct.Struct("PqPPii")
_ROTARY = struct.Struct("PPPPfii4x")
_SAMPLING = struct.Struct("fffiPPPP")
_FLOAT_MAX = 3.4028234663852886e38


def _call(name, *args):
    f = _functions.get(name)
    if f is None:
        f = getattr(lib(), name)
        f.argtypes, f.restype = _SIGNATURES[name], C.c_int
        _functions[name] = f
    code = f(*args)
    if code:
        check(code)


def _on_device(t, ctx, dtype, what):
    if t.dtype != dtype:
        raise OpError(1, f"IncorrectInputType: expected {str(dtype)[6:]} {what}")
    if t.get_device() != ctx.device:
        raise OpError(1, f"{what} must be on the context's GPU")


def _rows(t, ctx, what):
    """rtenhip_tensor of a float32 [tokens, heads, head_dim] tensor."""
    _on_device(t, ctx, _torch().float32, what)
    shape = t.shape
    if len(shape) != 3:
        raise OpError(3, "Expected [tokens, heads, head_dim] inputs")
    return _ROWS.pack(t.data_ptr(), 3, *shape, *t.stride())


def _vector(t, n, ctx, dtype, what):
    """Address of a contiguous 1-D device tensor of n elements (None: NULL)."""
    if t is None:
        return 0
    _on_device(t, ctx, dtype, what)
    if t.shape != (n,):
        raise OpError(3, f"{what} must have {n} elements")
    if n > 1 and t.stride(0) != 1:
        raise OpError(6, f"{what} must be contiguous")
    return t.data_ptr()


def _cache(k, v, ctx):
    """rtenhip_kv_cache of two [pages, page size, heads, head_dim] tensors."""
    shape, dtype = k.shape, k.dtype
    if len(shape) != 4 or v.shape != shape:
        raise OpError(3, "Caches must be [pages, page size, heads, head_dim] of the same shape")
    kind = _cache_dtype(dtype)
    _on_device(k, ctx, dtype, "cache")
    _on_device(v, ctx, dtype, "cache")
    n, page, heads, dim = shape
    k0, k1, k2, k3 = k.stride()
    v0, v1, v2, v3 = v.stride()
    if dim > 1 and (k3 != 1 or v3 != 1):
        raise OpError(6, "Cache rows must have unit stride")
    if max(page, heads, dim) > 0x7fffffff:
        raise OpError(5, "Invalid cache size")
    return _CACHE.pack(k.data_ptr(), v.data_ptr(), kind, page, n, heads, dim, k0, k1, k2, v0, v1, v2)


_cache_dtypes = {}


def _cache_dtype(dtype):
    if not _cache_dtypes:
        torch = _torch()
        _cache_dtypes.update({torch.float32: 0, torch.float16: 1, torch.bfloat16: 2})
    kind = _cache_dtypes.get(dtype)
    if kind is None:
        raise OpError(1, "IncorrectInputType: cache must be float32, float16 or bfloat16")
    return kind


def _sequences(page_table, kv_lens, q_starts, ctx):
    """rtenhip_sequences."""
    i32 = _torch().int32
    _on_device(page_table, ctx, i32, "page_table")
    if page_table.dim() != 2:
        raise OpError(3, "page_table must be [sequences, pages]")
    n, pages = page_table.shape
    row, unit = page_table.stride()
    if pages > 1 and unit != 1:
        raise OpError(6, "page_table rows must have unit stride")
    return _SEQUENCES.pack(page_table.data_ptr(), row, _vector(kv_lens, n, ctx, i32, "kv_lens"),
                           _vector(q_starts, n + 1, ctx, i32, "q_starts"), n, pages)


def _context(ctx):
    """The context of a call and whether torch allocates on its stream: the
    default context follows torch's current stream."""
    if ctx is None:
        return default_context(), True
    torch = _torch()
    return ctx, ctx._raw_stream == torch._C._cuda_getCurrentRawStream(ctx.device)


def _empty(like, shape, dtype, ctx, here):
    """A tensor on like's device whose memory belongs to the context's stream,
    which is the one that the call writes it on."""
    if here:
        return like.new_empty(shape, dtype=dtype)
    with _torch().cuda.stream(ctx.stream):
        return like.new_empty(shape, dtype=dtype)


def _rotary(inv_freq, positions, tokens, dim, q_scale, k_scale, epsilon, interleaved, ctx):
    """rtenhip_rotary."""
    torch = _torch()
    f32 = torch.float32
    half = 0
    if inv_freq is not None:
        if inv_freq.dim() != 1:
            raise OpError(3, "inv_freq must be 1-D")
        half = inv_freq.shape[0]
        if half > 128:
            raise OpError(6, "rotary_dim must be a multiple of 8 up to head_dim")
    if _FLOAT_MAX < epsilon < math.inf:
        raise OpError(5, "epsilon must be a float32 number")
    return _ROTARY.pack(_vector(q_scale, dim, ctx, f32, "q_scale"), _vector(k_scale, dim, ctx, f32, "k_scale"),
                        _vector(inv_freq, half, ctx, f32, "inv_freq"),
                        _vector(positions, tokens, ctx, torch.int32, "positions"), epsilon, 2 * half,
                        1 if interleaved else 0)


def _int32(n):
    return max(-1, min(int(n), 0x7fffffff))


def _check_3d(*tensors):
    for t in tensors:
        if t.dim() != 3:
            raise OpError(3, "Expected [tokens, heads, head_dim] inputs")


def qk_norm_rotary(q, k, positions, inv_freq, q_scale=None, k_scale=None, epsilon=1e-6, interleaved=False, q_out=None,
                   k_out=None, ctx=None):
    """RMS norm over head_dim (where a scale ``[head_dim]`` is given), then the
    rotation by ``positions[t] * inv_freq[i]``, of the head rows of q
    ``[tokens, q heads, head_dim]`` and k ``[tokens, k heads, head_dim]``.
    ``inv_freq`` has rotary_dim / 2 values (None: no rotation); pairs are
    (i, i + rotary_dim / 2), or neighbours if ``interleaved``.  Returns
    (q_out, k_out); either may be given, its input itself included."""
    ctx, here = _context(ctx)
    _check_3d(q, k)
    r = _rotary(inv_freq, positions, q.shape[0], q.shape[2], q_scale, k_scale, epsilon, interleaved, ctx)
    if q_out is None:
        q_out = _empty(q, q.shape, q.dtype, ctx, here)
    if k_out is None:
        k_out = _empty(k, k.shape, k.dtype, ctx, here)
    _call("rtenhip_qk_norm_rotary_f32", ctx.ptr, _rows(q, ctx, "q"), _rows(k, ctx, "k"), r, _rows(q_out, ctx, "q_out"),
          _rows(k_out, ctx, "k_out"))
    return q_out, k_out


def qk_norm_rotary_append(q, k, v, inv_freq, k_cache, v_cache, page_table, kv_lens, q_starts=None, positions=None,
                          q_scale=None, k_scale=None, epsilon=1e-6, interleaved=False, out=None, ctx=None):
    """:func:`qk_norm_rotary` of the new tokens of the sequences, with k's rows
    and v written into the cache.  ``positions`` (default: the tokens' places
    in their sequences) turn the rows only.  Returns q's rows (``out``, which
    may be q); rows of padding in a new ``out`` are not initialised."""
    ctx, here = _context(ctx)
    _check_3d(q, k, v)
    r = _rotary(inv_freq, positions, q.shape[0], q.shape[2], q_scale, k_scale, epsilon, interleaved, ctx)
    cache = _cache(k_cache, v_cache, ctx)
    seqs = _sequences(page_table, kv_lens, q_starts, ctx)
    if out is None:
        out = _empty(q, q.shape, q.dtype, ctx, here)
    _call("rtenhip_qk_norm_rotary_append_f32", ctx.ptr, _rows(q, ctx, "q"), _rows(k, ctx, "k"), _rows(v, ctx, "v"), r,
          cache, seqs, _rows(out, ctx, "out"))
    return out


def paged_attention(q, k_cache, v_cache, page_table, kv_lens, q_starts=None, scale=None, window=0, sinks=0, out=None,
                    ctx=None):
    """softmax(scale q k^T) v of the new tokens' queries ``[tokens, q heads,
    head_dim]`` over their sequences' cached tokens; query head h reads cache
    head h // (q heads / cache heads).  The token at position p sees the tokens
    up to p; with a ``window``, the last ``window`` of them and the first
    ``sinks``.  ``scale`` defaults to 1 / sqrt(head_dim).  A row that sees
    nothing gives zeros; rows of padding in a new ``out`` are not initialised."""
    ctx, here = _context(ctx)
    cache = _cache(k_cache, v_cache, ctx)
    seqs = _sequences(page_table, kv_lens, q_starts, ctx)
    qd = _rows(q, ctx, "q")
    if out is None:
        out = _empty(q, q.shape, q.dtype, ctx, here)
    need = C.c_size_t()
    _call("rtenhip_paged_attention_workspace", qd, cache, seqs, C.byref(need))
    n = need.value
    ws = _empty(q, (n,), _torch().uint8, ctx, here) if n else None
    _call("rtenhip_paged_attention_f32", ctx.ptr, qd, cache, seqs, 1 / math.sqrt(q.shape[2]) if scale is None else scale,
          _int32(window), _int32(sinks), ws.data_ptr() if n else None, n, _rows(out, ctx, "out"))
    return out


@functools.lru_cache(maxsize=256)
def _sample_workspace(rows, vocab):
    """A size that depends on these two numbers alone."""
    need = C.c_size_t()
    _call("rtenhip_sample_workspace", rows, vocab, C.byref(need))
    return need.value


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, ctx=None):
    """One token of each row of ``logits [rows, vocab]`` by the random numbers
    ``uniforms [rows]`` in [0, 1); returns (tokens int32 [rows], logprobs
    float32 [rows]).  The filters (see rtenhip_sample_f32; ``top_k`` 0,
    ``top_p`` 1 and ``min_p`` 0 keep all, ``temperature`` 0 takes the largest)
    are numbers, or device tensors with one for each row."""
    torch = _torch()
    ctx, here = _context(ctx)
    f32, i32 = torch.float32, torch.int32
    _on_device(logits, ctx, f32, "logits")
    if logits.dim() != 2:
        raise OpError(3, "Expected [rows, vocab] logits")
    rows, vocab = logits.shape

    def per_row(value, none, dtype, what):
        """(The number for all rows, the address of those of each.)"""
        if isinstance(value, torch.Tensor):
            return none, _vector(value, rows, ctx, dtype, what)
        return value if dtype is i32 else C.c_float(value).value, 0  # (past its range: infinity)

    t, ts = per_row(temperature, 1., f32, "temperature")
    k, ks = per_row(top_k, 0, i32, "top_k")
    p, ps = per_row(top_p, 1., f32, "top_p")
    m, ms = per_row(min_p, 0., f32, "min_p")
    s = _SAMPLING.pack(t, p, m, min(max(int(k), 0), vocab), ts, ps, ms, ks)
    u = _vector(uniforms, rows, ctx, f32, "uniforms")
    need = _sample_workspace(rows, vocab)
    tokens, logprobs = _empty(logits, (rows,), i32, ctx, here), _empty(logits, (rows,), f32, ctx, here)
    ws = _empty(logits, (need,), torch.uint8, ctx, here)
    _call("rtenhip_sample_f32", ctx.ptr, _MATRIX.pack(logits.data_ptr(), 2, rows, vocab, *logits.stride()), s, u,
          ws.data_ptr(), need, tokens.data_ptr(), logprobs.data_ptr())
    return tokens, logprobs
