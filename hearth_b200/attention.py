"""Attention operators on torch CUDA tensors (hxb_rope_*, hxb_kv_*, hxb_attn_decode_dev,
hxb_latent_decode_dev of include/hearth_b200.h): rotary positions, a paged key-value cache and attention of
one new token a sequence over it, for programs that keep their own decoder around these kernels.

    freqs, factor = rope_freqs(128, 1e6, scaling="yarn", factor=4.0, original=32768)
    cs = rope_table(freqs, n_pos, factor=factor)                   # once
    q = rope(q, pos, cs)                                           # [T, H, 128]
    kv_write(k, v, k_cache, v_cache, table, start, pos0, cs=cs)    # keys rotated as they are written
    out = decode_attention(q, k_cache, v_cache, table, lens, scale=128 ** -0.5)

Caches are plain tensors: k_cache, v_cache [n_pages, n_kv_heads, page_tokens, head_dim] in float16, bfloat16 or,
quantised in blocks of 64, int8 with k_scale, v_scale [n_pages, n_kv_heads, page_tokens, head_dim / 64] float32.
table [n_seqs, max_pages] int32 names the pages of each sequence (an expanded row is one table for all). Work is
enqueued on `stream` (default: torch's current stream of the tensors' device) without waiting, and what a call allocates
(outputs that are not given, scratch) belongs to that stream; tensors passed in have to live until the stream is done with
them. A wrong argument raises ValueError before anything is enqueued. The calls are made for inference: autograd does not see them,
and what they return has no graph, whatever their arguments require.
"""
from __future__ import annotations

import ctypes as C
import functools

import numpy as np

from . import _lib
from ._lib import KvCache, Rope, check, lib
from .moe import _CUDA_STREAM_LEGACY, _stream

_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}


@functools.lru_cache(None)
def _torch():
    """torch (imported with the first call), its element types as the library's, and a device's current stream."""
    import torch
    io = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
    cache = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.int8: _lib.Q8}
    raw = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda i: torch.cuda.current_stream(i).cuda_stream)
    return torch, io, cache, raw


def _bad(msg):
    raise ValueError(msg)


def _rows(t, what):
    """Pointer, strides and shape of a [tokens, heads, dim] tensor."""
    shape = t.shape
    if len(shape) != 3:
        _bad(f"{what} must be [tokens, heads, dim], got {tuple(shape)}")
    s0, s1, s2 = t.stride()
    if s2 != 1 and shape[2] > 1:
        _bad(f"{what}'s last dimension must be contiguous")
    return t.data_ptr(), s0, s1, shape


def _ints(t, what, n):
    if t.dtype != _torch()[0].int32 or t.dim() != 1 or (t.stride(0) != 1 and t.numel() > 1):
        _bad(f"{what} must be a contiguous int32 vector")
    if t.numel() != n:
        _bad(f"{what} must have {n} values, got {t.numel()}")
    return t.data_ptr()


class _on:
    """The tensors' device as the current one, and the stream to use there (`ptr` inside the with block)."""
    __slots__ = ("guard", "dev", "user", "ptr")

    def __init__(self, stream, *tensors):
        cuda = _torch()[0].cuda
        dev = tensors[0].device
        if dev.type != "cuda":
            _bad("tensors must be on a CUDA device")
        for t in tensors:
            if t is not None and t.device != dev:
                _bad("tensors must be on one CUDA device")
        if getattr(stream, "device", dev) != dev:
            _bad(f"stream is on {stream.device}, the tensors are on {dev}")
        self.guard = None if cuda.current_device() == dev.index else cuda.device(dev)
        self.dev, self.user = dev, stream
        self.ptr = (_torch()[3](dev.index) or _CUDA_STREAM_LEGACY) if stream is None else _stream(stream)

    def __enter__(self):
        if self.guard is not None:
            self.guard.__enter__()
        return self.ptr

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)

    def new(self, like, shape, dtype):
        """A new contiguous tensor beside `like`, in the memory of the call's stream."""
        cuda = _torch()[0].cuda
        if self.user is not None:
            with cuda.stream(self.user if hasattr(self.user, "cuda_stream") else cuda.ExternalStream(int(self.user), self.dev)):
                return like.new_empty(shape, dtype=dtype)
        if like.dtype == dtype and like.shape == shape and like.is_contiguous():
            return _torch()[0].empty_like(like)
        return like.new_empty(shape, dtype=dtype)

    def scratch(self, like, given, n):
        """n bytes for work on the call's stream."""
        uint8 = _torch()[0].uint8
        if given is None:
            return self.new(like, (n,), uint8)
        if given.dtype != uint8 or not given.is_contiguous() or given.numel() < n:
            _bad(f"workspace must be a contiguous uint8 tensor of at least {n} bytes")
        return given


def _done(rc, name):
    if rc:
        if rc in (_lib.HXB_E_ARG, _lib.HXB_E_UNSUPPORTED):
            _bad(f"{name}: {_lib.last_error()}")
        check(rc, name)


def _scales(dt, k, s, what):
    if k is None or dt != _lib.Q8:
        if s is not None:
            _bad(f"{what} goes with an int8 cache")
        return 0
    want = (*k.shape[:3], k.shape[3] // 64)
    if s is None or s.dtype != _torch()[0].float32 or s.shape != want or not s.is_contiguous():
        _bad(f"{what} must be float32 [pages, heads, page_tokens, dim / 64]")
    return s.data_ptr()


def _cache(k, v, table, k_scale, v_scale):
    torch, _, types, _ = _torch()
    shape = k.shape
    if len(shape) != 4 or not k.is_contiguous():
        _bad("k_cache must be contiguous [pages, heads, page_tokens, dim]")
    dt = types.get(k.dtype)
    if dt is None:
        _bad(f"a cache is float16, bfloat16 or int8, got {k.dtype}")
    if v is not None and (v.dtype != k.dtype or v.shape != shape or not v.is_contiguous()):
        _bad("v_cache must be like k_cache")
    ks, vs = _scales(dt, k, k_scale, "k_scale"), _scales(dt, v, v_scale, "v_scale")
    if table.dtype != torch.int32 or table.dim() != 2:
        _bad("table must be int32 [sequences, pages]")
    B, P = table.shape
    s0, s1 = table.stride()
    if s1 != 1 and P > 1:
        _bad("table rows must be contiguous")
    return KvCache(dt, shape[1], shape[3], shape[2], shape[0], k.data_ptr(), 0 if v is None else v.data_ptr(), ks, vs, table.data_ptr(),
                   s0 if B > 1 else P, P, B)


def _rope(cs, interleaved, offset):
    if cs.dtype != _torch()[0].float32 or cs.dim() != 3 or cs.shape[2] != 2 or not cs.is_contiguous():
        _bad("cs must be a contiguous float32 [positions, rope_dim / 2, 2] table")
    if not 0 <= offset < 1 << 31:      # C's int would wrap
        _bad(f"offset must not be negative or past a head, got {offset}")
    return Rope(cs.data_ptr(), cs.shape[0], 2 * cs.shape[1], offset, int(bool(interleaved)))


def _io(t, what):
    d = _torch()[1].get(t.dtype)
    if d is None:
        _bad(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return d


def rope_freqs(rope_dim: int, theta: float, *, scaling: str = "none", factor: float = 1.0, original: int = 4096,
               beta_fast: float = 32.0, beta_slow: float = 1.0) -> tuple[np.ndarray, float]:
    """Frequencies (float64 [rope_dim / 2]) and the factor for the table's values; scaling "none", "linear",
    "ntk" or "yarn" (hxb_rope_freqs)."""
    if scaling not in _SCALINGS:
        _bad(f"scaling must be one of {sorted(_SCALINGS)}, got {scaling!r}")
    if not 2 <= rope_dim <= 1024 or rope_dim % 2:
        _bad(f"rope_dim must be even, 2 to 1024, got {rope_dim}")
    if not -1 << 31 <= original < 1 << 31:      # C's int would wrap
        _bad(f"original must be a count of positions, got {original}")
    f, a = np.empty(rope_dim // 2, np.float64), C.c_double()
    _done(lib().hxb_rope_freqs(rope_dim, theta, _SCALINGS[scaling], factor, original, beta_fast, beta_slow, f.ctypes.data,
                               C.byref(a)), "hxb_rope_freqs")
    return f, a.value


def rope_table(freqs, n_pos: int, *, first: int = 0, factor: float = 1.0, out=None, device=None, stream=None):
    """cs [n_pos, rope_dim / 2, 2] float32: factor * (cos, sin) of positions first .. first + n_pos - 1."""
    torch = _torch()[0]
    f = np.ascontiguousarray(freqs, np.float64)
    if f.ndim != 1 or f.size < 1:
        _bad("freqs must be a vector")
    if n_pos < 0:
        _bad("n_pos must not be negative")
    if not -1 << 31 < first < 1 << 31 or n_pos > (1 << 31) - max(first, 0):
        _bad(f"positions must lie below 2^31, got {n_pos} from {first} on")
    if out is None:
        if device is None:
            device = stream.device if hasattr(stream, "device") else "cuda"
        beside = torch.empty(0, dtype=torch.float32, device=device)
        out = _on(stream, beside).new(beside, (n_pos, f.size, 2), torch.float32)
    if out.dtype != torch.float32 or out.shape != (n_pos, f.size, 2) or not out.is_contiguous():
        _bad("out must be a contiguous float32 [n_pos, len(freqs), 2] tensor")
    with _on(stream, out) as s:
        _done(lib().hxb_rope_table_dev(f.ctypes.data, 2 * f.size, factor, first, n_pos, out.data_ptr(), s), "hxb_rope_table_dev")
    return out


def rope(x, pos, cs, *, interleaved: bool = False, offset: int = 0, out=None, stream=None):
    """x [T, heads, dim] with values [offset, offset + rope_dim) of every head rotated by position pos[t] (int32
    [T]); into out (another element type is rounded to; x itself: in place), or a new tensor like x."""
    xp, xs, xh, shape = _rows(x, "x")
    T, H, D = shape
    r, p = _rope(cs, interleaved, offset), _ints(pos, "pos", T)
    on = _on(stream, x, pos, cs, out)
    if out is None:
        out = on.new(x, shape, x.dtype)
    yp, ys, yh, yshape = _rows(out, "out")
    if yshape != shape:
        _bad("out must have x's shape")
    dx, dy = _io(x, "x"), _io(out, "out")
    with on as s:
        _done(lib().hxb_rope_dev(C.byref(r), p, T, H, D, xp, dx, xs, xh, yp, dy, ys, yh, s), "hxb_rope_dev")
    return out


def _kv_args(k, v, cache, v_cache, start, pos0, what):
    kp, ks, kh, shape = _rows(k, what)
    if shape[1] != cache.n_kv_heads or shape[2] != cache.head_dim:
        _bad(f"{what} must be [tokens, {cache.n_kv_heads}, {cache.head_dim}]")
    if (v is None) != (v_cache is None):
        _bad("v goes with a v_cache")
    vp = vs = vh = 0
    if v is not None:
        vp, vs, vh, vshape = _rows(v, "v")
        if vshape != shape or v.dtype != k.dtype:
            _bad("v must be like k")
    B = cache.n_seqs
    return _ints(start, "start", B + 1), _ints(pos0, "pos0", B), shape[0], kp, ks, kh, vp, vs, vh, _io(k, what)


def kv_write(k, v, k_cache, v_cache, table, start, pos0, *, k_scale=None, v_scale=None, cs=None,
             interleaved: bool = False, offset: int = 0, stream=None) -> None:
    """Rows start[b] .. start[b + 1] - 1 of k and v [T, n_kv_heads, head_dim] become positions pos0[b], pos0[b] + 1,
    ... of sequence b; rows outside are padding. cs: the keys are rotated by their positions first. v and v_cache
    None: a latent cache. (hxb_kv_write_dev)"""
    c = _cache(k_cache, v_cache, table, k_scale, v_scale)
    args = _kv_args(k, v, c, v_cache, start, pos0, "k")
    r = None if cs is None else C.byref(_rope(cs, interleaved, offset))
    with _on(stream, k, v, k_cache, v_cache, table, start, pos0, k_scale, v_scale, cs) as s:
        _done(lib().hxb_kv_write_dev(C.byref(c), *args, r, s), "hxb_kv_write_dev")


def kv_read(k_cache, v_cache, table, start, pos0, k_out, v_out, *, k_scale=None, v_scale=None, stream=None) -> None:
    """The rows kv_write wrote, back into k_out and v_out [T, n_kv_heads, head_dim] of any element type; padding
    rows keep what they hold. (hxb_kv_read_dev)"""
    c = _cache(k_cache, v_cache, table, k_scale, v_scale)
    args = _kv_args(k_out, v_out, c, v_cache, start, pos0, "k_out")
    with _on(stream, k_out, v_out, k_cache, v_cache, table, start, pos0, k_scale, v_scale) as s:
        _done(lib().hxb_kv_read_dev(C.byref(c), *args, s), "hxb_kv_read_dev")


@functools.lru_cache(1024)
def _workspace(n_seqs, n_kv_heads, head_dim, heads, rank):
    c = KvCache(_lib.BF16, n_kv_heads, head_dim, 1, 0, 0, 0, 0, 0, 0, 0, 0, n_seqs)
    return int(lib().hxb_latent_decode_workspace(C.byref(c), heads, rank) if rank else lib().hxb_attn_decode_workspace(C.byref(c), heads))


def attention_workspace(n_seqs: int, heads: int, n_kv_heads: int, head_dim: int) -> int:
    """Bytes of scratch decode_attention needs for these sizes, whatever the cache's type and length
    (hxb_attn_decode_workspace)."""
    return _workspace(n_seqs, n_kv_heads, head_dim, heads, 0)


def latent_workspace(n_seqs: int, heads: int, rank: int, rope_dim: int) -> int:
    """Bytes of scratch latent_attention needs for these sizes (hxb_latent_decode_workspace)."""
    return _workspace(n_seqs, 1, rank + rope_dim, heads, rank)


def decode_attention(q, k_cache, v_cache, table, lens, *, scale: float, k_scale=None, v_scale=None, out=None,
                     return_lse: bool = False, lse=None, workspace=None, stream=None):
    """Attention of one new token a sequence, q [n_seqs, heads, head_dim], over positions 0 .. lens[b] - 1 of its
    pages; out like q, with return_lse (out, lse [n_seqs, heads] float32). A sequence of length 0 gives zeros
    and -inf. workspace: uint8 scratch of attention_workspace bytes that no other call in flight uses
    (default: from torch's allocator). (hxb_attn_decode_dev)"""
    c = _cache(k_cache, v_cache, table, k_scale, v_scale)
    if v_cache is None:
        _bad("decode_attention needs a v_cache (latent_attention reads a latent cache)")
    qp, qs, qh, shape = _rows(q, "q")
    B, H, D = shape
    if B != c.n_seqs or D != c.head_dim:
        _bad(f"q must be [{c.n_seqs}, heads, {c.head_dim}], got {tuple(shape)}")
    lp, dt = _ints(lens, "lens", B), _io(q, "q")
    torch = _torch()[0]
    on = _on(stream, q, k_cache, v_cache, table, lens, k_scale, v_scale, out, lse, workspace)
    if out is None:
        out = on.new(q, shape, q.dtype)
    op, os, oh, oshape = _rows(out, "out")
    if oshape != shape or out.dtype != q.dtype:
        _bad("out must be like q")
    if lse is None and return_lse:
        lse = on.new(q, (B, H), torch.float32)
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (B, H) or not lse.is_contiguous()):
        _bad("lse must be a contiguous float32 [n_seqs, heads] tensor")
    with on as s:
        ws = on.scratch(q, workspace, _workspace(B, c.n_kv_heads, D, H, 0))
        _done(lib().hxb_attn_decode_dev(C.byref(c), lp, qp, qs, qh, H, dt, scale, op, os, oh, None if lse is None else lse.data_ptr(),
                                        ws.data_ptr(), ws.numel(), s), "hxb_attn_decode_dev")
    return (out, lse) if return_lse else out


def latent_attention(q, w, c_cache, table, lens, *, scale: float, c_scale=None, out=None, workspace=None, stream=None):
    """Absorbed latent attention of one new token a sequence over a latent cache [n_pages, 1, page_tokens, rank +
    rope]: q [n_seqs, heads, nope + rope] (its rope part rotated), w [heads, nope + v_dim, rank] (the latent's
    expansion to each head's key and value); out [n_seqs, heads, v_dim]. workspace: uint8 scratch of latent_workspace
    bytes, as for decode_attention. (hxb_latent_decode_dev)"""
    c = _cache(c_cache, None, table, c_scale, None)
    qp, qs, qh, shape = _rows(q, "q")
    B, H, dq = shape
    if w.dim() != 3 or not w.is_contiguous() or w.dtype != q.dtype or w.shape[0] != H:
        _bad(f"w must be contiguous [{H}, nope + v_dim, rank] in q's type")
    R = w.shape[2]
    nope = dq - (c.head_dim - R)
    vd = w.shape[1] - nope
    if B != c.n_seqs or nope <= 0 or vd <= 0:
        _bad(f"q {tuple(shape)}, w {tuple(w.shape)} and rows of {c.head_dim} do not fit together")
    lp, dt = _ints(lens, "lens", B), _io(q, "q")
    on = _on(stream, q, w, c_cache, table, lens, c_scale, out, workspace)
    if out is None:
        out = on.new(q, (B, H, vd), q.dtype)
    op, os, oh, oshape = _rows(out, "out")
    if oshape != (B, H, vd) or out.dtype != q.dtype:
        _bad(f"out must be [{B}, {H}, {vd}] in q's type")
    with on as s:
        ws = on.scratch(q, workspace, _workspace(B, 1, c.head_dim, H, R))
        _done(lib().hxb_latent_decode_dev(C.byref(c), lp, qp, qs, qh, w.data_ptr(), H, R, nope, vd, dt, scale, op, os, oh,
                                          ws.data_ptr(), ws.numel(), s), "hxb_latent_decode_dev")
    return out
