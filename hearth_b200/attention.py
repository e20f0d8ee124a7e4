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
enqueued on `stream` (default: torch's current stream of the tensors' device) without waiting; a wrong argument
raises ValueError before anything is enqueued.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import KvCache, Rope, check, lib
from .moe import _stream

_SCALINGS = {"none": 0, "linear": 1, "ntk": 2, "yarn": 3}


def _dtype(t, what):
    import torch
    d = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}.get(t.dtype)
    if d is None:
        raise ValueError(f"{what} must be float32, float16 or bfloat16, got {t.dtype}")
    return d


def _need(ok, msg):
    if not ok:
        raise ValueError(msg)


def _rows(t, what):
    """A [tokens, heads, dim] tensor's pointer and strides."""
    _need(t.dim() == 3, f"{what} must be [tokens, heads, dim], got {tuple(t.shape)}")
    _need(t.shape[2] < 2 or t.stride(2) == 1, f"{what}'s last dimension must be contiguous")
    return t.data_ptr(), t.stride(0), t.stride(1)


def _ints(t, what, n=None):
    import torch
    _need(t.dtype == torch.int32 and t.dim() == 1 and (t.numel() < 2 or t.stride(0) == 1),
          f"{what} must be a contiguous int32 vector")
    _need(n is None or t.numel() == n, f"{what} must have {n} values, got {t.numel()}")
    return t.data_ptr()


class _on:
    """The tensors' device as the current one, and the stream to use there."""

    def __init__(self, stream, *tensors):
        import torch
        dev = tensors[0].device
        for t in tensors:
            if t is not None:
                _need(t.is_cuda, "tensors must be on a CUDA device")
                _need(t.device == dev, "tensors must be on one device")
        self.guard = None if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)
        self.dev, self.user = dev, stream

    def __enter__(self):
        import torch
        if self.guard is not None:
            self.guard.__enter__()
        return _stream(torch.cuda.current_stream(self.dev) if self.user is None else self.user)

    def __exit__(self, *a):
        if self.guard is not None:
            self.guard.__exit__(*a)

    def scratch(self, n):
        """n bytes for work on the call's stream."""
        import torch
        t = torch.empty(n, dtype=torch.uint8, device=self.dev)
        if self.user is not None:
            s = self.user if hasattr(self.user, "cuda_stream") else torch.cuda.ExternalStream(int(self.user), self.dev)
            t.record_stream(s)
        return t


def _call(name, *args):
    rc = getattr(lib(), name)(*args)
    if rc in (_lib.HXB_E_ARG, _lib.HXB_E_UNSUPPORTED):
        raise ValueError(f"{name}: {_lib.last_error()}")
    check(rc, name)


def _cache(k, v, table, k_scale, v_scale):
    import torch
    _need(k.dim() == 4 and k.is_contiguous(), "k_cache must be contiguous [pages, heads, page_tokens, dim]")
    n_pages, heads, pt, hd = k.shape
    dt = {torch.float16: _lib.F16, torch.bfloat16: _lib.BF16, torch.int8: _lib.Q8}.get(k.dtype)
    _need(dt is not None, f"a cache is float16, bfloat16 or int8, got {k.dtype}")
    _need(v is None or (v.dtype == k.dtype and v.shape == k.shape and v.is_contiguous()), "v_cache must be like k_cache")
    for s, p, what in ((k_scale, k, "k_scale"), (v_scale, v, "v_scale")):
        if p is None or dt != _lib.Q8:
            _need(s is None, f"{what} goes with an int8 cache")
        else:
            _need(s is not None and s.dtype == torch.float32 and s.is_contiguous()
                  and s.shape == (n_pages, heads, pt, hd // 64), f"{what} must be float32 [pages, heads, page_tokens, dim / 64]")
    _need(table.dtype == torch.int32 and table.dim() == 2, "table must be int32 [sequences, pages]")
    B, P = table.shape
    _need(P < 2 or table.stride(1) == 1, "table rows must be contiguous")
    ptr = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    return KvCache(dt, heads, hd, pt, n_pages, ptr(k), ptr(v), ptr(k_scale), ptr(v_scale), ptr(table),
                   table.stride(0) if B > 1 else P, P, B)


def _rope(cs, interleaved, offset):
    import torch
    _need(cs.dtype == torch.float32 and cs.dim() == 3 and cs.shape[2] == 2 and cs.is_contiguous(),
          "cs must be a contiguous float32 [positions, rope_dim / 2, 2] table")
    return Rope(cs.data_ptr(), cs.shape[0], 2 * cs.shape[1], offset, int(bool(interleaved)))


def rope_freqs(rope_dim: int, theta: float, *, scaling: str = "none", factor: float = 1.0, original: int = 4096,
               beta_fast: float = 32.0, beta_slow: float = 1.0) -> tuple[np.ndarray, float]:
    """Frequencies (float64 [rope_dim / 2]) and the factor for the table's values; scaling "none", "linear",
    "ntk" or "yarn" (hxb_rope_freqs)."""
    _need(scaling in _SCALINGS, f"scaling must be one of {sorted(_SCALINGS)}, got {scaling!r}")
    _need(2 <= rope_dim <= 1024 and rope_dim % 2 == 0, f"rope_dim must be even, 2 to 1024, got {rope_dim}")
    f, a = np.empty(rope_dim // 2, np.float64), C.c_double()
    _call("hxb_rope_freqs", rope_dim, theta, _SCALINGS[scaling], factor, original, beta_fast, beta_slow, f.ctypes.data,
          C.byref(a))
    return f, a.value


def rope_table(freqs, n_pos: int, *, first: int = 0, factor: float = 1.0, out=None, device=None, stream=None):
    """cs [n_pos, rope_dim / 2, 2] float32: factor * (cos, sin) of positions first .. first + n_pos - 1."""
    import torch
    f = np.ascontiguousarray(freqs, np.float64)
    _need(f.ndim == 1 and f.size >= 1, "freqs must be a vector")
    _need(n_pos >= 0, "n_pos must not be negative")
    if out is None:
        out = torch.empty((n_pos, f.size, 2), dtype=torch.float32, device="cuda" if device is None else device)
        if stream is not None and hasattr(stream, "cuda_stream"):
            out.record_stream(stream)
    _need(out.dtype == torch.float32 and out.shape == (n_pos, f.size, 2) and out.is_contiguous(),
          "out must be a contiguous float32 [n_pos, len(freqs), 2] tensor")
    with _on(stream, out) as s:
        _call("hxb_rope_table_dev", f.ctypes.data, 2 * f.size, factor, first, n_pos, out.data_ptr(), s)
    return out


def rope(x, pos, cs, *, interleaved: bool = False, offset: int = 0, out=None, stream=None):
    """x [T, heads, dim] with values [offset, offset + rope_dim) of every head rotated by position pos[t] (int32
    [T]); into out (another element type is rounded to; x itself: in place), or a new tensor like x."""
    import torch
    xa = _rows(x, "x")
    T, H, D = x.shape
    r, p = _rope(cs, interleaved, offset), _ints(pos, "pos", T)
    if out is None:
        out = torch.empty((T, H, D), dtype=x.dtype, device=x.device)
    ya = _rows(out, "out")
    _need(out.shape == x.shape, "out must have x's shape")
    dx, dy = _dtype(x, "x"), _dtype(out, "out")
    with _on(stream, x, pos, cs, out) as s:
        _call("hxb_rope_dev", C.byref(r), p, T, H, D, xa[0], dx, xa[1], xa[2], ya[0], dy, ya[1], ya[2], s)
    return out


def _kv_args(k, v, cache, v_cache, start, pos0, what):
    ka = _rows(k, what)
    _need(k.shape[1:] == (cache.n_kv_heads, cache.head_dim), f"{what} must be [tokens, {cache.n_kv_heads}, {cache.head_dim}]")
    _need((v is None) == (v_cache is None), "v goes with a v_cache")
    va = (0, 0, 0)
    if v is not None:
        va = _rows(v, "v")
        _need(v.shape == k.shape and v.dtype == k.dtype, "v must be like k")
    return (_ints(start, "start", cache.n_seqs + 1), _ints(pos0, "pos0", cache.n_seqs), k.shape[0], *ka, *va,
            _dtype(k, what))


def kv_write(k, v, k_cache, v_cache, table, start, pos0, *, k_scale=None, v_scale=None, cs=None,
             interleaved: bool = False, offset: int = 0, stream=None) -> None:
    """Rows start[b] .. start[b + 1] - 1 of k and v [T, n_kv_heads, head_dim] become positions pos0[b], pos0[b] + 1,
    ... of sequence b; rows outside are padding. cs: the keys are rotated by their positions first. v and v_cache
    None: a latent cache. (hxb_kv_write_dev)"""
    c = _cache(k_cache, v_cache, table, k_scale, v_scale)
    args = _kv_args(k, v, c, v_cache, start, pos0, "k")
    r = None if cs is None else C.byref(_rope(cs, interleaved, offset))
    with _on(stream, k, v, k_cache, v_cache, table, start, pos0, k_scale, v_scale, cs) as s:
        _call("hxb_kv_write_dev", C.byref(c), *args, r, s)


def kv_read(k_cache, v_cache, table, start, pos0, k_out, v_out, *, k_scale=None, v_scale=None, stream=None) -> None:
    """The rows kv_write wrote, back into k_out and v_out [T, n_kv_heads, head_dim] of any element type; padding
    rows keep what they hold. (hxb_kv_read_dev)"""
    c = _cache(k_cache, v_cache, table, k_scale, v_scale)
    args = _kv_args(k_out, v_out, c, v_cache, start, pos0, "k_out")
    with _on(stream, k_out, v_out, k_cache, v_cache, table, start, pos0, k_scale, v_scale) as s:
        _call("hxb_kv_read_dev", C.byref(c), *args, s)


def _workspace(on, given, n):
    import torch
    if given is None:
        return on.scratch(n)
    _need(given.dtype == torch.uint8 and given.is_contiguous() and given.numel() >= n,
          f"workspace must be a contiguous uint8 tensor of at least {n} bytes")
    return given


def decode_attention(q, k_cache, v_cache, table, lens, *, scale: float, k_scale=None, v_scale=None, out=None,
                     return_lse: bool = False, lse=None, workspace=None, stream=None):
    """Attention of one new token a sequence, q [n_seqs, heads, head_dim], over positions 0 .. lens[b] - 1 of its
    pages; out like q, with return_lse (out, lse [n_seqs, heads] float32). A sequence of length 0 gives zeros
    and -inf. workspace: uint8 scratch of attention_workspace bytes that no other call in flight uses
    (default: torch's allocator). (hxb_attn_decode_dev)"""
    import torch
    c = _cache(k_cache, v_cache, table, k_scale, v_scale)
    _need(v_cache is not None, "decode_attention needs a v_cache (latent_attention reads a latent cache)")
    qa = _rows(q, "q")
    B, H, D = q.shape
    _need((B, D) == (c.n_seqs, c.head_dim), f"q must be [{c.n_seqs}, heads, {c.head_dim}], got {tuple(q.shape)}")
    lp, dt = _ints(lens, "lens", B), _dtype(q, "q")
    if out is None:
        out = torch.empty((B, H, D), dtype=q.dtype, device=q.device)
    oa = _rows(out, "out")
    _need(out.shape == q.shape and out.dtype == q.dtype, "out must be like q")
    if lse is None and return_lse:
        lse = torch.empty((B, H), dtype=torch.float32, device=q.device)
    _need(lse is None or (lse.dtype == torch.float32 and lse.shape == (B, H) and lse.is_contiguous()),
          "lse must be a contiguous float32 [n_seqs, heads] tensor")
    on = _on(stream, q, k_cache, v_cache, table, lens, k_scale, v_scale, out, lse, workspace)
    with on as s:
        n = int(lib().hxb_attn_decode_workspace(C.byref(c), H))
        ws = _workspace(on, workspace, n)
        _call("hxb_attn_decode_dev", C.byref(c), lp, *qa, H, dt, scale, *oa, 0 if lse is None else lse.data_ptr(),
              ws.data_ptr(), ws.numel(), s)
    return (out, lse) if return_lse else out


def latent_attention(q, w, c_cache, table, lens, *, scale: float, c_scale=None, out=None, workspace=None, stream=None):
    """Absorbed latent attention of one new token a sequence over a latent cache [n_pages, 1, page_tokens, rank +
    rope]: q [n_seqs, heads, nope + rope] (its rope part rotated), w [heads, nope + v_dim, rank] (the latent's
    expansion to each head's key and value); out [n_seqs, heads, v_dim]. (hxb_latent_decode_dev)"""
    import torch
    c = _cache(c_cache, None, table, c_scale, None)
    qa = _rows(q, "q")
    B, H, dq = q.shape
    _need(w.dim() == 3 and w.is_contiguous() and w.dtype == q.dtype and w.shape[0] == H,
          f"w must be contiguous [{H}, nope + v_dim, rank] in q's type")
    R = w.shape[2]
    nope = dq - (c.head_dim - R)
    vd = w.shape[1] - nope
    _need(B == c.n_seqs and 0 < nope < w.shape[1], f"q {tuple(q.shape)}, w {tuple(w.shape)} and rows of {c.head_dim} do not fit together")
    lp, dt = _ints(lens, "lens", B), _dtype(q, "q")
    if out is None:
        out = torch.empty((B, H, vd), dtype=q.dtype, device=q.device)
    oa = _rows(out, "out")
    _need(out.shape == (B, H, vd) and out.dtype == q.dtype, f"out must be [{B}, {H}, {vd}] in q's type")
    on = _on(stream, q, w, c_cache, table, lens, c_scale, out, workspace)
    with on as s:
        n = int(lib().hxb_latent_decode_workspace(C.byref(c), H, R))
        ws = _workspace(on, workspace, n)
        _call("hxb_latent_decode_dev", C.byref(c), lp, *qa, w.data_ptr(), H, R, nope, vd, dt, scale, *oa,
              ws.data_ptr(), ws.numel(), s)
    return out
