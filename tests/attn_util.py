"""Oracles of the attention operators: plain torch in 64 bits on the CPU, and random paged caches."""
import math

import torch

F = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


def half_step(dtype):
    """Largest relative rounding of a value to dtype."""
    return torch.finfo(dtype).eps / 2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype)


def table_of(g, lens, pt, spare=2, width=None):
    """A shuffled page table ([n_seqs, width] int32, -1 past each sequence's pages) and the pool's page count."""
    need = [-(-max(n, 0) // pt) for n in lens]
    total = sum(need) + spare
    perm = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.full((len(lens), max(1, max(need)) if width is None else width), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def pool(g, total, heads, pt, hd, cache, fill=float("nan")):
    """An empty pool: garbage everywhere (NaN, or for Q8 random codes under NaN scales)."""
    if cache == "q8":
        return (torch.randint(-127, 128, (total, heads, pt, hd), generator=g).to(torch.int8),
                torch.full((total, heads, pt, hd // 64), fill))
    return torch.full((total, heads, pt, hd), fill).to(F[cache]), None


def put(pl, scale, table, b, pos, pt, x):
    """Row x [heads, hd] (f64 values) at position pos of sequence b, as the cache holds it; the value it stands for."""
    page, slot = int(table[b, pos // pt]), pos % pt
    if scale is None:
        pl[page, :, slot] = x.to(pl.dtype)
        return pl[page, :, slot].double()
    code, d = quant(x.float())
    pl[page, :, slot], scale[page, :, slot] = code, d
    return (code.double().view(*d.shape, 64) * d.double()[..., None]).view(x.shape)


def quant(x):
    """The activation blocks' quantiser on f32 rows [..., n]: int8 codes and f32 scales of blocks of 64. A block
    with a NaN or an infinity has a NaN scale."""
    blk = x.reshape(*x.shape[:-1], -1, 64)
    amax = torch.nan_to_num(blk.abs(), nan=0.0, posinf=float("inf")).amax(-1)
    d = amax / 127.0
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    v = torch.nan_to_num(blk * inv[..., None], nan=0.0, posinf=float("inf"), neginf=float("-inf")).clamp(-127, 127)
    code = torch.round(v).to(torch.int8).view(x.shape)
    return code, torch.where(torch.isfinite(blk).all(-1), d, torch.full_like(d, float("nan")))


def dequant(code, d):
    return (code.double().reshape(*d.shape, 64) * d.double()[..., None]).reshape(code.shape)


def rotate(x, cos, sin, interleaved, off, rnd=lambda v: v):
    """x [T, H, hd] f64 with [off, off + 2 half) rotated by cos, sin [T, half]."""
    half = cos.shape[-1]
    y = x.clone()
    for j in range(half):
        ia, ib = (off + 2 * j, off + 2 * j + 1) if interleaved else (off + j, off + j + half)
        a, b, c, s = x[..., ia], x[..., ib], cos[:, None, j], sin[:, None, j]
        y[..., ia] = rnd(rnd(a * c) - rnd(b * s))
        y[..., ib] = rnd(rnd(b * c) + rnd(a * s))
    return y


def attend(q, k, v, scale):
    """q [H, D], k [n, Hkv, D], v [n, Hkv, Dv] in f64: out [H, Dv], lse [H], and what error bounds need: the
    probability-weighted |v| [H, Dv] and the largest scale * sum |q k| [H]."""
    H, n = q.shape[0], k.shape[0]
    if n == 0:
        return (torch.zeros(H, v.shape[-1], dtype=torch.float64), torch.full((H,), -math.inf, dtype=torch.float64),
                torch.zeros(H, v.shape[-1], dtype=torch.float64), torch.zeros(H, dtype=torch.float64))
    g = torch.arange(H) // (H // k.shape[1])
    kk, vv = k[:, g], v[:, g]
    s = torch.einsum("hd,nhd->hn", q, kk) * scale
    big = (torch.einsum("hd,nhd->hn", q.abs(), kk.abs()) * abs(scale)).amax(-1)
    lse = torch.logsumexp(s, -1)
    p = torch.exp(s - lse[:, None])
    return torch.einsum("hn,nhd->hd", p, vv), lse, torch.einsum("hn,nhd->hd", p, vv.abs()), big
