"""What the attention operators' entry points promise, on the GPU: the quantiser's rule in every form of it, the bits that
weights and rows carry into the matrix products, far rotary positions, and batches with sequences that cannot be read.

Bounds are those of tests/test_gpu_attention.py with, for a weight, what the kernels carry of it: u is half a step of an
element type; two bf16 terms leave 2^-16 of a value (each 2^-8), three 2^-24, two f16 terms 2^-22, one f16 term 2^-11."""
import math
from fractions import Fraction

import numpy as np
import pytest
import torch

import hearth_b200 as hb
from tests.attn_util import F, attend, gen, half_step, put, pool, randn, table_of
from tests.test_gpu_attention import cu, filled

gpu_only = pytest.mark.gpu
W = 2.0 ** -24


def carried(cache, x):
    """What a decode weight loses as the matrix operands the kernel carries it in."""
    if cache == "bf16":
        return half_step(torch.bfloat16) ** (3 if x == "f32" else 2)
    return half_step(torch.float16) ** 2


def check_out(got, want, vabs, big, n, x, up, D):
    """An attention output's bound. Below 2^-14 the values of f16 are 2^-24 apart, so that rounding to it is off by up to 2^-25
    whatever the value's own size."""
    ds = (D + 16) * W * big[:, None]
    tol = half_step(F[x]) * want.abs() + (2.0 ** -25 if x == "f16" else 1e-30) + (2 * ds + up + 2.0 ** -21 + n * W) * vabs
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()


# ----------------------------------------------------------------------------------------- the quantiser's rule

@gpu_only
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rot", [0, 64])
def test_cache_rows_equal_their_plain_form(gpu, x, rot):
    """Rows of every type through a Q8 cache and back as f32: the calls' outputs, those of the plain form that the operators are
    measured against, and the rule in 64 bits are equal bit for bit (rows of few bits land on half a code often)."""
    from perf import operators as P
    case = dict(op="kv", B=3, n_new=700, Hkv=2, D=128, pt=16, cache="q8", x=x, y="f32", rot=rot, off=0, inter=False, past=40, latent=False)
    want = [t.float() for t in P.exact(case, 5)]
    try:
        for own in (False, True):
            P.own = own
            for got, ref in zip(P.run(P.prepare(case, 5)), want):
                assert torch.equal(got, ref), (own, (got != ref).sum())
    finally:
        P.own = False


# ----------------------------------------------------------------------------------------- the bits of the products

def check_lse(got, want, big, n, D):
    assert ((got.double() - want).abs() <= (D + 16) * W * big + 2.0 ** -20 + n * W + 2 * W * want.abs()).all(), (got.double() - want).abs().max()


@gpu_only
@pytest.mark.parametrize("x", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("H,Hkv", [(8, 1), (4, 4), (32, 2)])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_q8_keys_with_a_large_channel(gpu, x, H, Hkv, D):
    """One large key and value channel a block, which sets the block's scale, so that the other codes are 0 to 2; queries of one
    sign and scores of 20 to 50, whose terms hold no cancellation: the sums may lose a few f32 roundings of them."""
    g = gen(70)
    n, pt = 200, 16
    table, total = table_of(g, [n], pt)
    (kp, ks), (vp, vs) = (pool(g, total, Hkv, pt, D, "q8") for _ in range(2))
    step = 1.0 / 16
    k, v = ((torch.randint(0, 3, (n, Hkv, D), generator=g) * step).double() for _ in range(2))
    k[:, :, 5::64] = v[:, :, 17::64] = 127 * step
    krows, vrows = (torch.stack([put(p, s, table, 0, i, pt, r[i]) for i in range(n)]) for p, s, r in ((kp, ks, k), (vp, vs, v)))
    q = (0.5 + torch.rand((1, H, D), generator=g)).to(F[x])
    q[..., 5::64] = 0.01
    scale = 32.0 / (D * step)
    out, lse = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), scale=scale,
                                   k_scale=ks.cuda(), v_scale=vs.cuda(), return_lse=True)
    want, wl, vabs, big = attend(q[0].double(), krows, vrows, scale)
    assert 20 < big.min() and big.max() < 50
    check_lse(lse[0].cpu(), wl, big, n, D)
    check_out(out[0].cpu(), want, vabs, big, n, x, carried("q8", x), D)


T_OPPOSITE = [s * 2.0 ** -e for e in range(12) for s in (1.0, 1.25, 1.625)]      # exact in every type


def opposite_rows(g, D, cache):
    """Two positions with opposite values, and keys that are one value each: out = tanh(t) v, where nothing of the weights' own
    size is left, so that what a weight loses shows."""
    table, total = table_of(g, [2], 16)
    (kp, ks), (vp, vs) = (pool(g, total, 1, 16, D, cache) for _ in range(2))
    k = torch.zeros(1, D, dtype=torch.float64)
    k[0, 0] = 1.0
    v = randn(g, 1, D).double()
    krows, vrows = (torch.stack([put(p, s, table, 0, i, 16, r * (1 - 2 * i)) for i in range(2)]) for p, s, r in ((kp, ks, k), (vp, vs, v)))
    return kp, ks, vp, vs, table, krows, vrows


@gpu_only
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
def test_decode_weights_carry_their_terms(gpu, cache, x):
    D, B = 64, len(T_OPPOSITE)
    kp, ks, vp, vs, table, krows, vrows = opposite_rows(gen(71), D, cache)
    q = torch.zeros(B, 2, D, dtype=F[x])
    q[:, 0, 0], q[:, 1, 0] = torch.tensor(T_OPPOSITE, dtype=F[x]), -torch.tensor(T_OPPOSITE, dtype=F[x])
    out = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda().expand(B, -1), torch.full((B,), 2, dtype=torch.int32).cuda(), scale=1.0,
                              k_scale=cu(ks), v_scale=cu(vs)).cpu()
    for b in range(B):
        want, _, vabs, big = attend(q[b].double(), krows, vrows, 1.0)
        check_out(out[b], want, vabs, big, 2, x, carried(cache, x), D)


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
def test_a_term_less_is_seen(cache, x):
    """The bounds of the test above, with a term less planted in the oracle's weights: outside them."""
    D, op = 64, torch.bfloat16 if cache == "bf16" else torch.float16
    _, _, _, _, _, krows, vrows = opposite_rows(gen(71), D, cache)
    seen = 0
    for t in T_OPPOSITE:
        q = torch.zeros(1, D, dtype=torch.float64)
        q[0, 0] = t
        want, _, vabs, big = attend(q, krows, vrows, 1.0)
        s = krows[:, 0] @ q[0]
        p = torch.exp(s - s.max())
        w = p.float().to(op).double()
        if cache == "bf16" and x == "f32":                # two terms of three
            w = w + (p - w).float().to(op).double()
        got = ((w[:, None] * vrows[:, 0]).sum(0) / p.sum()).float().to(F[x])
        try:
            check_out(got[None], want, vabs, big, 2, x, carried(cache, x), D)
        except AssertionError:
            seen += 1
    assert seen >= 4, seen


def latent_opposite(g, R, cache, x):
    """The same for latent attention: latents c and -c, queries along c, value rows that pick the latent's own values."""
    dr, dn, dv, pt = 64, 16, min(R, 256), 16
    table, total = table_of(g, [2], pt)
    cp, cs = pool(g, total, 1, pt, R + dr, cache)
    c = torch.zeros(1, R + dr, dtype=torch.float64)
    c[0, :R] = (0.5 + torch.rand(R, generator=g)).double() * (1 - 2 * torch.randint(0, 2, (R,), generator=g))
    rows = torch.stack([put(cp, cs, table, 0, i, pt, c * (1 - 2 * i)) for i in range(2)])
    w = torch.zeros(1, dn + dv, R, dtype=F[x])
    w[0, 0] = (torch.sign(c[0, :R]) * (0.5 + torch.rand(R, generator=g))).to(F[x])
    w[0, dn:] = torch.eye(dv, R)
    q = torch.zeros(len(T_OPPOSITE), 1, dn + dr, dtype=F[x])
    q[:, 0, 0] = torch.tensor(T_OPPOSITE, dtype=F[x])
    return cp, cs, table, rows, w, q, dn, dv


def latent_bound(rows, w, q, b, R, dn, dv, cache, x, scale):
    """The 64-bit output and its bound: scores lose the queries' operands (and a Q8 row's, in f16), weights two terms or, over a
    Q8 cache, one, o its two terms; opposite rows round alike, so a Q8 row's rounding is relative to the output."""
    op = half_step(torch.bfloat16 if cache == "bf16" else torch.float16)
    qa = torch.cat([q[b, :, :dn].double() @ w[0, :dn].double(), q[b, :, dn:].double()], -1)
    o, _, vabs, big = attend(qa, rows, rows[..., :R], scale)
    ds = ((2 if cache == "q8" else 1) * op + (R + 96) * W) * big
    lost = op if cache == "q8" else op ** 2
    want, vabs = o[0, :dv], vabs[0, :dv]
    # 2^-25: half the distance of f16's values below 2^-14, 2^-24
    return want, (2.0 ** -25 if x == "f16" else 0.0) + (half_step(F[x]) + (op if cache == "q8" else 0.0) + 2.0 ** -15) * want.abs() + (2 * ds + lost + 2.0 ** -21 + (R + 16) * W) * vabs


@gpu_only
@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("f16", "f16"), ("q8", "f16"), ("q8", "bf16")])
@pytest.mark.parametrize("R", [128, 512])
def test_latent_weights_and_rows_carry_their_terms(gpu, cache, x, R):
    cp, cs, table, rows, w, q, dn, dv = latent_opposite(gen(72), R, cache, x)
    B, scale = len(T_OPPOSITE), 1.0 / R
    out = hb.latent_attention(q.cuda(), w.cuda(), cp.cuda(), table.cuda().expand(B, -1), torch.full((B,), 2, dtype=torch.int32).cuda(), scale=scale,
                              c_scale=cu(cs)).cpu()
    for b in range(B):
        want, tol = latent_bound(rows, w, q, b, R, dn, dv, cache, x, scale)
        err = (out[b, 0].double() - want).abs()
        assert (err <= tol).all(), (T_OPPOSITE[b], (err / tol).max())


@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("f16", "f16"), ("q8", "f16")])
def test_a_latent_term_less_is_seen(cache, x):
    """The bounds of the test above with a term less planted in the oracle's weights: one of the cache's type, for a Q8 cache one of
    bf16, in the rows too."""
    R, scale, seen = 128, 1.0 / 128, 0
    _, _, _, rows, w, q, dn, dv = latent_opposite(gen(72), R, cache, x)
    bf = lambda t: t.float().to(torch.float16 if cache == "f16" else torch.bfloat16).double()  # noqa: E731
    for b in range(len(T_OPPOSITE)):
        want, tol = latent_bound(rows, w, q, b, R, dn, dv, cache, x, scale)
        r = bf(rows) if cache == "q8" else rows
        qa = torch.cat([q[b, :, :dn].double() @ w[0, :dn].double(), q[b, :, dn:].double()], -1)
        s = (r[:, 0] @ qa[0]) * scale
        p = torch.exp(s - s.max())
        got = ((bf(p)[:, None] * r[:, 0, :dv]).sum(0) / p.sum()).float().to(F[x]).double()
        seen += bool(((got - want).abs() > tol).any())
    assert seen >= 4, seen


@gpu_only
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("D", [64, 128])
def test_f32_outputs_of_long_sums_do_not_drift(gpu, cache, D):
    """Equal weights and positive values: the output is the values' mean, and its error that of the sums alone. A CTA's warp adds
    its share of the tiles, t of them; the partial sums are half of the last one on average, so that their roundings are below t / 2
    half steps of it, and a tile's own two or three products, the pieces of the warps and CTAs and the division 24 more."""
    g = gen(77)
    n, Hkv, pt = 200_003, 4, 64
    pages = -(-n // pt)
    kp = torch.zeros(pages, Hkv, pt, D, device="cuda", dtype=torch.int8 if cache == "q8" else F[cache])
    if cache == "q8":
        vp, ks, vs = torch.randint(64, 128, kp.shape, generator=g).to(torch.int8).cuda(), *(torch.ones(pages, Hkv, pt, D // 64).cuda() / 64 for _ in range(2))
    else:
        vp, ks, vs = (1 + torch.rand(kp.shape, generator=g)).to(F[cache]).cuda(), None, None
    table = torch.randperm(pages, generator=g).to(torch.int32)[None].cuda()
    q = randn(g, 1, Hkv, D).cuda()
    out = hb.decode_attention(q, kp, vp, table, torch.tensor([n], dtype=torch.int32).cuda(), scale=0.1, k_scale=ks, v_scale=vs)[0]
    rows = vp[table[0].long()].transpose(1, 2).reshape(-1, Hkv, D)[:n].double() / (64 if cache == "q8" else 1)
    t = -(-pages * Hkv // (148 * 3)) + 3
    err = ((out.double() - rows.mean(0)).abs() / rows.mean(0)).max()
    assert err <= (t / 2 + 24) * W, err / W


@gpu_only
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_f32_scores_of_long_rows_do_not_drift(gpu, cache, D):
    """One position, positive keys and queries: lse is the score. Its 32 or 64 dims at a time are cut off by two products each and
    added with one rounding of a partial sum that is half of the last one on average; scaling and ln 2 are six roundings more."""
    g = gen(78)
    B = 64
    (kp, ks), (vp, vs) = (pool(g, B, 1, 16, D, cache) for _ in range(2))
    table = torch.arange(B, dtype=torch.int32)[:, None]
    k = (1 + torch.rand(B, 1, D, generator=g)).double()
    rows = torch.stack([put(kp, ks, table, b, 0, 16, k[b]) for b in range(B)])
    for b in range(B):
        put(vp, vs, table, b, 0, 16, k[b])
    q = 1 + torch.rand(B, 8, D, generator=g)
    _, lse = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), torch.ones(B, dtype=torch.int32).cuda(), scale=0.1, k_scale=cu(ks),
                                 v_scale=cu(vs), return_lse=True)
    want = torch.einsum("bhd,bd->bh", q.double(), rows[:, 0]) * float(np.float32(0.1))
    err = ((lse.cpu().double() - want).abs() / want).max()
    assert err <= (D / 32 / 2 + 4 + 6) * W, err / W


# ----------------------------------------------------------------------------------------- sequences out of range

@gpu_only
@pytest.mark.parametrize("cache", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("H,Hkv,D", [(8, 1, 64), (4, 4, 128), (40, 2, 64), (16, 2, 256)])
def test_decode_batch_with_sequences_out_of_range(gpu, cache, H, Hkv, D):
    """Negative, empty and too long sequences and one with a bad page between ones that can be read: zeros, NaN, and the
    others' values."""
    g = gen(73)
    lens = [40, -7, 33, 2 ** 31 - 1, 64, 0, 1, 130, 65, 17, 200, 10 ** 6, 5, -2 ** 31, 129]
    pools, table, (krows, vrows) = filled(g, [max(0, min(n, 200)) for n in lens], Hkv, 16, D, cache)
    table[7, 4] = 10 ** 6                                    # no such page
    (kp, ks), (vp, vs) = pools
    q = randn(g, len(lens), H, D, dtype=torch.float16)
    out, lse = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale=D ** -0.5,
                                   k_scale=cu(ks), v_scale=cu(vs), return_lse=True)
    out, lse = out.cpu(), lse.cpu()
    for b, n in enumerate(lens):
        if n <= 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
        elif n > 200 or b == 7:
            assert torch.isnan(out[b]).all() and torch.isnan(lse[b]).all()
        else:
            want, wl, vabs, big = attend(q[b].double(), krows[b], vrows[b], D ** -0.5)
            check_out(out[b], want, vabs, big, n, "f16", carried(cache, "f16"), D)
            check_lse(lse[b], wl, big, n, D)


@gpu_only
@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_pools_without_pages(gpu, cache):
    """No position has a page: nothing is written, rows read back and outputs are NaN, empty sequences stay zeros."""
    dt, x = (torch.int8 if cache == "q8" else torch.bfloat16), torch.bfloat16
    kp, vp = (torch.empty(0, 2, 16, 64, dtype=dt, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(0, 2, 16, 1, device="cuda") if cache == "q8" else None for _ in range(2))
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    table, start, pos0 = torch.zeros(2, 4, dtype=torch.int32).cuda(), i32(0, 3, 5), i32(0, 7)
    k = randn(gen(74), 5, 2, 64, dtype=x).cuda()
    hb.kv_write(k, k, kp, vp, table, start, pos0, k_scale=ks, v_scale=vs)
    ko, vo = torch.zeros_like(k), torch.zeros_like(k)
    hb.kv_read(kp, vp, table, start, pos0, ko, vo, k_scale=ks, v_scale=vs)
    assert torch.isnan(ko).all() and torch.isnan(vo).all()
    out = hb.decode_attention(k[:2].expand(2, 2, 64).contiguous(), kp, vp, table, i32(30, 0), scale=0.1, k_scale=ks, v_scale=vs)
    assert torch.isnan(out[0]).all() and (out[1] == 0).all()
    cp = torch.empty(0, 1, 16, 192, dtype=dt, device="cuda")
    cs = torch.empty(0, 1, 16, 3, device="cuda") if cache == "q8" else None
    q, w = randn(gen(75), 2, 4, 32 + 64, dtype=x).cuda(), randn(gen(76), 4, 32 + 16, 128, dtype=x).cuda()
    out = hb.latent_attention(q, w, cp, table, i32(30, 0), scale=0.1, c_scale=cs)
    assert torch.isnan(out[0]).all() and (out[1] == 0).all()


@gpu_only
@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_outputs_by_head(gpu, cache):
    """Outputs whose tokens lie closer than their heads ([heads, tokens, dim] seen as [tokens, heads, dim]), with room between
    them that keeps what it holds."""
    g = gen(79)
    lens = [40, 0, 70, 9, 1]
    pools, table, _ = filled(g, lens, 2, 16, 192, cache)
    (kp, ks), (vp, vs) = ((cu(a), cu(b)) for a, b in pools)
    n, q = torch.tensor(lens, dtype=torch.int32).cuda(), randn(g, 5, 8, 192, dtype=torch.bfloat16).cuda()
    by_head = lambda d: torch.full((8, 5, d + 8), 7.0, dtype=torch.bfloat16).cuda()  # noqa: E731
    out = by_head(192)
    hb.decode_attention(q, kp, vp, table.cuda(), n, scale=0.07, k_scale=ks, v_scale=vs, out=out.transpose(0, 1)[..., :192])
    assert torch.equal(out.transpose(0, 1)[..., :192], hb.decode_attention(q, kp, vp, table.cuda(), n, scale=0.07, k_scale=ks, v_scale=vs))
    assert (out[..., 192:] == 7.0).all()
    cp, cs = kp[:, :1].contiguous(), None if ks is None else ks[:, :1].contiguous()
    ql, w, out = randn(g, 5, 8, 32 + 64, dtype=torch.bfloat16).cuda(), randn(g, 8, 32 + 48, 128, dtype=torch.bfloat16, scale=0.1).cuda(), by_head(48)
    hb.latent_attention(ql, w, cp, table.cuda(), n, scale=0.1, c_scale=cs, out=out.transpose(0, 1)[..., :48])
    assert torch.equal(out.transpose(0, 1)[..., :48], hb.latent_attention(ql, w, cp, table.cuda(), n, scale=0.1, c_scale=cs))
    assert (out[..., 48:] == 7.0).all()


# ----------------------------------------------------------------------------------------- far rotary positions

def _pi():
    """pi * 2^220 by Machin's formula."""
    def atan_inv(m):
        total, term, k = 0, (1 << 260) // m, 0
        while term:
            total += (-1) ** k * (term // (2 * k + 1))
            term //= m * m
            k += 1
        return total
    return (16 * atan_inv(5) - 4 * atan_inv(239)) >> 40


def exact_table(freqs, first, n):
    """cos and sin of p * f with the angle reduced as a fraction: [n, len(freqs), 2]."""
    quarter, out = _pi() // 2, np.empty((n, len(freqs), 2))
    for j, f in enumerate(freqs):
        num, den = Fraction(float(f)).as_integer_ratio()
        for i in range(n):
            a = ((first + i) * num << 220) // den
            k = (2 * a + quarter) // (2 * quarter)
            r = (a - k * quarter) / (1 << 220)
            c, s = math.cos(r), math.sin(r)
            out[i, j] = ((c, s), (-s, c), (-c, -s), (s, -c))[k % 4]
    return torch.from_numpy(out)


def test_exact_table():
    f = [1.0, 0.731, -3e-5, 0.0]
    a = torch.arange(-3, 40, dtype=torch.float64)[:, None] * torch.tensor(f, dtype=torch.float64)
    assert (exact_table(f, -3, 43) - torch.stack([a.cos(), a.sin()], -1)).abs().max() < 1e-14


@gpu_only
@pytest.mark.parametrize("first", [2 ** 31 - 400, -2 ** 31 + 1, 10 ** 9 + 7, 131072, 0])
@pytest.mark.parametrize("scaling,factor", [("none", 1.0), ("yarn", 7.3)])
def test_rope_table_at_far_positions(gpu, first, scaling, factor):
    """The phase loses nothing at any position: against angles reduced as fractions, 2^-22 of the value (an ulp of sincospif and
    two roundings) and 2^-44 of the factor (the fraction's rest to first order)."""
    f, a = hb.rope_freqs(64, 1e4, scaling=scaling, factor=factor)
    f = np.concatenate([f, [1.0, -1.0, 6.5, 300.25, math.pi, 2 * math.pi, 1e-7]])
    got = hb.rope_table(f, 400, first=first, factor=a).cpu().double()
    want = exact_table(f, first, 400) * a
    err, tol = (got - want).abs(), 2.0 ** -22 * want.abs() + a * 2.0 ** -44
    assert (err <= tol).all(), ((err / tol).max(), (err > tol).sum())
