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
