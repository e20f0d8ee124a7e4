"""The attention operators on the GPU against plain 64-bit forms on the CPU.

Tolerances. u(t) is half a step of an element type (tests/attn_util.half_step), w = 2^-24 that of f32. Stored
values are one rounding of a value known to 64 bits: u(t), plus what the f32 steps before it lose. An attention
output is off by at most u(out) |o| + (2 ds + up + 2^-21 + n w) sum_r p_r |v_r|: each weight exp(s_r) / sum is off by twice
the largest score error ds, by the rounding up of a weight as an operand of the matrix instructions (none where
operands carry f32's bits) and by the f32 exponential and rescalings (2^-21 together), and a sum of n terms by n w."""
import itertools
import math

import pytest
import torch

import hearth_b200 as hb
from tests.attn_util import F, attend, dequant, gen, half_step, pool, put, quant, randn, rotate, table_of

pytestmark = pytest.mark.gpu
W = 2.0 ** -24
r32 = lambda v: v.float().double()  # noqa: E731


def cu(x):
    return None if x is None else x.cuda()


def table64(dim, n_pos, theta=1e4):
    f = theta ** (-torch.arange(dim // 2, dtype=torch.float64) * 2 / dim)
    a = torch.arange(n_pos, dtype=torch.float64)[:, None] * f
    return a.cos(), a.sin()


def cs_of(cos, sin):
    return torch.stack([cos, sin], -1).float()


# ----------------------------------------------------------------------------------------- rotary positions

@pytest.mark.parametrize("dim,first,n,scaling", [(2, 0, 7, "none"), (64, 0, 1000, "none"), (128, 999_983, 517, "linear"),
                                                 (80, 2_147_483_000, 600, "none"), (64, -300, 400, "yarn"),
                                                 (1024, 12345, 33, "ntk")])
def test_rope_table(gpu, dim, first, n, scaling):
    f, a = hb.rope_freqs(dim, 1e6, scaling=scaling, factor=1.0 if scaling == "none" else 8.0)
    got = hb.rope_table(f, n, first=first, factor=a).cpu().double()
    ang = torch.arange(first, first + n, dtype=torch.float64)[:, None] * torch.from_numpy(f)
    want = torch.stack([ang.cos(), ang.sin()], -1) * a
    # 2 ulp of the value (4 half steps), and the 64-bit phase: angle * 2^-52
    tol = 4 * W * want.abs() + a * (ang.abs() * 2.0 ** -51)[..., None] + 2.0 ** -40
    assert (got - want).abs().le(tol).all(), ((got - want).abs() / tol).max()


def test_rope_table_empty(gpu):
    assert hb.rope_table([1.0], 0).shape == (0, 1, 2)


ROPES = [dict(T=1, H=1, D=64, rot=64, off=0), dict(T=5, H=3, D=80, rot=40, off=40), dict(T=7, H=2, D=192, rot=64, off=128),
         dict(T=3, H=4, D=50, rot=18, off=3), dict(T=130, H=5, D=128, rot=128, off=0), dict(T=9, H=64, D=576, rot=64, off=512),
         dict(T=4, H=2, D=10, rot=2, off=8), dict(T=2, H=3, D=256, rot=24, off=8)]


@pytest.mark.parametrize("shape", ROPES, ids=str)
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("x,y", [("f32", "f32"), ("f32", "bf16"), ("bf16", "bf16"), ("f16", "f16"), ("bf16", "f32"), ("f16", "bf16")])
def test_rope(gpu, shape, inter, x, y):
    T, H, D, rot, off = (shape[k] for k in ("T", "H", "D", "rot", "off"))
    g = gen(1)
    cos, sin = table64(rot, 300)
    pos = torch.randint(0, 300, (T,), generator=g, dtype=torch.int32)
    xs = randn(g, T, H, D, dtype=F[x])
    cs = cs_of(cos, sin)
    want = rotate(xs.double(), cs[pos.long(), :, 0].double(), cs[pos.long(), :, 1].double(), inter, off, r32).to(F[y])
    wide = torch.zeros(T, H + 1, D + 5, dtype=F[x])        # odd strides: the element path
    wide[:, :H, :D] = xs
    out = torch.full((T, H, D), 7.0, dtype=F[y]).cuda()
    for src in (xs.cuda(), wide.cuda()[:, :H, :D]):
        got = hb.rope(src, pos.cuda(), cs.cuda(), interleaved=inter, offset=off, out=out.fill_(7.0))
        assert torch.equal(got.cpu(), want)                 # the f32 steps are defined: equal bits
    if x == y:
        buf = xs.cuda()
        assert torch.equal(hb.rope(buf, pos.cuda(), cs.cuda(), interleaved=inter, offset=off, out=buf).cpu(), want)
        buf = wide.cuda()
        hb.rope(buf[:, :H, :D], pos.cuda(), cs.cuda(), interleaved=inter, offset=off, out=buf[:, :H, :D])
        assert torch.equal(buf[:, :H, :D].cpu(), want)
        assert (buf[:, H:] == 0).all() and (buf[:, :, D:] == 0).all()


def test_rope_positions_outside_the_table_and_no_tokens(gpu):
    cs = cs_of(*table64(64, 50)).cuda()
    x = randn(gen(2), 4, 2, 96, dtype=torch.bfloat16).cuda()
    for inter in (False, True):
        y = hb.rope(x, torch.tensor([0, -1, 50, 49], dtype=torch.int32).cuda(), cs, interleaved=inter)
        bad = torch.isnan(y).all(-1).cpu(), torch.isnan(y[..., :64]).all(-1).cpu()
        assert bad[1].tolist() == [[False] * 2, [True] * 2, [True] * 2, [False] * 2] and not bad[0].any()
        assert torch.equal(y[..., 64:], x[..., 64:])
    assert hb.rope(x[:0], torch.zeros(0, dtype=torch.int32).cuda(), cs).shape == (0, 2, 96)


# ----------------------------------------------------------------------------------------- cache rows

KV = [dict(news=[1], past=[0], Hkv=1, D=64, pt=16), dict(news=[3, 0, 40, 1], past=[5, 9, 30, 0], Hkv=2, D=128, pt=16),
      dict(news=[17, 5], past=[3, 1], Hkv=3, D=64, pt=1), dict(news=[70, 9, 33], past=[0, 63, 64], Hkv=1, D=576, pt=32, latent=True),
      dict(news=[9, 2], past=[2, 2], Hkv=5, D=256, pt=8), dict(news=[6, 130], past=[1, 250], Hkv=2, D=64, pt=128)]


def kv_case(g, c, cache, x):
    B, lens = len(c["news"]), [a + b for a, b in zip(c["news"], c["past"])]
    table, total = table_of(g, lens, c["pt"])
    start = torch.tensor([0] + list(itertools.accumulate(c["news"])), dtype=torch.int32) + 2    # two padding rows in front
    T = int(start[-1]) + 3                                                                      # three behind
    k, v = (randn(g, T, c["Hkv"], c["D"], dtype=F[x]) for _ in range(2))
    pools = [pool(g, total, c["Hkv"], c["pt"], c["D"], cache, fill=3.0) for _ in range(2)]
    return B, lens, table, start, torch.tensor(c["past"], dtype=torch.int32), T, k, v, pools


def bits(t):
    return t.contiguous().view(torch.uint8)


@pytest.mark.parametrize("c", KV, ids=str)
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("rope", [None, "half", "inter"])
def test_kv_write_and_read(gpu, c, cache, x, rope):
    g = gen(3)
    latent = c.get("latent", False)
    B, lens, table, start, pos0, T, k, v, ((kp, ks), (vp, vs)) = kv_case(g, c, cache, x)
    rot, off = (64, 512) if latent else (c["D"] // 2, 0)
    cs = cs_of(*table64(rot, max(lens)))
    rows = [(b, t, int(pos0[b]) + t - int(start[b])) for b in range(B) for t in range(int(start[b]), int(start[b + 1]))]
    kd = k.double()
    if rope:
        for b, t, p in rows:
            kd[t] = rotate(kd[t:t + 1], cs[p:p + 1, :, 0].double(), cs[p:p + 1, :, 1].double(), rope == "inter", off, r32)[0]
    dev = [cu(t) for t in (kp, None if latent else vp, ks, None if latent else vs)]
    wide = torch.zeros(T, c["Hkv"] + 1, c["D"] + 4, dtype=F[x])
    wide[:, :c["Hkv"], :c["D"]] = k
    for src in (k.cuda(), wide.cuda()[:, :c["Hkv"], :c["D"]]):
        hb.kv_write(src, None if latent else v.cuda(), dev[0], dev[1], table.cuda(), start.cuda(), pos0.cuda(), k_scale=dev[2], v_scale=dev[3],
                    cs=cu(cs) if rope else None, interleaved=rope == "inter", offset=off)
    want = {}
    for b, t, p in rows:
        want[t] = put(kp, ks, table, b, p, c["pt"], kd[t]), None if latent else put(vp, vs, table, b, p, c["pt"], v[t].double())
    for got, ref in zip(dev, (kp, vp, ks, vs)):     # what was written, and every other byte
        assert got is None or torch.equal(bits(got.cpu()), bits(ref))
    for y in ("f32", "f16", "bf16"):
        outs = [torch.full((T, c["Hkv"], c["D"]), 9.0, dtype=F[y]).cuda() for _ in range(1 if latent else 2)]
        hb.kv_read(dev[0], dev[1], table.cuda(), start.cuda(), pos0.cuda(), outs[0], None if latent else outs[1], k_scale=dev[2], v_scale=dev[3])
        for i, o in enumerate(outs):
            o = o.cpu()
            for t in range(T):
                ref = want[t][i].float().to(F[y]) if t in want else torch.full((c["Hkv"], c["D"]), 9.0, dtype=F[y])
                assert torch.equal(o[t], ref), (y, i, t)


def test_kv_bad_pages_and_positions(gpu):
    """Ids outside the pool, positions outside the table or negative: nothing written, NaN read; the rest works."""
    kp, vp = torch.zeros(4, 1, 8, 64, dtype=torch.bfloat16).cuda(), torch.zeros(4, 1, 8, 64, dtype=torch.bfloat16).cuda()
    table = torch.tensor([[2, 4], [-7, 1], [3, 2_000_000_000]], dtype=torch.int32).cuda()
    start = torch.tensor([0, 17, 33, 43], dtype=torch.int32).cuda()
    pos0 = torch.tensor([0, 0, -2], dtype=torch.int32).cuda()
    k = randn(gen(4), 43, 1, 64, dtype=torch.bfloat16).cuda()
    hb.kv_write(k, k, kp, vp, table, start, pos0)
    assert torch.equal(kp[2, 0], k[:8, 0]) and torch.equal(kp[1, 0], k[25:33, 0]) and torch.equal(kp[3, 0], k[35:43, 0])
    assert (kp[0] == 0).all()
    ko, vo = torch.zeros_like(k), torch.zeros_like(k)
    hb.kv_read(kp, vp, table, start, pos0, ko, vo)
    good = torch.zeros(43, dtype=torch.bool)
    good[:8] = good[25:33] = good[35:43] = True
    assert torch.equal(ko[good.cuda()], k[good.cuda()]) and torch.isnan(ko[~good.cuda()]).all() and torch.isnan(vo[~good.cuda()]).all()


def test_kv_q8_values_at_the_edges(gpu):
    """Zero blocks, blocks of subnormal and of the largest values, ties, and blocks that hold NaN or infinities."""
    x = randn(gen(5), 12, 1, 128)
    x[0] = 0
    x[1, 0, :64] *= 1e-42
    x[2, 0, :64] *= 1e38
    x[3, 0, 5] = float("nan")
    x[4, 0, 70] = float("inf")
    x[5, 0, 3] = -float("inf")
    x[6, 0, :64] = torch.arange(64) - 31.5
    x[6, 0, 0] = 127.0
    x[7] = -0.0
    kp, ks = torch.zeros(1, 1, 16, 128, dtype=torch.int8), torch.zeros(1, 1, 16, 2)
    dev = [t.cuda() for t in (kp, ks)]
    tab, start, p0 = torch.zeros(1, 1, dtype=torch.int32), torch.tensor([0, 12], dtype=torch.int32), torch.tensor([0], dtype=torch.int32)
    hb.kv_write(x.cuda(), None, dev[0], None, tab.cuda(), start.cuda(), p0.cuda(), k_scale=dev[1])
    code, d = quant(x)
    fin = torch.isfinite(d)
    assert torch.equal(torch.isfinite(dev[1][0, 0, :12].cpu()), fin[:, 0])
    assert torch.equal(dev[1][0, 0, :12].cpu()[fin[:, 0]], d[:, 0][fin[:, 0]])
    got = dev[0][0, 0, :12].cpu().view(12, 2, 64)
    assert torch.equal(got[fin[:, 0]], code.view(12, 2, 64)[fin[:, 0]])
    out = torch.zeros(12, 1, 128).cuda()
    hb.kv_read(dev[0], None, tab.cuda(), start.cuda(), p0.cuda(), out, None, k_scale=dev[1])
    assert torch.equal(torch.isnan(out.cpu()).view(12, 2, 64).all(-1), ~fin[:, 0])
    blk = (out.cpu().double() - x.double()).abs().view(12, 2, 64)[fin[:, 0]]
    dd = d[:, 0][fin[:, 0]].double()[:, None]
    # half a code and the f32 steps (the scale's own rounding is at most half of 2^-149, 127 times over); where
    # 1 / scale passes f32's range (scales under 2^-128) every code is 0 or +-127: off by less than the block's maximum
    assert (blk <= torch.where(dd < 2.0 ** -128, 127 * dd, (0.5 + 127 * 3 * W) * dd) + 2.0 ** -149 * 64).all()


# ----------------------------------------------------------------------------------------- decode attention

def filled(g, lens, Hkv, pt, D, cache, width=None, scale=1.0, sides=2):
    """A cache with its sequences' rows: pools, scales, table, and the f64 rows [n, Hkv, D] of each sequence."""
    table, total = table_of(g, lens, pt, width=width)
    pools, rows = [], []
    for _ in range(sides):
        p, s = pool(g, total, Hkv, pt, D, cache)
        seqs = []
        for b, n in enumerate(lens):
            x = randn(g, max(n, 0), Hkv, D, scale=scale).double()
            seqs.append(torch.stack([put(p, s, table, b, i, pt, x[i]) for i in range(n)]) if n > 0 else x)
        pools.append((p, s))
        rows.append(seqs)
    return pools, table, rows


def operand(cache, x):
    """Half a step of a softmax weight as an operand: none for f32 queries."""
    if x == "f32":
        return 0.0
    return half_step(torch.float16 if cache == "f16" else torch.bfloat16)


def check_out(got, want, vabs, big, n, x, up, D):
    ds = (D + 16) * W * big[:, None]
    tol = half_step(F[x]) * want.abs() + (2 * ds + up + 2.0 ** -21 + n * W) * vabs + 1e-30
    err = (got.double() - want).abs()
    assert (err <= tol).all(), (err / tol).max()


def check_attn(lens, H, Hkv, D, pt, cache, x, seed=6, width=None, qscale=1.0, **kw):
    g = gen(seed)
    pools, table, (krows, vrows) = filled(g, lens, Hkv, pt, D, cache, width)
    q = randn(g, len(lens), H, D, dtype=F[x], scale=qscale)
    (kp, ks), (vp, vs) = pools
    scale = D ** -0.5
    out, lse = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale=scale,
                                   k_scale=cu(ks), v_scale=cu(vs), return_lse=True, **kw)
    out, lse = out.cpu(), lse.cpu()
    for b, n in enumerate(lens):
        want, wl, vabs, big = attend(q[b].double(), krows[b], vrows[b], scale)
        if n <= 0:
            assert (out[b] == 0).all() and (lse[b] == -math.inf).all()
            continue
        check_out(out[b], want, vabs, big, n, x, operand(cache, x), D)
        assert ((lse[b].double() - wl).abs() <= (D + 16) * W * big + 2.0 ** -20 + n * W + 2 * W * wl.abs()).all()


LENS = [[1], [0], [2, 1, 0, 15, 16, 17], [31, 33, 63, 64, 65, 127, 129, 0, 255, 257], [700, 3], [1100]]


@pytest.mark.parametrize("lens", LENS, ids=str)
@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
def test_decode_attention_lengths(gpu, lens, cache, x):
    check_attn(lens, 8, 2, 128, 16, cache, x)


@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 3), (4, 1), (7, 1), (8, 1), (9, 1), (24, 2), (32, 2), (40, 1), (64, 1), (33, 11)])
@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("q8", "f32"), ("f16", "f16")])
def test_decode_attention_heads(gpu, H, Hkv, cache, x):
    check_attn([37, 5, 130], H, Hkv, 64, 16, cache, x)


@pytest.mark.parametrize("D", [16, 32, 48, 64, 80, 96, 112, 128, 144, 160, 192, 240, 256])
@pytest.mark.parametrize("cache,x", [("f16", "f32"), ("bf16", "bf16"), ("q8", "bf16")])
def test_decode_attention_dims(gpu, D, cache, x):
    if cache == "q8" and D % 64:
        pytest.skip("Q8 rows come in blocks of 64")
    check_attn([50, 129, 1], 6, 2, D, 32, cache, x)


@pytest.mark.parametrize("pt", [1, 2, 4, 8, 16, 32, 64, 128, 1024])
@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_decode_attention_pages(gpu, pt, cache):
    check_attn([73, 0, 200, 6], 8, 2, 64, pt, cache, "bf16")


def test_decode_attention_large_scores(gpu):
    for x in ("f32", "bf16", "f16"):
        check_attn([300, 40], 8, 2, 128, 16, "f16", x, qscale=30.0)
        check_attn([300, 40], 8, 2, 128, 16, "bf16", x, qscale=30.0)


def test_decode_attention_query_ranges(gpu):
    """Queries whose size is far from one, in both directions, against every cache: nothing overflows or is flushed."""
    for cache, s in itertools.product(("f16", "bf16", "q8"), (1e-6, 3e4)):
        g = gen(7)
        pools, table, (krows, vrows) = filled(g, [90], 1, 16, 64, cache)
        q = randn(g, 1, 4, 64, dtype=torch.bfloat16, scale=s)
        scale = 1.0 / (8.0 * s)
        (kp, ks), (vp, vs) = pools
        out = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), torch.tensor([90], dtype=torch.int32).cuda(), scale=scale,
                                  k_scale=cu(ks), v_scale=cu(vs)).cpu()
        want, _, vabs, big = attend(q[0].double(), krows[0], vrows[0], scale)
        check_out(out[0], want, vabs, big, 90, "bf16", operand(cache, "bf16"), 64)


def test_decode_attention_one_heavy_among_many_light(gpu):
    """One position takes nearly all the weight; the others' small weights still add up."""
    n, D = 3000, 64
    for cache, x in itertools.product(("f16", "bf16", "q8"), ("f32", "bf16", "f16")):
        g = gen(8)
        pools, table, (krows, vrows) = filled(g, [n], 1, 64, D, cache, scale=0.25)
        (kp, ks), (vp, vs) = pools
        q = randn(g, 1, 2, D, dtype=F[x], scale=0.1)
        q[..., 0] = 12.0
        heavy = torch.zeros(1, D, dtype=torch.float64)
        heavy[0, 0] = 8.0
        krows[0][1234] = put(kp, ks, table, 0, 1234, 64, heavy)
        scale = 0.15
        out = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), scale=scale,
                                  k_scale=cu(ks), v_scale=cu(vs)).cpu()
        want, _, vabs, big = attend(q[0].double(), krows[0], vrows[0], scale)
        check_out(out[0], want, vabs, big, n, x, operand(cache, x), D)


def test_decode_attention_bad_pages_and_infinities(gpu):
    g = gen(9)
    pools, table, (krows, vrows) = filled(g, [40, 40, 40, 40, 40], 1, 16, 64, "bf16")
    (kp, _), (vp, _) = pools
    q = randn(g, 5, 8, 64, dtype=torch.bfloat16)
    q[..., 0] = q[..., 0].abs() + 0.5
    table[1, 1] = 99                                          # no such page
    lens = torch.tensor([40, 40, 40, 40, 1000], dtype=torch.int32)   # the last is longer than its table
    kp[int(table[2, 0]), 0, 3, 0] = float("inf")              # a score of +inf: the formula gives NaN
    kp[int(table[3, 0]), 0, 3, 0] = -float("inf")             # -inf: no weight
    krows[3][3, 0, 0] = -float("inf")
    out, lse = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), table.cuda(), lens.cuda(), scale=0.125, return_lse=True)
    out, lse = out.cpu(), lse.cpu()
    assert torch.isnan(out[[1, 2, 4]]).all() and torch.isnan(lse[[1, 4]]).all()
    for b in (0, 3):
        keep = [i for i in range(40) if not (b == 3 and i == 3)]
        want, wl, vabs, big = attend(q[b].double(), krows[b][keep], vrows[b][keep], 0.125)
        check_out(out[b], want, vabs, big, 40, "bf16", operand("bf16", "bf16"), 64)


def test_decode_attention_all_scores_minus_infinity(gpu):
    """A row whose scores leave nothing gives zeros and -inf, like an empty one."""
    kp = torch.full((2, 1, 16, 64), -float("inf"), dtype=torch.bfloat16)
    vp = torch.ones_like(kp)
    q = torch.ones(1, 4, 64, dtype=torch.bfloat16)
    out, lse = hb.decode_attention(q.cuda(), kp.cuda(), vp.cuda(), torch.tensor([[0, 1]], dtype=torch.int32).cuda(),
                                   torch.tensor([20], dtype=torch.int32).cuda(), scale=1.0, return_lse=True)
    assert (out == 0).all() and (lse == -math.inf).all()


def test_decode_attention_strides_shared_table_and_scratch(gpu):
    """Padded query and output rows, one table row for several tokens of a sequence, a scratch of the caller's full
    of NaN, and the same bits again."""
    g = gen(10)
    (kp, _), (vp, _) = (p := filled(g, [200], 2, 16, 128, "bf16"))[0]
    table, (krows, vrows) = p[1], p[2]
    lens = [197, 198, 199, 200, 1, 0]
    wide = randn(g, 6, 9, 136, dtype=torch.bfloat16).cuda()
    q = wide[:, :8, 3:131]
    out = torch.full((6, 9, 136), 5.0, dtype=torch.bfloat16).cuda()
    shared = table.cuda().expand(6, -1)
    ws = torch.full((1 << 24,), 255, dtype=torch.uint8).cuda()
    args = (q, kp.cuda(), vp.cuda(), shared, torch.tensor(lens, dtype=torch.int32).cuda())
    hb.decode_attention(*args, scale=0.1, out=out[:, :8, 3:131], workspace=ws)
    again = hb.decode_attention(*args, scale=0.1)
    assert torch.equal(again, out[:, :8, 3:131])
    rest = out.clone()
    rest[:, :8, 3:131] = 5.0
    assert (rest == 5.0).all()
    for b, n in enumerate(lens):
        want, _, vabs, big = attend(q[b].cpu().double(), krows[0][:n], vrows[0][:n], 0.1)
        check_out(again[b].cpu(), want, vabs, big, n, "bf16", operand("bf16", "bf16"), 128)
    with pytest.raises(ValueError, match="workspace"):
        hb.decode_attention(*args, scale=0.1, workspace=ws[:8])


def test_decode_attention_many_sequences(gpu):
    """More sequences than CTAs, lengths from nothing to a few pages."""
    g = gen(11)
    lens = [int(v) for v in torch.randint(0, 40, (701,), generator=g)]
    check_attn(lens, 4, 2, 64, 8, "bf16", "bf16", seed=12)


def test_decode_attention_long_split_over_the_cache(gpu):
    """A context long enough that every CTA has a share of one sequence, beside short ones."""
    g = gen(13)
    n, D = 70_001, 64
    k = torch.randn((2, 1100, 1, 64, D), generator=g, dtype=torch.float32).to(torch.bfloat16)
    perm = torch.randperm(1100, generator=g)[:1094].to(torch.int32)
    table = torch.stack([perm, perm])
    table[1, 0] = perm[5]
    q = randn(g, 2, 8, D, dtype=torch.float32)
    out = hb.decode_attention(q.cuda(), k[0].cuda(), k[1].cuda(), table.cuda(), torch.tensor([n, 7], dtype=torch.int32).cuda(), scale=0.125).cpu()
    for b, m in ((0, n), (1, 7)):
        kr, vr = (k[i][table[b].long()].transpose(1, 2).reshape(-1, 1, D)[:m].double() for i in (0, 1))
        want, _, vabs, big = attend(q[b].double(), kr, vr, 0.125)
        check_out(out[b], want, vabs, big, m, "f32", 0.0, D)


# ----------------------------------------------------------------------------------------- latent attention

def check_latent(lens, H, R, dr, dn, dv, pt, cache, x, seed=20, c_rows=None, **kw):
    g = gen(seed)
    pools, table, (rows,) = filled(g, lens, 1, pt, R + dr, cache, sides=1)
    cp, cs = pools[0]
    q = randn(g, len(lens), H, dn + dr, dtype=F[x])
    w = randn(g, H, dn + dv, R, dtype=F[x], scale=R ** -0.5)
    scale = (dn + dr) ** -0.5
    out = hb.latent_attention(q.cuda(), w.cuda(), cp.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale=scale,
                              c_scale=cu(cs), **kw).cpu()
    mma = torch.bfloat16 if cache == "q8" else F[x]
    up = half_step(mma)
    for b, n in enumerate(lens):
        if n <= 0:
            assert (out[b] == 0).all()
            continue
        qa = torch.einsum("hd,hdr->hr", q[b, :, :dn].double(), w[:, :dn].double())
        qf = torch.cat([qa, q[b, :, dn:].double()], -1)
        o, _, vabs, big = attend(qf, rows[b], rows[b][..., :R], scale)
        wv = w[:, dn:].double()
        want = torch.einsum("hr,hvr->hv", o, wv)
        wabs = torch.einsum("hr,hvr->hv", vabs, wv.abs())
        # scores: qa rounded to an operand, and f32 sums; weights rounded to an operand; o split in two operands
        # (its rest is below 2^-15); f32 sums over n and R terms
        ds = (up + (R + dr + dn + 32) * W) * big[:, None]
        tol = half_step(F[x]) * want.abs() + (2 * ds + up + 2.0 ** -15 + (n + R + 16) * W) * wabs
        err = (out[b].double() - want).abs()
        assert (err <= tol).all(), (b, (err / tol).max())
        # the roundings are independent: in the 2-norm at most the three operands' and the output's half steps together
        assert err.norm() <= 4 * max(up, half_step(F[x])) * want.norm(), (b, err.norm() / want.norm())


@pytest.mark.parametrize("lens", [[1], [0], [3, 0, 15, 16, 17], [63, 64, 65, 127, 128, 129, 0, 200], [1000, 2]], ids=str)
@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("f16", "f16"), ("q8", "bf16"), ("q8", "f16")])
def test_latent_attention_lengths(gpu, lens, cache, x):
    check_latent(lens, 16, 512, 64, 128, 128, 64, cache, x)


@pytest.mark.parametrize("H", [1, 2, 7, 8, 16, 24, 40, 64, 65, 128, 200])
def test_latent_attention_heads(gpu, H):
    check_latent([70, 1, 130], H, 512, 64, 64, 64, 32, "bf16", "bf16")
    check_latent([70, 1, 130], H, 512, 64, 64, 64, 32, "q8", "bf16")


@pytest.mark.parametrize("R,dr,dn,dv", [(128, 16, 16, 16), (256, 64, 64, 128), (384, 32, 128, 64), (512, 48, 48, 256), (512, 64, 256, 16)])
@pytest.mark.parametrize("cache,x", [("bf16", "bf16"), ("f16", "f16"), ("q8", "bf16")])
def test_latent_attention_dims(gpu, R, dr, dn, dv, cache, x):
    if cache == "q8" and dr % 64:
        pytest.skip("Q8 rows come in blocks of 64")
    check_latent([90, 33], 12, R, dr, dn, dv, 16, cache, x)


@pytest.mark.parametrize("pt", [1, 2, 8, 16, 32, 64, 128, 1024])
@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_latent_attention_pages(gpu, pt, cache):
    check_latent([73, 0, 150], 16, 512, 64, 64, 64, pt, cache, "bf16")


def test_latent_attention_many_sequences(gpu):
    g = gen(21)
    check_latent([int(v) for v in torch.randint(0, 30, (331,), generator=g)], 8, 128, 64, 16, 16, 8, "bf16", "bf16")


@pytest.mark.parametrize("cache,x,pt", [("bf16", "bf16", 64), ("f16", "f16", 16), ("bf16", "bf16", 128), ("bf16", "bf16", 8), ("q8", "bf16", 32)])
@pytest.mark.parametrize("H,R", [(64, 512), (16, 512), (100, 512), (24, 256), (8, 128)])
def test_latent_attention_many_tiles_a_cta(gpu, cache, x, pt, H, R):
    """Long rows of tiles in every CTA, runs that end inside and at the end of a tile, in any order: the buffers turn over
    many times. Pages are drawn from a small pool, so sequences share them."""
    g = gen(23)
    lens = [6000, 64, 640, 1, 5993, 0, 128, 4097, 63, 6001, 3000, 2000, 64 * 90, 17, 5000, 6003] + [64 * i + i % 3 - 1 for i in range(1, 60)]
    W, pages = R + 64, 12000 // pt
    if cache == "q8":
        cp, cs = torch.randint(-127, 128, (pages, 1, pt, W), generator=g).to(torch.int8), torch.rand((pages, 1, pt, W // 64), generator=g) / 64
        val = dequant(cp.reshape(-1, W), cs.reshape(-1, W // 64)).view(pages, pt, W)
    else:
        cp, cs = randn(g, pages, 1, pt, W, dtype=F[x]), None
        val = cp.double()[:, 0]
    table = torch.randint(0, pages, (len(lens), -(-6003 // pt)), generator=g, dtype=torch.int32)
    q, w = randn(g, len(lens), H, 64 + 64, dtype=F[x]), randn(g, H, 128, R, dtype=F[x], scale=R ** -0.5)
    out = hb.latent_attention(q.cuda(), w.cuda(), cp.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale=0.09, c_scale=cu(cs))
    val, wd, qd, td = val.cuda(), w.cuda().double(), q.cuda().double(), table.cuda().long()
    for b, n in enumerate(lens):
        if n == 0:
            assert (out[b] == 0).all()
            continue
        c = val[td[b, :-(-n // pt)]].reshape(-1, W)[:n]
        qa = torch.cat([torch.einsum("hd,hdr->hr", qd[b, :, :64], wd[:, :64]), qd[b, :, 64:]], -1)
        p = torch.softmax((qa @ c.T) * 0.09, -1)
        want = torch.einsum("hr,hvr->hv", p @ c[:, :R], wd[:, 64:])
        err = (out[b].double() - want).norm() / want.norm()
        assert err <= 4 * half_step(torch.bfloat16 if x == "bf16" else F[x]), (b, n, err)   # qa, the weights, o's rest, out


def test_latent_attention_bad_pages_strides_and_scratch(gpu):
    g = gen(22)
    pools, table, (rows,) = filled(g, [100, 100, 100], 1, 16, 576, "bf16", sides=1)
    cp = pools[0][0].cuda()
    wide = randn(g, 3, 17, 200, dtype=torch.bfloat16).cuda()
    q, w = wide[:, :16, 8:200], randn(g, 16, 256, 512, dtype=torch.bfloat16, scale=0.05).cuda()
    lens = torch.tensor([100, 100, 100], dtype=torch.int32).cuda()
    good = hb.latent_attention(q, w, cp, table.cuda(), lens, scale=0.07)
    out = torch.full((3, 17, 131), 5.0, dtype=torch.bfloat16).cuda()
    ws = torch.full((1 << 26,), 255, dtype=torch.uint8).cuda()
    hb.latent_attention(q, w, cp, table.cuda(), lens, scale=0.07, out=out[:, :16, 2:130], workspace=ws)
    assert torch.equal(out[:, :16, 2:130], good)
    rest = out.clone()
    rest[:, :16, 2:130] = 5.0
    assert (rest == 5.0).all()
    assert torch.equal(hb.latent_attention(q.contiguous(), w, cp, table.cuda(), lens, scale=0.07), good)
    table[1, 2] = -5
    lens[2] = 10_000
    got = hb.latent_attention(q, w, cp, table.cuda(), lens, scale=0.07)
    assert torch.equal(got[0], good[0]) and torch.isnan(got[1:]).all()


# ----------------------------------------------------------------------------------------- together

def run_decode(dec, steps, graph):
    """Steps of a decoder's attention: queries rotated, keys rotated into the cache, attention; `graph`: the first step
    captured, the others replayed with new inputs in the same buffers."""
    outs = []
    if graph:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            dec.load(0)
            dec.step()
        torch.cuda.current_stream().wait_stream(side)
        G = torch.cuda.CUDAGraph()
        with torch.cuda.graph(G):
            dec.step()
    for i in range(steps):
        dec.load(i)
        if graph:
            G.replay()
        else:
            dec.step()
        outs.append(dec.out.cpu().clone())
    return outs


class _Gqa:
    def __init__(self, cache, B=3, H=8, Hkv=2, D=128, pt=16, steps=20):
        g = gen(30)
        self.B, self.H, self.Hkv, self.D, self.steps = B, H, Hkv, D, steps
        self.q, self.k, self.v = (randn(g, steps, B, n, D) for n in (H, Hkv, Hkv))
        self.past = [0, 13, 30]
        table, total = table_of(g, [p + steps for p in self.past], pt)
        (kp, ks), (vp, vs) = (pool(g, total, Hkv, pt, D, cache) for _ in range(2))
        self.dev = [cu(t) for t in (kp, vp, ks, vs, table)]
        freqs, a = hb.rope_freqs(D, 1e4)
        self.cs = hb.rope_table(freqs, 64, factor=a)
        self.start = torch.arange(B + 1, dtype=torch.int32).cuda()
        self.bq, self.bk, self.bv = (torch.zeros(B, n, D).cuda() for n in (H, Hkv, Hkv))
        self.pos, self.lens = torch.zeros(B, dtype=torch.int32).cuda(), torch.zeros(B, dtype=torch.int32).cuda()
        self.qr, self.out = torch.zeros(B, H, D).cuda(), torch.zeros(B, H, D).cuda()
        # the past of each sequence
        pk, pv = (randn(g, sum(self.past), Hkv, D) for _ in range(2))
        st = torch.tensor([0] + list(itertools.accumulate(self.past)), dtype=torch.int32)
        hb.kv_write(pk.cuda(), pv.cuda(), self.dev[0], self.dev[1], self.dev[4], st.cuda(), torch.zeros(B, dtype=torch.int32).cuda(),
                    k_scale=self.dev[2], v_scale=self.dev[3], cs=self.cs)
        self.seqs = [([pk[st[b]:st[b + 1]]], [pv[st[b]:st[b + 1]]]) for b in range(B)]

    def load(self, i):
        for buf, x in ((self.bq, self.q[i]), (self.bk, self.k[i]), (self.bv, self.v[i])):
            buf.copy_(x)
        self.pos.copy_(torch.tensor([p + i for p in self.past], dtype=torch.int32))
        self.lens.copy_(torch.tensor([p + i + 1 for p in self.past], dtype=torch.int32))

    def step(self):
        kp, vp, ks, vs, table = self.dev
        hb.rope(self.bq, self.pos, self.cs, out=self.qr)
        hb.kv_write(self.bk, self.bv, kp, vp, table, self.start, self.pos, k_scale=ks, v_scale=vs, cs=self.cs)
        hb.decode_attention(self.qr, kp, vp, table, self.lens, scale=self.D ** -0.5, k_scale=ks, v_scale=vs, out=self.out)

    def want(self, i, b, cache):
        cos, sin = (t.float().double() for t in table64(self.D, 64))
        n = self.past[b] + i + 1
        k = torch.cat([self.seqs[b][0][0], self.k[:i + 1, b]]).double()
        v = torch.cat([self.seqs[b][1][0], self.v[:i + 1, b]]).double()
        k = rotate(k, cos[:n], sin[:n], False, 0, r32)
        store = (lambda t: dequant(*quant(t.float()))) if cache == "q8" else (lambda t: t.to(F[cache]).double())
        p = n - 1
        q = rotate(self.q[i, b:b + 1].double(), cos[p:p + 1], sin[p:p + 1], False, 0, r32)[0]
        return (*attend(q, store(k), store(v), self.D ** -0.5), n)


@pytest.mark.parametrize("cache", ["f16", "bf16", "q8"])
@pytest.mark.parametrize("graph", [False, True])
def test_decoder_steps(gpu, cache, graph):
    """Twenty steps of three sequences with pages filling up, eager and replayed from one captured graph. The table
    is within 2 ulp of the oracle's, which moves a rotated key by 4 w and now and then a stored value by one step."""
    d = _Gqa(cache)
    for i, out in enumerate(run_decode(d, d.steps, graph)):
        for b in range(d.B):
            want, _, vabs, big, n = d.want(i, b, cache)
            step = {"f16": 2.0 ** -10, "bf16": 2.0 ** -7, "q8": 1 / 100}[cache]
            err = (out[b].double() - want).abs()
            assert (err <= (2 * (step / 8 + 160 * W) * big[:, None] + 2.0 ** -20) * vabs).all(), (i, b)
            assert err.norm() <= 1e-3 * want.norm()


def test_latent_decoder_steps_with_rotation_and_prompt(gpu):
    """A latent prompt written in one call, then single tokens; several query tokens of one sequence by a shared table."""
    g = gen(31)
    H, R, dr, dn, dv, pt, n0, steps = 8, 512, 64, 64, 64, 16, 37, 5
    freqs, a = hb.rope_freqs(dr, 1e4, scaling="yarn", factor=4.0)
    cs = hb.rope_table(freqs, 64, factor=a)
    table, total = table_of(g, [n0 + steps], pt)
    cp = pool(g, total, 1, pt, R + dr, "bf16")[0].cuda()
    rows = randn(g, n0 + steps, 1, R + dr)
    w, q = randn(g, H, dn + dv, R, scale=0.05, dtype=torch.bfloat16), randn(g, n0 + steps, H, dn + dr, dtype=torch.bfloat16)
    td = table.cuda()
    i32 = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    hb.kv_write(rows[:n0].cuda(), None, cp, None, td, i32(0, n0), i32(0), cs=cs, interleaved=True, offset=R)
    for i in range(steps):
        hb.kv_write(rows[n0 + i:n0 + i + 1].cuda(), None, cp, None, td, i32(0, 1), i32(n0 + i), cs=cs, interleaved=True, offset=R)
    n = n0 + steps
    pos = torch.arange(n, dtype=torch.int32).cuda()
    qr = hb.rope(q.cuda(), pos, cs, interleaved=True, offset=dn)
    out = hb.latent_attention(qr, w.cuda(), cp, td.expand(n, -1), pos + 1, scale=0.1).cpu()
    cos, sin = cs[..., 0].cpu().double(), cs[..., 1].cpu().double()
    c = rotate(rows.double(), cos[:n], sin[:n], True, R, r32).to(torch.bfloat16).double()
    qq = rotate(q.double(), cos[:n], sin[:n], True, dn, r32).to(torch.bfloat16).double()
    for t in range(n):
        qa = torch.einsum("hd,hdr->hr", qq[t, :, :dn], w[:, :dn].double())
        o, _, _, _ = attend(torch.cat([qa, qq[t, :, dn:]], -1), c[:t + 1], c[:t + 1, :, :R], 0.1)
        want = torch.einsum("hr,hvr->hv", o, w[:, dn:].double())
        assert (out[t].double() - want).norm() <= 4 * half_step(torch.bfloat16) * want.norm(), t


def test_two_streams_and_two_graphs_at_once(gpu):
    """Calls on two streams at once, and two captured graphs replayed side by side, each with its own scratch."""
    cases = []
    for seed in (40, 41):
        g = gen(seed)
        (kp, _), (vp, _) = (f := filled(g, [3000, 10], 2, 64, 64, "bf16"))[0]
        q = randn(g, 2, 8, 64, dtype=torch.bfloat16).cuda()
        cases.append((q, kp.cuda(), vp.cuda(), f[1].cuda(), torch.tensor([3000, 10], dtype=torch.int32).cuda()))
    want = [hb.decode_attention(*c, scale=0.1) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(20):
        got = []
        for c, s in zip(cases, streams):
            got.append(hb.decode_attention(*c, scale=0.1, stream=s, out=torch.empty_like(c[0])))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs, outs = [], []
    for c in cases:
        G = torch.cuda.CUDAGraph()
        with torch.cuda.graph(G):
            outs.append(hb.decode_attention(*c, scale=0.1))
        graphs.append(G)
    for _ in range(20):
        for G, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                G.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_calls_on_another_stream_allocate_there(gpu):
    """Outputs and scratch that a call makes itself are usable on the stream it was given, with no other synchronisation."""
    g = gen(50)
    (kp, _), (vp, _) = (f := filled(g, [500, 77], 2, 16, 64, "bf16"))[0]
    q = randn(g, 2, 8, 64, dtype=torch.bfloat16).cuda()
    args = (q, kp.cuda(), vp.cuda(), f[1].cuda(), torch.tensor([500, 77], dtype=torch.int32).cuda())
    cs = hb.rope_table(hb.rope_freqs(64, 1e4)[0], 100)
    pos = torch.tensor([3, 99], dtype=torch.int32).cuda()
    want = hb.decode_attention(*args, scale=0.1, return_lse=True), hb.rope(q, pos, cs)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    for stream in (s, s.cuda_stream):
        junk = torch.full((1 << 24,), float("nan")).cuda()      # work on the current stream whose memory is freed at once
        del junk
        got = hb.decode_attention(*args, scale=0.1, return_lse=True, stream=stream)
        rot = hb.rope(q, pos, cs, stream=stream)
        table = hb.rope_table(hb.rope_freqs(64, 1e4)[0], 100, stream=stream)
        s.synchronize()
        assert torch.equal(got[0], want[0][0]) and torch.equal(got[1], want[0][1]) and torch.equal(rot, want[1]) and torch.equal(table, cs)
        torch.cuda.synchronize()


@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_latent_attention_captured(gpu, cache):
    """One captured call follows new queries, rows, lengths and pages in the same buffers; the scratch is used again and again."""
    g = gen(51)
    pools, table, (rows,) = filled(g, [150, 70, 9], 1, 16, 320, cache, sides=1)
    cp, cs = (cu(t) for t in pools[0])
    w, td = randn(g, 8, 64, 256, dtype=torch.bfloat16, scale=0.06).cuda(), table.cuda()
    q, lens = torch.zeros(3, 8, 96, dtype=torch.bfloat16).cuda(), torch.zeros(3, dtype=torch.int32).cuda()
    hb.latent_attention(q, w, cp, td, lens, scale=0.1, c_scale=cs)
    G = torch.cuda.CUDAGraph()
    with torch.cuda.graph(G):
        out = hb.latent_attention(q, w, cp, td, lens, scale=0.1, c_scale=cs)
    for i, ls in enumerate([[150, 70, 9], [1, 0, 2], [64, 65, 1], [149, 70, 0], [0, 0, 0]]):
        q.copy_(randn(g, 3, 8, 96, dtype=torch.bfloat16))
        lens.copy_(torch.tensor(ls, dtype=torch.int32))
        G.replay()
        assert torch.equal(out, hb.latent_attention(q, w, cp, td, lens, scale=0.1, c_scale=cs)), i
        for b, n in enumerate(ls):
            if n == 0:
                assert (out[b] == 0).all()
                continue
            qc = q[b].cpu().double()
            qa = torch.cat([torch.einsum("hd,hdr->hr", qc[:, :32], w.cpu()[:, :32].double()), qc[:, 32:]], -1)
            o, _, _, _ = attend(qa, rows[b][:n], rows[b][:n, :, :256], 0.1)
            want = torch.einsum("hr,hvr->hv", o, w.cpu()[:, 32:].double())
            assert (out[b].cpu().double() - want).norm() <= 4 * half_step(torch.bfloat16) * want.norm()


def test_workspace_sizes(gpu):
    """The sizes the size functions give are enough, and no fewer bytes are taken."""
    g = gen(52)
    for cache in ("bf16", "q8"):
        (kp, ks), (vp, vs) = (f := filled(g, [40], 2, 16, 64, cache))[0]
        args = (randn(g, 1, 8, 64, dtype=torch.bfloat16).cuda(), kp.cuda(), vp.cuda(), f[1].cuda(), torch.tensor([40], dtype=torch.int32).cuda())
        n = hb.attention_workspace(1, 8, 2, 64)
        kw = dict(scale=0.1, k_scale=cu(ks), v_scale=cu(vs))
        a = hb.decode_attention(*args, workspace=torch.zeros(n, dtype=torch.uint8).cuda(), **kw)
        assert torch.equal(a, hb.decode_attention(*args, **kw))
        with pytest.raises(ValueError):
            hb.decode_attention(*args, workspace=torch.zeros(n - 16, dtype=torch.uint8).cuda(), **kw)
    assert hb.latent_workspace(4, 16, 512, 64) > 4 * 16 * 576 * 4


# ----------------------------------------------------------------------------------------- the edges of the calls

@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_offsets_past_32_bits(gpu, cache):
    """Pages at the far end of a pool of more than 2^31 elements: the same bits as from its first pages."""
    g = gen(60)
    pt, D, lens = 64, 128, [300, 129, 64]
    n_pages = (1 << 31) // (pt * D) + 40
    dt = torch.int8 if cache == "q8" else torch.bfloat16
    kp, vp = (torch.empty(n_pages, 1, pt, D, dtype=dt, device="cuda") for _ in range(2))
    ks, vs = (torch.empty(n_pages, 1, pt, D // 64, device="cuda") if cache == "q8" else None for _ in range(2))
    near = torch.tensor([[0, 3, 1, 2, 4], [5, 7, 6, -1, -1], [8, -1, -1, -1, -1]], dtype=torch.int32)
    far = torch.where(near >= 0, n_pages - 1 - near, near)
    k, v = (randn(g, sum(lens), 1, D).cuda() for _ in range(2))
    q = randn(g, 3, 8, D, dtype=torch.bfloat16).cuda()
    start = torch.tensor([0, 300, 429, 493], dtype=torch.int32).cuda()
    zero, n = torch.zeros(3, dtype=torch.int32).cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    got = []
    for table in (near.cuda(), far.cuda()):
        hb.kv_write(k, v, kp, vp, table, start, zero, k_scale=ks, v_scale=vs)
        ko, vo = torch.zeros_like(k), torch.zeros_like(v)
        hb.kv_read(kp, vp, table, start, zero, ko, vo, k_scale=ks, v_scale=vs)
        got.append((ko, vo, *hb.decode_attention(q, kp, vp, table, n, scale=0.09, k_scale=ks, v_scale=vs, return_lse=True)))
    for a, b in zip(*got):
        assert torch.equal(a, b) and torch.isfinite(a).all()
    assert (got[1][0] - k).abs().max() <= (k.abs().max() / 127 if cache == "q8" else half_step(torch.bfloat16) * k.abs().max())
    del kp, vp
    w = randn(g, 4, 64, 128, dtype=torch.bfloat16, scale=0.08).cuda()
    n_pages = (1 << 31) // (pt * 192) + 40
    cp = torch.empty(n_pages, 1, pt, 192, dtype=dt, device="cuda")
    cs = torch.empty(n_pages, 1, pt, 3, device="cuda") if cache == "q8" else None
    far = torch.where(near >= 0, n_pages - 1 - near, near)
    c, ql = randn(g, sum(lens), 1, 192).cuda(), randn(g, 3, 4, 32 + 64, dtype=torch.bfloat16).cuda()
    got = []
    for table in (near.cuda(), far.cuda()):
        hb.kv_write(c, None, cp, None, table, start, zero, k_scale=cs)
        got.append(hb.latent_attention(ql, w, cp, table, n, scale=0.1, c_scale=cs))
    assert torch.equal(*got) and torch.isfinite(got[0]).all()


def test_rows_of_many_sequences(gpu):
    """More sequences than a CTA's threads, most of them without a row, padding at both ends; the table of one page each."""
    g = gen(61)
    B, pt = 1500, 4
    count = torch.randint(-3, 4, (B,), generator=g).clamp(min=0)
    start = torch.cat([torch.zeros(1, dtype=torch.int64), count.cumsum(0)]) + 5
    T = int(start[-1]) + 7
    pages = torch.randperm(B, generator=g).to(torch.int32)
    x = randn(g, T, 1, 64)
    cp = torch.full((B, 1, pt, 64), 9.0, dtype=torch.bfloat16)
    want = cp.clone()
    for b in range(B):
        for i in range(int(count[b])):
            want[pages[b], 0, i] = x[int(start[b]) + i, 0].to(torch.bfloat16)
    dev, st, p0 = cp.cuda(), start.to(torch.int32).cuda(), torch.zeros(B, dtype=torch.int32).cuda()
    hb.kv_write(x.cuda(), None, dev, None, pages[:, None].cuda(), st, p0)
    assert torch.equal(dev.cpu(), want)
    out = torch.full((T, 1, 64), 3.0).cuda()
    hb.kv_read(dev, None, pages[:, None].cuda(), st, p0, out, None)
    ref = torch.full((T, 1, 64), 3.0)
    ref[5:T - 7] = x[5:T - 7].to(torch.bfloat16).float()
    assert torch.equal(out.cpu(), ref)


@pytest.mark.parametrize("cache", ["bf16", "q8"])
def test_lengths_out_of_range(gpu, cache):
    """Negative lengths are empty, ones past the table give NaN, whatever else is in the batch; a table without pages."""
    g = gen(62)
    lens = [40, -7, 33, 40, -2 ** 31, 2 ** 31 - 1]
    pools, table, _ = filled(g, [40] * 6, 1, 8, 192, cache)
    (kp, ks), (vp, vs) = ((cu(a), cu(b)) for a, b in pools)
    t, n = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    t4 = t[:, :4]                                       # rows of 32 positions only: 33 and 40 are past them
    q = randn(g, 6, 4, 192, dtype=torch.bfloat16).cuda()
    w = randn(g, 4, 48 + 16, 128, dtype=torch.bfloat16, scale=0.1).cuda()
    ql = randn(g, 6, 4, 48 + 64, dtype=torch.bfloat16).cuda()
    att = lambda tb, ln: hb.decode_attention(q, kp, vp, tb, ln, scale=0.1, k_scale=ks, v_scale=vs, return_lse=True)  # noqa: E731
    lat = lambda tb, ln: hb.latent_attention(ql, w, kp, tb, ln, scale=0.1, c_scale=ks)  # noqa: E731
    for b in range(6):
        alone = torch.zeros(6, dtype=torch.int32).cuda()
        alone[b] = lens[b]
        assert torch.equal(att(t, n)[0][b].view(torch.int16), att(t, alone)[0][b].view(torch.int16)) or lens[b] > 0
    out, lse = att(t, n)
    lo = lat(t, n)
    assert torch.isfinite(out[[0, 2, 3]]).all() and torch.isfinite(lse[[0, 2, 3]]).all() and torch.isfinite(lo[[0, 2, 3]]).all()
    assert (out[[1, 4]] == 0).all() and (lse[[1, 4]] == -math.inf).all() and (lo[[1, 4]] == 0).all()
    assert torch.isnan(out[5]).all() and torch.isnan(lse[5]).all() and torch.isnan(lo[5]).all()
    out, lse = att(t4, n)
    lo = lat(t4, n)
    assert torch.isnan(out[[0, 2, 3, 5]]).all() and torch.isnan(lo[[0, 2, 3, 5]]).all() and (out[[1, 4]] == 0).all() and (lo[[1, 4]] == 0).all()
    t0 = torch.empty(6, 0, dtype=torch.int32).cuda()
    out, lse = att(t0, n)
    lo = lat(t0, n)
    assert torch.isnan(out[[0, 2, 3, 5]]).all() and torch.isnan(lo[[0, 2, 3, 5]]).all() and (out[[1, 4]] == 0).all() and (lo[[1, 4]] == 0).all()


@pytest.mark.parametrize("cache,R,H", [("bf16", 128, 16), ("q8", 512, 64), ("bf16", 512, 130), ("f16", 256, 8)])
def test_latent_calls_in_a_row_and_side_by_side(gpu, cache, R, H):
    """Many calls without a wait in between, one scratch, other queries and lengths each time; then on two streams at once."""
    g = gen(63)
    W, pt, B = R + 64, 64, 7
    pages = 40
    if cache == "q8":
        cp, cs = torch.randint(-127, 128, (pages, 1, pt, W), generator=g).to(torch.int8), torch.rand((pages, 1, pt, W // 64), generator=g) / 64
        x = torch.bfloat16
    else:
        cp, cs, x = randn(g, pages, 1, pt, W, dtype=F[cache]), None, F[cache]
    cp, cs = cp.cuda(), cu(cs)
    w = randn(g, H, 64 + 64, R, dtype=x, scale=R ** -0.5).cuda()
    table = torch.randint(0, pages, (B, 60), generator=g, dtype=torch.int32).cuda()
    lens = [torch.tensor(v, dtype=torch.int32).cuda() for v in
            ([3000, 1, 0, 64, 65, 700, 128], [0, 0, 0, 0, 0, 0, 3], [3840] * 7, [64] * 7, [1, 2, 3, 4, 5, 6, 3840], [0] * 7)]
    qs = [randn(g, B, H, 64 + 64, dtype=x).cuda() for _ in range(6)]
    call = lambda i, **kw: hb.latent_attention(qs[i % 6], w, cp, table, lens[(i + i // 6) % 6], scale=0.09, c_scale=cs, **kw)  # noqa: E731
    want = []
    for i in range(36):
        want.append(call(i))
        torch.cuda.synchronize()
        assert torch.isfinite(want[-1]).all()
    ws = torch.empty(hb.latent_workspace(B, H, R, 64), dtype=torch.uint8, device="cuda")
    outs = [torch.empty_like(want[0]) for _ in range(36)]
    for _ in range(3):
        for o in outs:
            o.fill_(9.0)
        for i in range(36):
            call(i, workspace=ws, out=outs[i])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    got = [call(i, stream=(a, b)[i % 2]) for i in range(36)]
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_attention_calls_in_a_row(gpu):
    """Many calls without a wait in between on one scratch, from one CTA's work to all."""
    g = gen(64)
    kp, vp = (randn(g, 60, 2, 32, 128, dtype=torch.bfloat16).cuda() for _ in range(2))
    table = torch.randint(0, 60, (5, 100), generator=g, dtype=torch.int32).cuda()
    lens = [torch.tensor(v, dtype=torch.int32).cuda() for v in ([3200] * 5, [0, 1, 0, 0, 0], [3000, 17, 64, 65, 0], [0] * 5, [1, 2, 3, 4, 5])]
    q = [randn(g, 5, 16, 128, dtype=torch.bfloat16).cuda() for _ in range(4)]
    ws = torch.empty(hb.attention_workspace(5, 16, 2, 128), dtype=torch.uint8, device="cuda")
    want = []
    for i in range(20):
        want.append(hb.decode_attention(q[i % 4], kp, vp, table, lens[i % 5], scale=0.09))
        torch.cuda.synchronize()
    for _ in range(5):
        got = [hb.decode_attention(q[i % 4], kp, vp, table, lens[i % 5], scale=0.09, workspace=ws) for i in range(20)]
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_calls_that_are_refused(gpu):
    """Outputs that are the queries themselves, more sequences than a launch takes, a stream of nowhere."""
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device="cuda")  # noqa: E731
    i32 = torch.int32
    kc = z(2, 1, 16, 64)
    q = z(2, 4, 64)
    with pytest.raises(ValueError, match="in place"):
        hb.decode_attention(q, kc, kc, z(2, 1, dtype=i32), z(2, dtype=i32), scale=1.0, out=q)
    with pytest.raises(ValueError, match="65535"):
        hb.decode_attention(z(65536, 1, 64), kc, kc, z(65536, 1, dtype=i32), z(65536, dtype=i32), scale=1.0)
    cl = z(1, 1, 16, 192)
    ql = z(2, 4, 32 + 64)
    with pytest.raises(ValueError, match="in place"):
        hb.latent_attention(ql, z(4, 32 + 96, 128), cl, z(2, 1, dtype=i32), z(2, dtype=i32), scale=1.0, out=ql)
    with pytest.raises(ValueError, match="65535"):
        hb.latent_attention(z(65536, 1, 32 + 64), z(1, 48, 128), cl, z(65536, 1, dtype=i32), z(65536, dtype=i32), scale=1.0)


@pytest.mark.parametrize("cache", ["bf16", "f16", "q8"])
@pytest.mark.parametrize("H", [4, 128])
def test_latent_batch_with_rows_out_of_range(gpu, cache, H):
    """Sequences that cannot be read between ones that can, with few heads (a sequence's pieces joined by several warps) and
    many (a warp a sequence): zeros, NaN, and the others as without them."""
    g = gen(65)
    lens = [40, -3, 33, 10 ** 6, 64, 0, 1, 130, 65, 17, 200, 5, 129]
    x = "f16" if cache == "f16" else "bf16"
    pools, table, (rows,) = filled(g, [max(0, min(n, 200)) for n in lens], 1, 16, 320, cache, sides=1)
    table[7, 4] = 10 ** 6                                    # no such page
    cp, cs = (cu(t) for t in pools[0])
    q, w = randn(g, 13, H, 64 + 64, dtype=F[x]), randn(g, H, 64 + 128, 256, dtype=F[x], scale=0.06)
    out = hb.latent_attention(q.cuda(), w.cuda(), cp, table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), scale=0.09, c_scale=cs).cpu()
    assert (out[[1, 5]] == 0).all() and torch.isnan(out[[3, 7]]).all()
    for b in (0, 2, 4, 6, 8, 9, 10, 11, 12):
        qd, wd = q[b].double(), w.double()
        qa = torch.cat([torch.einsum("hd,hdr->hr", qd[:, :64], wd[:, :64]), qd[:, 64:]], -1)
        o, _, _, _ = attend(qa, rows[b], rows[b][..., :256], 0.09)
        want = torch.einsum("hr,hvr->hv", o, wd[:, 64:])
        # in the 2-norm at most the half steps of the queries, the weights and the output as operands together
        assert (out[b].double() - want).norm() <= 4 * half_step(torch.bfloat16 if cache == "q8" else F[x]) * want.norm(), b


def test_rope_table_of_any_frequencies(gpu):
    """Frequencies of more than a turn, tiny, negative and zero ones, at positions of either sign."""
    f = torch.tensor([0.0, 1.0, -1.0, 6.5, -300.25, 1e-7, -1e-7, 1e-12, 2 * math.pi, 3e-3, 0.5, 1e4], dtype=torch.float64)
    for first in (-2 ** 31 + 1, -5, 0, 2 ** 31 - 40):
        got = hb.rope_table(f.numpy(), 40, first=first).cpu().double()
        ang = torch.arange(first, first + 40, dtype=torch.float64)[:, None] * f
        want = torch.stack([ang.cos(), ang.sin()], -1)
        # 2 ulp of the value (4 half steps), and the 64-bit phase: angle * 2^-52, each side's
        tol = 4 * W * want.abs() + (ang.abs() * 2.0 ** -51)[..., None] + 2.0 ** -40
        assert (got - want).abs().le(tol).all(), (first, ((got - want).abs() / tol).max())
