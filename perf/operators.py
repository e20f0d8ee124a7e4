"""What the device-side attention operators are measured on: rotary positions, the paged key-value cache
(written, quantised, read back), decode attention over its pages, and latent attention (absorbed form).

``run`` computes an operator in its plain form (elementary torch operations in 32 bits) or, where ``own``
is true, through hearth_b200's entry points; ``exact`` computes it from its definition in 64 bits.
"""
import math
import random

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
DEV = "cuda"


# --------------------------------------------------------------------------------------- the cases

def listed():
    return [
        # One decode step of 3 streams: 32 query heads of 128 (the Qwen3-30B-A3B shape); latency counts.
        dict(name="rope_decode", op="rope", T=3, H=32, D=128, rot=128, off=0, inter=False, x="bf16", y="bf16",
             n_pos=40960, first=511, pad=0),
        # A prompt chunk of latent-attention queries: 64 heads of 128 + 64, the last 64 rotated in interleaved
        # pairs at far positions, f32 projections (rows of a wider buffer) rounded to bf16 on the way out.
        dict(name="rope_prompt_tail", op="rope", T=4099, H=64, D=192, rot=64, off=128, inter=True, x="f32", y="bf16",
             n_pos=131072, first=120000, pad=64),
        # The table of a model opened for 131072 positions with frequencies scaled for long contexts.
        dict(name="rope_table_scaled", op="table", rot=128, n_pos=131072, first=0, theta=1e6, kind="yarn", factor=32.0),
        # One decode step of 64 streams into a Q8 cache of 4 heads of 128, keys rotated as they are written,
        # and the new rows read back.
        dict(name="kv_decode_q8", op="kv", B=64, n_new=1, Hkv=4, D=128, pt=64, cache="q8", x="f32", y="f32", rot=128,
             off=0, inter=False, past=3000, latent=False),
        # Ragged prompts of 8 streams, 8 heads of 128, from bf16 into a Q8 cache, and read back to bf16.
        dict(name="kv_prompt_q8", op="kv", B=8, n_new=4096, Hkv=8, D=128, pt=64, cache="q8", x="bf16", y="bf16",
             rot=0, off=0, inter=False, past=130, latent=False),
        # Ragged prompts into a bf16 latent cache (512 + 64 values a token, the 64 rotated in pairs).
        dict(name="kv_prompt_latent", op="kv", B=5, n_new=3001, Hkv=1, D=576, pt=32, cache="bf16", x="f32", y="bf16",
             rot=64, off=512, inter=True, past=77, latent=True),
        # One stream, 16 heads each with its own keys and values (the OLMoE-1B-7B shape), a short context, f32
        # activations over an f16 cache.
        dict(name="attn_one_short", op="attn", B=1, L=777, H=16, Hkv=16, D=128, pt=16, cache="f16", x="f32"),
        # 48 streams of uneven lengths (one just opened, empty), 8 query heads to a key head, Q8 cache.
        dict(name="attn_batch_q8", op="attn", B=48, L=6011, H=32, Hkv=4, D=128, pt=64, cache="q8", x="bf16"),
        # One stream with a very long context: the work is split over the cache's length.
        dict(name="attn_one_long", op="attn", B=1, L=262147, H=32, Hkv=4, D=128, pt=64, cache="bf16", x="bf16"),
        # One stream of latent attention, 64 heads (the Kimi-K2 shape), a context of a few pages.
        dict(name="latent_one", op="latent", B=1, L=1531, H=64, R=512, dr=64, dn=128, dv=128, pt=64, cache="bf16",
             x="bf16"),
        # 32 streams of uneven lengths, the same shape.
        dict(name="latent_batch", op="latent", B=32, L=8191, H=64, R=512, dr=64, dn=128, dv=128, pt=64, cache="bf16",
             x="bf16"),
        # A GPU's share of the heads (16 of 64) over a long Q8 latent cache.
        dict(name="latent_long_q8", op="latent", B=4, L=65536, H=16, R=512, dr=64, dn=128, dv=128, pt=128, cache="q8",
             x="bf16"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    op = rng.choice(["rope", "table", "kv", "attn", "attn", "latent"])
    if op == "rope":
        D = rng.choice([64, 80, 128, 192, 256])
        rot = rng.choice([D, D // 2, D // 4])
        off = rng.choice([0, D - rot])
        H = rng.choice([1, 4, 16, 28, 32, 64])
        T = _log(rng, 1, min(4099, 4099 * 64 * 192 // (H * D)))
        n_pos = _log(rng, max(T, 2048), 200000)
        return dict(op=op, T=T, H=H, D=D, rot=rot, off=off, inter=rng.random() < 0.5,
                    x=rng.choice(["f32", "f16", "bf16"]), y=rng.choice(["f32", "f16", "bf16"]), n_pos=n_pos,
                    first=rng.randint(0, n_pos - T), pad=rng.choice([0, 0, 8, 72]))
    if op == "table":
        n_pos = _log(rng, 2049, 131072)
        return dict(op=op, rot=rng.choice([32, 64, 80, 128]), n_pos=n_pos, first=_log(rng, 1, 1000000),
                    theta=rng.choice([1e4, 5e5, 1e6]), kind=rng.choice(["none", "linear", "ntk", "yarn"]),
                    factor=rng.choice([2.0, 4.0, 32.0]))
    pt = rng.choice([8, 16, 32, 64, 128])
    if op == "kv":
        latent = rng.random() < 0.25
        cache = rng.choice(["f16", "bf16", "q8", "q8"])
        D = 576 if latent else rng.choice([64, 128, 256] if cache == "q8" else [64, 80, 128, 256])
        B = _log(rng, 1, 64)
        Hkv = 1 if latent else rng.choice([1, 2, 4, 8])
        rot = 64 if latent else rng.choice([0, D, D // 2])
        return dict(op=op, B=B, n_new=_log(rng, 1, max(1, 16384 * 1024 // (B * max(1024, Hkv * D)))), Hkv=Hkv, D=D, pt=pt, cache=cache, x=rng.choice(["f32", "f16", "bf16"]), y=rng.choice(["f32", "f16", "bf16"]),
                    rot=rot, off=512 if latent else 0, inter=rng.random() < 0.5, past=_log(rng, 1, 4000),
                    latent=latent)
    B = _log(rng, 1, 64)
    if op == "attn":
        cache = rng.choice(["f16", "bf16", "q8"])
        H, Hkv = rng.choice([(32, 4), (16, 16), (32, 8), (8, 1), (24, 2), (14, 2), (64, 4)])
        D = rng.choice([64, 128, 256] if cache == "q8" else [64, 80, 128, 256])
        L = _log(rng, 1, min(262147, 262147 * 512 // (B * Hkv * D)))
        return dict(op=op, B=B, L=L, H=H, Hkv=Hkv, D=D, pt=pt, cache=cache, x=rng.choice(["f32", "f16", "bf16"]))
    t = rng.choice(["f16", "bf16"])
    H = rng.choice([8, 16, 40, 64, 128])
    return dict(op=op, B=B, L=_log(rng, 1, min(65536, 9000000 // (B * H))), H=H, R=rng.choice([256, 512, 512]), dr=64,
                dn=rng.choice([64, 128]), dv=rng.choice([64, 128]), pt=pt, cache=rng.choice([t, t, "q8"]), x=t)


# --------------------------------------------------------------------------------------- inputs

def _lens(case):
    """The streams' lengths: uneven, the first the longest, one of four or more empty."""
    r = random.Random(case["B"] * 1000003 + case["L"])
    lens = [case["L"]] + [max(1, int(case["L"] * r.uniform(0.1, 1.0))) for _ in range(case["B"] - 1)]
    if case["B"] >= 4:
        lens[case["B"] // 2] = 0
    return lens


def _news(case):
    """(new tokens, tokens already cached) of each stream of a cache case."""
    if case["n_new"] == 1:
        n = [1] * case["B"]
    else:
        r = random.Random(case["B"] * 1000003 + case["n_new"])
        n = [case["n_new"]] + [max(1, int(case["n_new"] * r.uniform(0.1, 1.0))) for _ in range(case["B"] - 1)]
    r = random.Random(case["past"])
    return n, [r.randint(0, case["past"]) for _ in n]


def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _randn(g, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=g, device=DEV) * scale).to(dtype)


def _freqs(case):
    """The frequencies of a case in 64 bits, on the CPU, and the factor on the values, from the definitions."""
    n = case["rot"] // 2
    theta, kind, s = case.get("theta", 1e4), case.get("kind", "none"), case.get("factor", 1.0)
    if kind == "ntk":
        theta = theta * s ** (case["rot"] / (case["rot"] - 2))
    f = theta ** (-torch.arange(n, dtype=torch.float64) * 2 / case["rot"])
    if kind == "linear":
        return f / s, 1.0
    if kind == "yarn":
        turns = torch.tensor([32.0, 1.0], dtype=torch.float64)   # fast, slow; 4096 positions of training
        lo, hi = (case["rot"] * torch.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(theta))).tolist()
        lo, hi = max(math.floor(lo), 0), min(math.ceil(hi), case["rot"] - 1)
        ramp = ((torch.arange(n, dtype=torch.float64) - lo) / max(hi - lo, 0.001)).clamp(0, 1)
        return f * (1 - ramp) + f / s * ramp, 0.1 * math.log(s) + 1.0
    return f, 1.0


def _angles(freqs, first, n_pos):
    p = torch.arange(first, first + n_pos, dtype=torch.float64, device=DEV)
    return p[:, None] * freqs.to(DEV)[None, :]


def _table64(freqs, first, n_pos, factor=1.0):
    a = _angles(freqs, first, n_pos)
    return torch.stack([torch.cos(a) * factor, torch.sin(a) * factor], dim=-1)


def _pages(lens, pt, g):
    """A page table over a shuffled pool with a few pages to spare; entries past a stream's end are -1."""
    need = [-(-n // pt) for n in lens]
    total = sum(need) + 3
    perm = torch.randperm(total, generator=g, device=DEV).to(torch.int32)
    width = max(1, max(need))
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n]
        at += n
    return table, total


def _live(table, lens_t, pt, total):
    """[pages, slots]: the slots that hold a token."""
    width = table.shape[1]
    p = torch.arange(width * pt, device=DEV)
    rows, cols = torch.nonzero(p[None, :] < lens_t[:, None], as_tuple=True)
    live = torch.zeros(total * pt, dtype=torch.bool, device=DEV)
    live[table[rows, cols // pt].long() * pt + cols % pt] = True
    return live.view(total, pt)


def _pool(g, total, Hkv, pt, D, cache, live):
    """One pool of rows (and their scales): the tokens' values, NaN wherever no token is."""
    dead = ~live[:, None, :, None]
    if cache == "q8":
        codes = (torch.randn((total, Hkv, pt, D), generator=g, device=DEV, dtype=torch.bfloat16) * 42).clamp_(-127, 127)
        scale = (0.5 + torch.rand((total, Hkv, pt, D // 64), generator=g, device=DEV)) / 42
        return codes.round_().to(torch.int8), scale.masked_fill_(dead, float("nan"))
    x = torch.randn((total, Hkv, pt, D), generator=g, device=DEV, dtype=DTYPES[cache])
    return x.masked_fill_(dead, float("nan")), None


def prepare(case, seed):
    g = _gen(seed)
    op = case["op"]
    s = dict(case=case)
    if op == "table":
        freqs, factor = _freqs(case)
        # the angles' scale comes from the model's configuration: another seed, another model
        s["theta"] = case["theta"] * (1 + 0.01 * (seed % 97))
        freqs, factor = _freqs(dict(case, theta=s["theta"]))
        s["freqs"], s["factor"] = freqs, factor
        return s
    if op in ("rope", "kv") and case["rot"]:
        n_pos = case["n_pos"] if op == "rope" else max(a + b for a, b in zip(*_news(case)))
        s["cs"] = _table64(_freqs(case)[0], 0, n_pos).float().contiguous()
    if op == "rope":
        wide = _randn(g, (case["T"], case["H"] * case["D"] + case["pad"]), DTYPES[case["x"]])
        s["x"] = wide[:, :case["H"] * case["D"]].view(case["T"], case["H"], case["D"])
        s["pos"] = case["first"] + torch.arange(case["T"], dtype=torch.int32, device=DEV)
        s["y"] = torch.empty((case["T"], case["H"], case["D"]), dtype=DTYPES[case["y"]], device=DEV)
        return s
    if op == "kv":
        n, past = _news(case)
        lens = [a + b for a, b in zip(n, past)]
        s["table"], total = _pages(lens, case["pt"], g)
        start = [0]
        for k in n:
            start.append(start[-1] + k)
        s["start"] = torch.tensor(start, dtype=torch.int32, device=DEV)
        s["pos0"] = torch.tensor(past, dtype=torch.int32, device=DEV)
        live = _live(s["table"], torch.tensor(lens, device=DEV), case["pt"], total)
        shape = (start[-1], case["Hkv"], case["D"])
        for name in ("k",) if case["latent"] else ("k", "v"):
            s[name] = _randn(g, shape, DTYPES[case["x"]])
            s[name + "_cache"], s[name + "_scale"] = _pool(g, total, case["Hkv"], case["pt"], case["D"], case["cache"], live)
            s[name + "_out"] = torch.empty(shape, dtype=DTYPES[case["y"]], device=DEV)
        return s
    lens = _lens(case)
    s["table"], total = _pages(lens, case["pt"], g)
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device=DEV)
    live = _live(s["table"], s["lens"], case["pt"], total)
    if op == "attn":
        s["scale"] = case["D"] ** -0.5
        s["q"] = _randn(g, (case["B"], case["H"], case["D"]), DTYPES[case["x"]], 1.5)
        s["k_cache"], s["k_scale"] = _pool(g, total, case["Hkv"], case["pt"], case["D"], case["cache"], live)
        s["v_cache"], s["v_scale"] = _pool(g, total, case["Hkv"], case["pt"], case["D"], case["cache"], live)
    else:
        s["scale"] = (case["dn"] + case["dr"]) ** -0.5
        t = DTYPES[case["x"]]
        s["q"] = _randn(g, (case["B"], case["H"], case["dn"] + case["dr"]), t)
        s["w"] = _randn(g, (case["H"], case["dn"] + case["dv"], case["R"]), t, case["R"] ** -0.5)
        s["c"], s["c_scale"] = _pool(g, total, 1, case["pt"], case["R"] + case["dr"], case["cache"], live)
    return s


# --------------------------------------------------------------------------------------- one pass

def _run_own(s):
    import hearth_b200 as hb
    case, op = s["case"], s["case"]["op"]
    if op == "table":
        freqs, factor = hb.rope_freqs(case["rot"], s["theta"], scaling=case["kind"], factor=case["factor"],
                                      original=4096)
        return hb.rope_table(freqs, case["n_pos"], first=case["first"], factor=factor)
    if op == "rope":
        return hb.rope(s["x"], s["pos"], s["cs"], interleaved=case["inter"], offset=case["off"], out=s["y"])
    if op == "kv":
        v = not case["latent"]
        pools = dict(k_scale=s["k_scale"], v_scale=s["v_scale"] if v else None)
        vc = s["v_cache"] if v else None
        hb.kv_write(s["k"], s["v"] if v else None, s["k_cache"], vc, s["table"], s["start"], s["pos0"],
                    cs=s.get("cs"), interleaved=case["inter"], offset=case["off"], **pools)
        hb.kv_read(s["k_cache"], vc, s["table"], s["start"], s["pos0"], s["k_out"], s["v_out"] if v else None, **pools)
        return (s["k_out"], s["v_out"]) if v else s["k_out"]
    if op == "attn":
        return hb.decode_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], scale=s["scale"],
                                   k_scale=s["k_scale"], v_scale=s["v_scale"], return_lse=True)
    return hb.latent_attention(s["q"], s["w"], s["c"], s["table"], s["lens"], scale=s["scale"], c_scale=s["c_scale"])


def _rotate(x, cs, inter, off):
    """x [T, heads, D] in f32 with its values [off, off + rot) rotated by cs [T, rot / 2, 2]."""
    rot = 2 * cs.shape[1]
    r = x[..., off:off + rot]
    a, b = (r[..., 0::2], r[..., 1::2]) if inter else (r[..., :rot // 2], r[..., rot // 2:])
    c, s = cs[:, None, :, 0], cs[:, None, :, 1]
    na, nb = a * c - b * s, b * c + a * s
    y = x.clone()
    if inter:
        y[..., off:off + rot:2], y[..., off + 1:off + rot:2] = na, nb
    else:
        y[..., off:off + rot // 2], y[..., off + rot // 2:off + rot] = na, nb
    return y


def _places(s):
    """Page, slot and position of every row of a cache case."""
    t = torch.arange(s["k"].shape[0], device=DEV)
    b = torch.searchsorted(s["start"][1:].long(), t, right=True)
    pos = s["pos0"].long()[b] + t - s["start"].long()[b]
    pt = s["case"]["pt"]
    return s["table"][b, pos // pt].long(), pos % pt, pos


def _codes(x):
    """The Q8 codes and scales of blocks of 64 (the activation blocks' rule)."""
    blk = x.view(*x.shape[:-1], x.shape[-1] // 64, 64)
    # by a tensor: a Python number on the right becomes a product with the rounded 1 / 127 on a GPU, a scale in twenty off by an ulp
    d = blk.abs().amax(-1) / torch.full((), 127.0, device=x.device)
    inv = torch.where(d != 0, 1.0 / d, torch.zeros_like(d))
    return (blk * inv[..., None]).clamp(-127, 127).round().to(torch.int8).view(x.shape), d


def _run_kv(s):
    case = s["case"]
    page, slot, pos = _places(s)

    def one(name, rotate):
        x, pool, scale = s[name].float(), s[name + "_cache"], s[name + "_scale"]
        if rotate:
            x = _rotate(x, s["cs"][pos], case["inter"], case["off"])
        if scale is None:
            pool[page, :, slot] = x.to(pool.dtype)
            s[name + "_out"].copy_(pool[page, :, slot])
        else:
            pool[page, :, slot], scale[page, :, slot] = _codes(x)
            rows = pool[page, :, slot].float().view(*x.shape[:-1], -1, 64) * scale[page, :, slot][..., None]
            s[name + "_out"].copy_(rows.view(x.shape))
        return s[name + "_out"]

    k = one("k", bool(case["rot"]))
    return k if case["latent"] else (k, one("v", False))


def _rows(pool, scale, table):
    """The rows of every stream's pages in f32: [B, Hkv, positions, D]."""
    at = table.clamp(min=0).long()
    x = pool[at].float()                                   # [B, pages, Hkv, pt, D]
    if scale is not None:
        x = (x.view(*x.shape[:-1], -1, 64) * scale[at][..., None]).view(x.shape)
    B, P, Hkv, pt, D = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, P * pt, D)


def _attend(q, k, v, lens, scale):
    """Softmax attention of q [B, Hkv, G, D] over the first lens rows; an empty stream gives zeros, -inf."""
    live = torch.arange(k.shape[2], device=DEV)[None, :] < lens[:, None]
    sc = (q @ k.transpose(-1, -2)) * scale
    sc = sc.masked_fill(~live[:, None, None, :], float("-inf"))
    m = sc.amax(-1, keepdim=True)
    m = torch.where(torch.isinf(m), torch.zeros_like(m), m)
    p = torch.exp(sc - m)
    l = p.sum(-1, keepdim=True)
    o = p @ v.masked_fill(~live[:, None, :, None], 0.0)
    return torch.where(l > 0, o / l, torch.zeros_like(o)), (m + torch.log(l))[..., 0]


def run(state):
    s = state
    if own:
        return _run_own(s)
    case, op = s["case"], s["case"]["op"]
    if op == "table":
        a = _angles(s["freqs"], case["first"], case["n_pos"])
        return (torch.stack([torch.cos(a), torch.sin(a)], dim=-1) * s["factor"]).float()
    if op == "rope":
        s["y"].copy_(_rotate(s["x"].float(), s["cs"][s["pos"].long()], case["inter"], case["off"]))
        return s["y"]
    if op == "kv":
        return _run_kv(s)
    if op == "attn":
        q = s["q"].float().view(case["B"], case["Hkv"], -1, case["D"])
        o, lse = _attend(q, _rows(s["k_cache"], s["k_scale"], s["table"]), _rows(s["v_cache"], s["v_scale"], s["table"]),
                         s["lens"], s["scale"])
        return o.reshape(s["q"].shape).to(s["q"].dtype), lse.reshape(case["B"], case["H"])
    dn, R = case["dn"], case["R"]
    q, w = s["q"].float(), s["w"].float()
    qa = torch.cat([torch.einsum("bhd,hdr->bhr", q[..., :dn], w[:, :dn]), q[..., dn:]], dim=-1)
    c = _rows(s["c"], s["c_scale"], s["table"])
    o, _ = _attend(qa[:, None], c, c[..., :R], s["lens"], s["scale"])
    return torch.einsum("bhr,hvr->bhv", o[:, 0], w[:, dn:]).to(s["q"].dtype)


# --------------------------------------------------------------------------------------- work

def work(case):
    size = {"f32": 4, "f16": 2, "bf16": 2, "q8": 1}
    op = case["op"]
    if op == "table":
        return dict(bytes=case["n_pos"] * case["rot"] * 4, flops=case["n_pos"] * case["rot"] * 40)
    if op == "rope":
        n = case["T"] * case["H"] * case["D"]
        return dict(bytes=n * (size[case["x"]] + size[case["y"]]) + case["T"] * (case["rot"] * 4 + 4),
                    flops=case["T"] * case["H"] * case["rot"] * 3)
    row = lambda D: D * size[case["cache"]] + (D // 64 * 4 if case["cache"] == "q8" else 0)  # noqa: E731
    if op == "kv":
        T = sum(_news(case)[0])
        n = T * case["Hkv"] * (1 if case["latent"] else 2)
        return dict(bytes=n * (case["D"] * (size[case["x"]] + size[case["y"]]) + 2 * row(case["D"])) + T * case["rot"] * 4,
                    flops=n * case["D"] * 8)
    lens = _lens(case)
    n, pages = sum(lens), sum(-(-x // case["pt"]) for x in lens)
    if op == "attn":
        return dict(bytes=n * case["Hkv"] * 2 * row(case["D"]) + 4 * pages
                    + case["B"] * case["H"] * (2 * case["D"] * size[case["x"]] + 4),
                    flops=4 * n * case["H"] * case["D"])
    d = case["dn"] + case["dv"]
    return dict(bytes=n * row(case["R"] + case["dr"]) + 4 * pages + 2 * case["H"] * d * case["R"]
                + case["B"] * case["H"] * (d + case["dr"]) * 2,
                flops=2 * n * case["H"] * (2 * case["R"] + case["dr"]) + 2 * case["B"] * case["H"] * d * case["R"])


# --------------------------------------------------------------------------------------- 64 bits

def _r32(x):
    return x.float().double()


def _turn64(x, cs, inter, off, rnd):
    """The rotation of one block of rows by explicit index lists; rnd rounds each product and sum."""
    half = cs.shape[1]
    j = torch.arange(half, device=x.device)
    ia, ib = (off + 2 * j, off + 2 * j + 1) if inter else (off + j, off + half + j)
    a, b, c, s = x[..., ia], x[..., ib], cs[:, None, :, 0], cs[:, None, :, 1]
    y = x.clone()
    y[..., ia] = rnd(rnd(a * c) - rnd(b * s))
    y[..., ib] = rnd(rnd(b * c) + rnd(a * s))
    return y


def _exact_kv(case, s):
    """Rows after a write and a read: the rotation and the quantiser are defined in 32-bit steps, so each of
    them is computed in 64 bits and rounded; what is read back is code times scale."""
    n, past = _news(case)
    out = []
    for name in ("k",) if case["latent"] else ("k", "v"):
        x = s[name].double()
        if name == "k" and case["rot"]:
            pos = torch.cat([torch.arange(p, p + m) for m, p in zip(n, past)]).to(DEV).double()
            ang = pos[:, None] * _freqs(case)[0].to(DEV)[None, :]
            x = _turn64(x, _r32(torch.stack([torch.cos(ang), torch.sin(ang)], -1)), case["inter"], case["off"], _r32)
        if case["cache"] == "q8":
            T, h, D = x.shape
            blk = x.view(T, h, D // 64, 64)
            d = _r32(blk.abs().max(-1).values / 127)
            code = torch.round(_r32(blk * _r32(1 / d)[..., None]))
            out.append((code * d[..., None]).view(T, h, D))
        else:
            out.append(x.to(DTYPES[case["cache"]]).double())
    return out[0] if case["latent"] else tuple(out)


def _gather64(pool, scale, pages, n):
    x = pool[pages.long()].double()                        # [pages, Hkv, pt, D]
    if scale is not None:
        x = x * scale[pages.long()].double().repeat_interleave(64, dim=-1)
    return x.transpose(0, 1).reshape(x.shape[1], -1, x.shape[-1])[:, :n]


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "table":
        return _table64(s["freqs"], case["first"], case["n_pos"], s["factor"])
    if op == "rope":
        ang = s["pos"].double()[:, None] * _freqs(case)[0].to(DEV)[None, :]
        cs = torch.stack([torch.cos(ang), torch.sin(ang)], -1)
        return _turn64(s["x"].double(), cs, case["inter"], case["off"], lambda v: v)
    if op == "kv":
        return _exact_kv(case, s)
    outs, lses = [], []
    for b, n in enumerate(_lens(case)):
        pages = s["table"][b, :-(-n // case["pt"])]
        q = s["q"][b].double()
        if op == "attn":
            k, v = (_gather64(s[x + "_cache"], s[x + "_scale"], pages, n) for x in "kv")
            q = q.view(case["Hkv"], -1, case["D"])
        else:
            w = s["w"].double()
            k = _gather64(s["c"], s["c_scale"], pages, n)
            v = k[..., :case["R"]]
            qn = torch.matmul(q[:, None, :case["dn"]], w[:, :case["dn"]])[:, 0]
            q = torch.cat([qn, q[:, case["dn"]:]], -1)[None]
        if n:
            sc = torch.matmul(q, k.transpose(1, 2)) * s["scale"]
            lse = torch.logsumexp(sc, -1)
            o = torch.matmul(torch.exp(sc - lse[..., None]), v)
        else:
            lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device=DEV)
            o = torch.zeros((*q.shape[:2], v.shape[-1]), dtype=torch.float64, device=DEV)
        if op == "latent":
            o = torch.matmul(o[0][:, None], w[:, case["dn"]:].transpose(1, 2))[:, 0]
        outs.append(o.reshape(case["H"], -1))
        lses.append(lse.reshape(case["H"]))
    return (torch.stack(outs), torch.stack(lses)) if op == "attn" else torch.stack(outs)
