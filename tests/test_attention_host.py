"""The attention operators' host side (CPU only): rotary frequencies against their formulas, the C structs'
layout, and every refusal of the C entry points and of the Python calls, which come before any device work."""
import ctypes as C
import math
import os
import shutil
import subprocess

import numpy as np
import pytest
import torch

import hearth_b200 as hb
from hearth_b200 import _lib

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
ARG, UNSUP = _lib.HXB_E_ARG, _lib.HXB_E_UNSUPPORTED


@pytest.mark.parametrize("dim", [2, 32, 80, 128])
def test_rope_freqs_plain_linear_ntk(dim):
    j = np.arange(dim // 2)
    f, a = hb.rope_freqs(dim, 1e4)
    np.testing.assert_allclose(f, 1e4 ** (-2 * j / dim), rtol=1e-14)
    assert a == 1.0
    g, a = hb.rope_freqs(dim, 1e4, scaling="linear", factor=8.0)
    np.testing.assert_allclose(g, f / 8, rtol=1e-14)
    assert a == 1.0
    if dim > 2:
        g, _ = hb.rope_freqs(dim, 1e4, scaling="ntk", factor=4.0)
        np.testing.assert_allclose(g, (1e4 * 4 ** (dim / (dim - 2))) ** (-2 * j / dim), rtol=1e-13)


def test_rope_freqs_yarn_between_plain_and_linear():
    f, _ = hb.rope_freqs(64, 1e4)
    g, a = hb.rope_freqs(64, 1e4, scaling="yarn", factor=40.0, original=4096)
    assert a == pytest.approx(0.1 * math.log(40.0) + 1, rel=1e-15)
    keep = (g - f / 40) / (f - f / 40)
    turns = 4096 * f / (2 * math.pi)
    assert np.all(keep[turns > 40] > 1 - 1e-12) and np.all(np.abs(keep[turns < 0.7]) < 1e-12)
    assert np.all(np.diff(keep) <= 1e-12) and 0.2 < keep[(turns > 3) & (turns < 9)].mean() < 0.8


@pytest.mark.parametrize("kw", [dict(scaling="other"), dict(scaling="linear", factor=0.5), dict(scaling="yarn", factor=2.0, original=0),
                                dict(scaling="yarn", factor=2.0, beta_fast=1.0, beta_slow=2.0),
                                dict(scaling="ntk", factor=float("nan"))])
def test_rope_freqs_refuses(kw):
    with pytest.raises(ValueError):
        hb.rope_freqs(64, 1e4, **kw)


def test_rope_freqs_refuses_shapes():
    for dim, theta in ((0, 1e4), (7, 1e4), (2048, 1e4), (64, 1.0), (64, float("inf"))):
        with pytest.raises(ValueError):
            hb.rope_freqs(dim, theta)
    with pytest.raises(ValueError):
        hb.rope_freqs(2, 1e4, scaling="ntk", factor=2.0)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
def test_struct_layout_matches_the_header(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "hearth_b200.h"', "int main(void) {"]
    structs = {"hxb_rope": _lib.Rope, "hxb_kv_cache": _lib.KvCache}
    for name, py in structs.items():
        lines.append(f'    printf("{name} size %zu\\n", sizeof({name}));')
        lines += [f'    printf("{name} {f} %zu\\n", offsetof({name}, {f}));' for f, _ in py._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines + ["    return 0;", "}"]))
    subprocess.run(["gcc", "-std=c11", "-I", os.path.join(REPO, "include"), str(src), "-o", str(exe)], check=True)
    for line in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines():
        name, field, off = line.split()
        want = C.sizeof(structs[name]) if field == "size" else getattr(structs[name], field).offset
        assert int(off) == want, line


P = 1 << 20   # stands for a device pointer: every call below is refused before it is used


def cache(**kw):
    d = dict(dtype=hb.BF16, n_kv_heads=2, head_dim=64, page_tokens=16, n_pages=4, k=P, v=P, k_scale=0, v_scale=0, table=P,
             table_stride=2, table_pages=2, n_seqs=3)
    d.update(kw)
    return _lib.KvCache(*[d[f] for f, _ in _lib.KvCache._fields_])


BAD_CACHE = [(dict(dtype=0), UNSUP), (dict(dtype=4), UNSUP), (dict(n_kv_heads=0), ARG), (dict(head_dim=12), ARG),
             (dict(head_dim=2048), ARG), (dict(dtype=3, head_dim=80, k_scale=P, v_scale=P), ARG), (dict(page_tokens=24), ARG),
             (dict(page_tokens=2048), ARG), (dict(page_tokens=0), ARG), (dict(n_pages=-1), ARG), (dict(k=0), ARG),
             (dict(k=P + 8), ARG), (dict(v=P + 2), ARG), (dict(table=0), ARG), (dict(table_stride=1), ARG), (dict(table_pages=-1), ARG),
             (dict(n_seqs=-1), ARG), (dict(dtype=3), ARG), (dict(k_scale=P), ARG), (dict(v=0), ARG),
             (dict(table_pages=1 << 28, table_stride=1 << 28), ARG),
             (dict(page_tokens=1, table_pages=0x7fffffff, table_stride=0x7fffffff), ARG)]


@pytest.mark.parametrize("kw,code", BAD_CACHE)
def test_bad_caches_are_refused(kw, code):
    L, c = hb.lib(), cache(**kw)
    assert L.hxb_kv_write_dev(C.byref(c), P, P, 5, P, 128, 64, P, 128, 64, 2, None, None) in (code, ARG)
    assert L.hxb_kv_read_dev(C.byref(c), P, P, 5, P, 128, 64, P, 128, 64, 2, None) in (code, ARG)
    assert L.hxb_attn_decode_dev(C.byref(c), P, P, 256, 64, 4, 2, 1.0, P, 256, 64, None, P, 1 << 30, None) == code
    assert hb.last_error()


def test_rows_refusals():
    L, c = hb.lib(), cache()
    ok = dict(start=P, pos0=P, T=5, k=P, ks=128, kh=64, v=P, vs=128, vh=64, dt=2)

    def write(rope=None, **kw):
        d = dict(ok, **kw)
        return L.hxb_kv_write_dev(C.byref(c), d["start"], d["pos0"], d["T"], d["k"], d["ks"], d["kh"], d["v"], d["vs"], d["vh"],
                                  d["dt"], rope, None)

    def read(**kw):
        d = dict(ok, **kw)
        return L.hxb_kv_read_dev(C.byref(c), d["start"], d["pos0"], d["T"], d["k"], d["ks"], d["kh"], d["v"], d["vs"], d["vh"],
                                 d["dt"], None)
    assert write(T=0) == 0 and read(T=0) == 0
    for kw in (dict(T=-1), dict(start=0), dict(pos0=0), dict(k=0), dict(v=0), dict(dt=3), dict(dt=-1), dict(ks=-1), dict(k=P + 1),
               dict(start=P + 2)):
        assert write(**kw) == ARG, kw
        assert read(**kw) == ARG, kw
    for kw in (dict(ks=0), dict(kh=0), dict(kh=32), dict(ks=100)):   # reads may not write one place twice
        assert read(**kw) == ARG, kw
    for r in (dict(rope_dim=66), dict(rope_dim=3), dict(rope_dim=0), dict(offset=8), dict(style=2), dict(n_pos=0), dict(cs=0), dict(offset=-2)):
        d = dict(cs=P, n_pos=10, rope_dim=64, offset=0, style=0)
        d.update(r)
        assert write(rope=C.byref(_lib.Rope(**d))) == ARG, r


def test_rope_refusals():
    L = hb.lib()
    r = _lib.Rope(P, 100, 64, 0, 0)
    ok = dict(r=C.byref(r), pos=P, T=3, H=2, hd=64, x=P, dx=0, xs=128, xh=64, y=2 * P, dy=2, ys=128, yh=64)

    def call(**kw):
        d = dict(ok, **kw)
        return L.hxb_rope_dev(*[d[k] for k in ("r", "pos", "T", "H", "hd", "x", "dx", "xs", "xh", "y", "dy", "ys", "yh")], None)
    assert call(T=0) == 0
    for kw in (dict(r=None), dict(T=-1), dict(H=0), dict(hd=32), dict(hd=4096), dict(dx=3), dict(dy=9), dict(pos=0), dict(x=0), dict(y=0),
               dict(ys=0), dict(yh=32), dict(ys=100), dict(y=P), dict(y=P, dy=0, ys=256), dict(x=P + 2), dict(xs=-1)):
        assert call(**kw) == ARG, kw


def test_rope_table_refusals():
    L = hb.lib()
    f = np.ones(32)
    fp = f.ctypes.data
    assert L.hxb_rope_table_dev(fp, 64, 1.0, 0, 0, None, None) == 0
    for a in ((0, 64, 1.0, 0, 4, P), (fp, 63, 1.0, 0, 4, P), (fp, 2048, 1.0, 0, 4, P), (fp, 64, 1.0, 0, -1, P), (fp, 64, 1.0, 0, 4, 0),
              (fp, 64, 1.0, 0, 4, P + 4), (fp, 64, 1.0, 1 << 31, 4, P), (fp, 64, 1.0, 5, (1 << 31) - 4, P)):
        assert L.hxb_rope_table_dev(*a, None) == ARG, a
    f[3] = np.inf
    assert L.hxb_rope_table_dev(fp, 64, 1.0, 0, 4, P, None) == ARG


def test_attention_refusals():
    L = hb.lib()
    ok = dict(c=cache(), lens=P, q=P, qs=256, qh=64, H=4, dt=2, scale=1.0, out=P + (1 << 20), os=256, oh=64, lse=None, ws=P, n=1 << 30)

    def call(**kw):
        d = dict(ok, **kw)
        return L.hxb_attn_decode_dev(C.byref(d["c"]), *[d[k] for k in ("lens", "q", "qs", "qh", "H", "dt", "scale", "out", "os", "oh",
                                                                       "lse", "ws", "n")], None)
    assert call(c=cache(n_seqs=0)) == 0
    assert call(c=cache(head_dim=72)) == UNSUP and call(c=cache(head_dim=512)) == UNSUP
    for kw in (dict(H=3), dict(H=0), dict(dt=3), dict(lens=0), dict(q=0), dict(out=0), dict(ws=0), dict(ws=P + 8), dict(n=0), dict(oh=32),
               dict(os=128), dict(qs=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(q=P + 1), dict(lse=P + 2), dict(out=P),
               dict(c=cache(n_seqs=65536))):
        assert call(**kw) == ARG, kw
    assert L.hxb_attn_decode_workspace(C.byref(ok["c"]), 4) > 0


def test_latent_refusals():
    L = hb.lib()
    lat = lambda **kw: cache(**dict(dict(n_kv_heads=1, head_dim=576, v=0), **kw))  # noqa: E731
    ok = dict(c=lat(), lens=P, q=P, qs=4 * 192, qh=192, w=P, H=4, R=512, dn=128, dv=128, dt=2, scale=1.0, out=P + (1 << 20), os=512, oh=128, ws=P,
              n=1 << 30)

    def call(**kw):
        d = dict(ok, **kw)
        return L.hxb_latent_decode_dev(C.byref(d["c"]), *[d[k] for k in ("lens", "q", "qs", "qh", "w", "H", "R", "dn", "dv", "dt", "scale",
                                                                         "out", "os", "oh", "ws", "n")], None)
    assert call(c=lat(n_seqs=0)) == 0
    for kw in (dict(R=500), dict(R=64), dict(R=384), dict(R=576), dict(dn=8), dict(dv=100), dict(dv=512), dict(c=lat(head_dim=520))):
        assert call(**kw) == UNSUP, kw
    for kw in (dict(c=lat(v=P)), dict(c=lat(n_kv_heads=2)), dict(c=lat(dtype=1)), dict(dt=0), dict(H=0), dict(H=512), dict(w=0),
               dict(w=P + 2), dict(ws=0), dict(n=16), dict(lens=0), dict(oh=64), dict(out=P), dict(c=lat(n_seqs=65536))):
        assert call(**kw) == ARG, kw
    assert L.hxb_latent_decode_workspace(C.byref(ok["c"]), 4, 512) > 0


def test_python_calls_refuse_before_device_work():
    f32, i32 = torch.float32, torch.int32
    kc = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16)
    table, lens = torch.zeros(3, 2, dtype=i32), torch.zeros(3, dtype=i32)
    start, pos0 = torch.zeros(4, dtype=i32), torch.zeros(3, dtype=i32)
    k = torch.zeros(5, 2, 64)
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    cs = torch.zeros(10, 32, 2)
    bad = [
        lambda: hb.kv_write(k, k, kc, kc, table, start, pos0),                       # on the CPU
        lambda: hb.kv_write(k, None, kc, kc, table, start, pos0),
        lambda: hb.kv_write(k.double(), k.double(), kc, kc, table, start, pos0),
        lambda: hb.kv_write(k, k[:4], kc, kc, table, start, pos0),
        lambda: hb.kv_write(k, k, kc, kc, table.long(), start, pos0),
        lambda: hb.kv_write(k, k, kc, kc, table, start[:3], pos0),
        lambda: hb.kv_write(k, k, kc, kc, table, start, pos0, k_scale=torch.zeros(4, 2, 16, 1)),
        lambda: hb.kv_write(k, k, kc.to(torch.int8), kc.to(torch.int8), table, start, pos0),
        lambda: hb.kv_write(k, k, kc, kc, table, start, pos0, cs=cs[..., :1]),
        lambda: hb.kv_read(kc.transpose(1, 2), kc, table, start, pos0, k, k),
        lambda: hb.rope(k, pos0, cs),
        lambda: hb.rope(k.transpose(1, 2), torch.zeros(5, dtype=i32), cs),
        lambda: hb.rope(k, torch.zeros(5), cs),
        lambda: hb.rope_table(np.zeros((2, 2)), 4),
        lambda: hb.rope_table(np.zeros(2), 4, out=torch.zeros(4, 2, 2, dtype=torch.float64)),
        lambda: hb.decode_attention(q, kc, None, table, lens, scale=1.0),
        lambda: hb.decode_attention(q[:2], kc, kc, table, lens, scale=1.0),
        lambda: hb.decode_attention(q, kc, kc, table, lens, scale=1.0, out=torch.zeros(3, 4, 64)),
        lambda: hb.decode_attention(q, kc, kc, table, lens, scale=1.0, lse=torch.zeros(3, 5)),
        lambda: hb.decode_attention(q, kc, kc, table, lens, scale=1.0),              # on the CPU
        lambda: hb.latent_attention(q, q, kc, table, lens, scale=1.0),
    ]
    for i, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {i} was accepted")
    assert f32 is torch.float32


def test_empty_pools_need_no_pointers():
    """A pool of no pages (its tensors have no memory) is taken by every call, with keys and values and latent."""
    L = hb.lib()
    for heads in (1, 2):
        c = cache(n_kv_heads=heads, n_pages=0, k=0, v=0)
        for v in (P, None):
            assert L.hxb_kv_write_dev(C.byref(c), P, P, 0, P, 128, 64, v, 128, 64, 2, None, None) == 0, hb.last_error()
            assert L.hxb_kv_read_dev(C.byref(c), P, P, 0, P, 128, 64, v, 128, 64, 2, None) == 0, hb.last_error()
    c = cache(v=0)
    assert L.hxb_kv_write_dev(C.byref(c), P, P, 5, P, 128, 64, P, 128, 64, 2, None, None) == ARG and "without v" in hb.last_error()
    assert L.hxb_kv_write_dev(C.byref(c), P, P, 5, P, 128, 64, None, 0, 0, 2, None, None) == ARG


def test_numbers_that_c_would_wrap_are_refused():
    x, cs, pos = torch.zeros(5, 2, 64), torch.zeros(10, 32, 2), torch.zeros(5, dtype=torch.int32)
    for f, msg in ((lambda: hb.rope(x, pos, cs, offset=1 << 32), "offset"), (lambda: hb.rope(x, pos, cs, offset=-1 << 32), "offset"),
                   (lambda: hb.rope_freqs(64, 1e4, scaling="yarn", factor=2.0, original=(1 << 32) + 4096), "original"),
                   (lambda: hb.rope_table([1.0], 4, first=1 << 64), "positions"), (lambda: hb.rope_table([1.0], 4, first=-1 << 31), "positions"),
                   (lambda: hb.rope_table([1.0], 1 << 40), "positions"), (lambda: hb.rope_table([1.0], 3, first=(1 << 31) - 2), "positions")):
        with pytest.raises(ValueError, match=msg):
            f()


@pytest.mark.parametrize("original,slow", [(1, 1.0), (6, 1.0), (100, 20.0), (4096, 700.0)])
def test_rope_freqs_yarn_where_no_frequency_turns(original, slow):
    """Where even the first frequency makes beta_slow turns or fewer over the original positions, all are divided."""
    assert original / (2 * math.pi) <= slow
    f, _ = hb.rope_freqs(64, 1e4)
    g, _ = hb.rope_freqs(64, 1e4, scaling="yarn", factor=8.0, original=original, beta_fast=32 * slow, beta_slow=slow)
    np.testing.assert_allclose(g, f / 8, rtol=1e-14)


@pytest.mark.parametrize("factor", [float("nan"), float("inf"), 1e39])
def test_rope_table_refuses_factors(factor):
    f = (C.c_double * 2)(1.0, 0.5)
    assert hb.lib().hxb_rope_table_dev(f, 4, factor, 0, 10, P, None) == ARG and "factor" in hb.last_error()
