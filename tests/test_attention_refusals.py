"""Every refusal of the attention operators' Python calls by its own message: a call that is right but for one argument. What
does not need the device is tested on the CPU too, where a call that passed its check would end at the device's message."""
import numpy as np
import pytest
import torch

import hearth_b200 as hb


class Calls:
    """Right arguments of each call (5 rows or 3 sequences, 2 kv heads of 64, pages of 16), to be changed one by one."""

    def __init__(self, dev):
        z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, dtype=dtype, device=dev)  # noqa: E731
        i32, f32, i8 = torch.int32, torch.float32, torch.int8
        self.z, self.dev = z, dev
        self.table, self.lens, self.start, self.pos0, self.pos = z(3, 2, dtype=i32), z(3, dtype=i32), z(4, dtype=i32), z(3, dtype=i32), z(5, dtype=i32)
        self.k, self.kc, self.cs = z(5, 2, 64), z(4, 2, 16, 64), z(10, 32, 2, dtype=f32)
        self.k8, self.s8 = z(4, 2, 16, 64, dtype=i8), z(4, 2, 16, 1, dtype=f32)
        self.q, self.ql, self.w, self.cl = z(3, 4, 64), z(3, 4, 32 + 64), z(4, 32 + 48, 128), z(4, 1, 16, 192)

    def kv_write(self, **kw):
        d = dict(k=self.k, v=self.k.clone(), k_cache=self.kc, v_cache=self.kc.clone(), table=self.table, start=self.start, pos0=self.pos0)
        hb.kv_write(**{**d, **kw})

    def kv_read(self, **kw):
        d = dict(k_cache=self.kc, v_cache=self.kc.clone(), table=self.table, start=self.start, pos0=self.pos0, k_out=self.k, v_out=self.k.clone())
        hb.kv_read(**{**d, **kw})

    def rope(self, **kw):
        hb.rope(**{**dict(x=self.k, pos=self.pos, cs=self.cs), **kw})

    def rope_table(self, **kw):
        hb.rope_table(**{**dict(freqs=[1.0, 0.5], n_pos=4, device=self.dev), **kw})

    def attend(self, **kw):
        d = dict(q=self.q, k_cache=self.kc, v_cache=self.kc.clone(), table=self.table, lens=self.lens, scale=1.0)
        hb.decode_attention(**{**d, **kw})

    def latent(self, **kw):
        hb.latent_attention(**{**dict(q=self.ql, w=self.w, c_cache=self.cl, table=self.table, lens=self.lens, scale=1.0), **kw})


f64, i64, f32 = torch.float64, torch.int64, torch.float32
# (the call and what is wrong with it, its message)
EARLY = [
    (lambda c: c.kv_write(k=c.z(5, 128)), "tokens, heads, dim"), (lambda c: c.kv_write(k=c.z(5, 3, 64)), r"k must be \[tokens, 2, 64\]"),
    (lambda c: c.kv_write(v=None), "v goes with a v_cache"), (lambda c: c.kv_write(v=c.k[:4]), "v must be like k"),
    (lambda c: c.kv_write(v=c.k.float()), "v must be like k"), (lambda c: c.kv_write(k=c.k.to(f64), v=c.k.to(f64)), "k must be float32"),
    (lambda c: c.kv_write(k=c.z(5, 64, 2).transpose(1, 2)), "last dimension"), (lambda c: c.kv_write(table=c.table.long()), "table must be int32"),
    (lambda c: c.kv_write(table=c.z(2, 3, dtype=torch.int32).t()), "table rows"), (lambda c: c.kv_write(start=c.start[:3]), "start must have 4"),
    (lambda c: c.kv_write(pos0=c.pos0.long()), "pos0 must be a contiguous int32"), (lambda c: c.kv_write(k_scale=c.s8), "k_scale goes with an int8"),
    (lambda c: c.kv_write(k_cache=c.k8, v_cache=c.k8), "k_scale must be float32"),
    (lambda c: c.kv_write(k_cache=c.k8, v_cache=c.k8, k_scale=c.s8, v_scale=c.s8.to(f64)), "v_scale must be float32"),
    (lambda c: c.kv_write(k_cache=c.kc.float(), v_cache=c.kc.float()), "a cache is float16"), (lambda c: c.kv_write(v_cache=c.kc[:3]), "v_cache must be like"),
    (lambda c: c.kv_write(k_cache=c.kc.transpose(1, 2)), "k_cache must be contiguous"), (lambda c: c.kv_write(cs=c.cs[..., :1]), "cs must be"),
    (lambda c: c.kv_write(cs=c.cs, offset=-1), "offset"), (lambda c: c.kv_read(k_out=c.z(5, 2, 64, dtype=torch.int32), v_out=c.z(5, 2, 64, dtype=torch.int32)), "k_out must be float32"),
    (lambda c: c.rope(x=c.z(5, 64)), "tokens, heads, dim"), (lambda c: c.rope(pos=c.pos[:4]), "pos must have 5"),
    (lambda c: c.rope(pos=c.pos.float()), "pos must be a contiguous int32"), (lambda c: c.rope(cs=c.cs.to(f64)), "cs must be"),
    (lambda c: c.rope_table(freqs=np.zeros((2, 2))), "freqs must be a vector"), (lambda c: c.rope_table(n_pos=-1), "n_pos"),
    (lambda c: c.rope_table(out=c.z(4, 2, 2, dtype=f64)), "out must be a contiguous float32"), (lambda c: c.rope_table(out=c.z(4, 3, 2, dtype=f32)), "out must be"),
    (lambda c: c.attend(v_cache=None), "needs a v_cache"), (lambda c: c.attend(q=c.q[:2]), r"q must be \[3, heads, 64\]"),
    (lambda c: c.attend(q=c.z(3, 4, 128)), r"q must be \[3, heads, 64\]"), (lambda c: c.attend(lens=c.lens[:2]), "lens must have 3"),
    (lambda c: c.attend(q=c.q.to(f64)), "q must be float32"), (lambda c: c.latent(w=c.w.float()), "in q's type"),
    (lambda c: c.latent(w=c.w[:3]), "w must be contiguous"), (lambda c: c.latent(q=c.ql[:2]), "do not fit together"),
    (lambda c: c.latent(w=c.z(4, 32, 128)), "do not fit together"), (lambda c: c.latent(lens=c.lens.long()), "lens must be a contiguous int32"),
    (lambda c: c.latent(c_scale=c.s8), "k_scale goes with an int8|c_scale"),
]
LATE = [
    (lambda c: c.rope(out=c.z(5, 2, 32)), "out must have x's shape"), (lambda c: c.rope(out=c.z(5, 2, 64, dtype=f64)), "out must be float32"),
    (lambda c: c.rope(offset=4), "rotation of 64 values at 4"), (lambda c: c.rope(out=c.z(1, 2, 64).expand(5, 2, 64)), "bad strides"),
    (lambda c: c.kv_write(cs=c.cs, offset=8), "rotation of 64 values at 8"), (lambda c: c.kv_read(k_out=c.z(1, 2, 64).expand(5, 2, 64)), "bad strides"),
    (lambda c: c.rope_table(factor=float("nan")), "not finite"), (lambda c: c.rope_table(freqs=[float("inf")]), "not finite"),
    (lambda c: c.attend(out=c.q.float()), "out must be like q"), (lambda c: c.attend(out=c.z(3, 4, 32)), "out must be like q"),
    (lambda c: c.attend(out=c.z(1, 4, 64).expand(3, 4, 64)), "bad strides"), (lambda c: c.attend(out=c.q), "in place"),
    (lambda c: c.attend(lse=c.z(3, 5, dtype=f32)), "lse must be"), (lambda c: c.attend(lse=c.z(3, 4)), "lse must be"),
    (lambda c: c.attend(lse=c.z(4, 3, dtype=f32).t()), "lse must be"), (lambda c: c.attend(workspace=c.z(1 << 24)), "workspace must be"),
    (lambda c: c.attend(workspace=c.z(64, dtype=torch.uint8)), "workspace must be"), (lambda c: c.attend(workspace=c.z((1 << 24) + 8, dtype=torch.uint8)[8:]), "workspace of"),
    (lambda c: c.attend(scale=float("inf")), "scale is not finite"), (lambda c: c.attend(q=c.z(3, 3, 64)), "3 heads over 2"),
    (lambda c: c.latent(out=c.z(3, 4, 32)), r"out must be \[3, 4, 48\]"), (lambda c: c.latent(out=c.z(3, 4, 48, dtype=f32)), r"out must be \[3, 4, 48\]"),
    (lambda c: c.latent(workspace=c.z(64, dtype=torch.uint8)), "workspace must be"), (lambda c: c.latent(scale=float("nan")), "scale is not finite"),
    (lambda c: c.latent(q=c.ql.float(), w=c.w.float()), "dtype 0"), (lambda c: c.latent(q=c.ql.half(), w=c.w.half()), "has the type of q"),
    (lambda c: c.latent(w=c.z(4, 32 + 40, 128)), "v_dim 40"),
]


@pytest.mark.parametrize("i", range(len(EARLY)))
def test_refused_before_the_device_is_looked_at(i):
    call, msg = EARLY[i]
    with pytest.raises(ValueError, match=msg):
        call(Calls("cpu"))


@pytest.mark.parametrize("name", ["kv_write", "kv_read", "rope", "attend", "latent"])
def test_right_calls_on_the_cpu_end_at_the_device(name):
    with pytest.raises(ValueError, match="CUDA device"):
        getattr(Calls("cpu"), name)()


@pytest.mark.gpu
def test_refused_on_the_gpu(gpu):
    """Each by its message, with nothing enqueued and the outputs untouched; the right calls are taken."""
    c = Calls("cuda")
    for call in (c.kv_write, c.kv_read, c.rope, c.rope_table, c.attend, c.latent):
        call()
    for i, (call, msg) in enumerate(EARLY + LATE):
        with pytest.raises(ValueError, match=msg):
            call(c)
            pytest.fail(f"call {i} ({msg}) was accepted")
    for call in (c.rope, c.attend, c.latent):
        with pytest.raises(ValueError, match="one CUDA device"):
            call(**{"pos" if call == c.rope else "lens": torch.zeros(5 if call == c.rope else 3, dtype=torch.int32)})
    torch.cuda.synchronize()
