"""The latent-attention oracle against independent computations (CPU): torch
autograd and finite differences for the gradients, the expanded form for the
absorbed one, and the host layer's refusals that need no GPU."""
import ctypes
import shutil
import subprocess

import pytest
import torch

from atomic_ops import _lib, latent
from oracle import latent as ol

F = torch.float64


def _inputs(B, T, S, H, dn, dr, dv, seed):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F)
    return r(B, T, H, dn + dr), r(B, S, H, dn + dv), r(B, S, dr), r(B, T, H, dv)


@pytest.mark.parametrize("T,S,causal,ql,kl", [(5, 5, True, None, None), (7, 4, True, None, None),
                                              (3, 9, False, [3, 2], [9, 0]), (6, 8, True, [6, 1], [2, 8])])
def test_gradients_follow_autograd_and_differences(T, S, causal, ql, kl):
    q, kv, k_pe, do = _inputs(2, T, S, 2, 6, 4, 5, seed=T * S)
    x = [t.clone().requires_grad_(True) for t in (q, kv, k_pe)]
    dn, loss = 6, 0.0
    for b in range(2):
        see = ol.visible(T, S, T if ql is None else ql[b], S if kl is None else kl[b], causal)
        for h in range(2):
            k = torch.cat((x[1][b, :, h, :dn], x[2][b]), 1)
            s = (x[0][b, :, h] @ k.t() * 0.3).masked_fill(~see, -1e300)
            p = torch.softmax(s, 1) * see.any(1, keepdim=True)
            loss = loss + (p @ x[1][b, :, h, dn:] * do[b, :, h]).sum()
    want = torch.autograd.grad(loss, x)
    got, size = ol.expanded_grads(q, kv, k_pe, do, 0.3, causal, ql, kl)
    f = lambda *a: (ol.expanded(*a, 0.3, causal, ql, kl)[0] * do).sum().item()
    for i, (a, b) in enumerate(zip(got, want)):
        assert (a - b).abs().max() < 1e-12
        assert (a.abs() <= size[i] + 1e-12).all()
        u = torch.randn(a.shape, generator=torch.Generator().manual_seed(i), dtype=F)
        hi, lo = [q, kv, k_pe], [q, kv, k_pe]
        hi[i], lo[i] = hi[i] + 1e-5 * u, lo[i] - 1e-5 * u
        # central differences: error of the order of the step's square
        assert abs((f(*hi) - f(*lo)) / 2e-5 - (a * u).sum().item()) < 1e-7


def test_absorbed_form_is_the_expanded_one():
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g, dtype=F)
    B, n, H, dn, dr, dv, dc, page, ln = 2, 3, 2, 6, 4, 5, 7, 4, 10
    cos, sin = torch.cos(r(16, dr // 2)), torch.sin(r(16, dr // 2))
    cos, sin = cos / (cos ** 2 + sin ** 2).sqrt(), sin / (cos ** 2 + sin ** 2).sqrt()
    w, cache = r(H, dn + dv, dc), r(8, page, dc + dr)
    table = torch.tensor([[4, 1, 7], [0, 2, 5]])
    q = r(B, n, H, dn + dr)
    o = ol.decode(q, w, cache, table, [ln, ln], 0.4, cos, sin, True)
    rows = cache[table].reshape(B, -1, dc + dr)[:, :ln]
    kv = torch.einsum("bsc,hdc->bshd", rows[..., :dc], w)
    qr = q.clone()
    for b in range(B):
        qr[b, :, :, dn:] = ol.rotate(q[b, :, :, dn:], torch.arange(ln - n, ln), cos, sin, True)
    want = ol.expanded(qr, kv, rows[..., dc:], 0.4)[0]
    assert (o - want).abs().max() < 1e-12


def test_rotation_keeps_lengths_and_relative_positions():
    g = torch.Generator().manual_seed(1)
    d = 8
    ang = torch.arange(32, dtype=F)[:, None] * torch.tensor([1.0, 0.3, 0.1, 0.01], dtype=F)
    x, y = (torch.randn(1, d, generator=g, dtype=F) for _ in range(2))
    for inter in (False, True):
        at = lambda t, p: ol.rotate(t, torch.tensor([p]), ang.cos(), ang.sin(), inter)
        assert abs(at(x, 9).norm() - x.norm()) < 1e-12
        assert abs((at(x, 9) * at(y, 4)).sum() - (at(x, 25) * at(y, 20)).sum()) < 1e-12


STRUCTS = [(_lib.LatentArgs, "atomic_latent_args"), (_lib.LatentAppendArgs, "atomic_latent_append_args"),
           (_lib.LatentDecodeArgs, "atomic_latent_decode_args")]


def test_struct_layouts_match_the_header(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    lines = ['#include <stdio.h>', '#include <stddef.h>', f'#include "{_lib.HEADER}"', "int main(void) {"]
    for s, c in STRUCTS:
        lines.append(f'printf("{c} %zu\\n", sizeof({c}));')
        lines += [f'printf("{c}.{f[0]} %zu\\n", offsetof({c}, {f[0]}));' for f in s._fields_]
    src, exe = tmp_path / "l.c", tmp_path / "l"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([gcc, "-std=c11", str(src), "-o", str(exe)], check=True)
    out = dict(l.split() for l in subprocess.run([str(exe)], check=True, capture_output=True,
                                                 text=True).stdout.splitlines())
    for s, c in STRUCTS:
        assert int(out[c]) == ctypes.sizeof(s)
        for f in s._fields_:
            assert int(out[f"{c}.{f[0]}"]) == getattr(s, f[0]).offset, (c, f[0])


def _args(**k):
    d = dict(batch=2, tq=5, tk=9, heads=3, dn=64, dr=32, dv=64, dtype=1, causal=1, scale=0.1)
    st = dict(q_stride=(1440, 288, 96), kv_stride=(3456, 384, 128), kpe_stride=(288, 32), do_stride=(960, 192, 64))
    st.update({n: k.pop(n) for n in list(k) if n.endswith("stride")})
    return _lib.LatentArgs(*{**d, **k}.values(), *st.values())


def test_the_library_refuses_what_it_cannot_run():
    lib = _lib.load()
    size = lambda a: lib.atomic_latent_bwd_workspace_size(ctypes.byref(a))
    assert size(_args()) > 0
    for bad in (dict(dn=12), dict(dn=136), dict(dr=0), dict(dr=72), dict(dv=0), dict(dv=132), dict(tq=0), dict(tk=0),
                dict(heads=0), dict(batch=0), dict(causal=2), dict(dtype=3), dict(tq=(1 << 30) + 1),
                dict(batch=1 << 20, heads=1 << 20), dict(q_stride=(1440, 288, 92)), dict(kv_stride=(-8, 384, 128))):
        assert size(_args(**bad)) == 0, bad
    null = ctypes.c_void_p(0)
    assert lib.atomic_latent_fwd(ctypes.byref(_args()), *[null] * 9, 0, null) == -5
    assert lib.atomic_latent_fwd(None, *[null] * 9, 0, null) == -5
    one = ctypes.c_void_p(16)
    # operands off 16 bytes and a missing workspace are refused before anything is launched
    assert lib.atomic_latent_fwd(ctypes.byref(_args()), ctypes.c_void_p(8), one, one, null, null, one, one, null, null, 0,
                                 null) == -1
    assert lib.atomic_latent_bwd(ctypes.byref(_args()), one, one, one, null, null, one, one, null, *[one] * 4, null, 0, null) == -3
    d = lambda **k: _lib.LatentDecodeArgs(*{**dict(batch=2, tokens=1, heads=4, dn=64, dr=32, dv=64, dc=128, dtype=1,
                                                   page=16, pages=9, table_pages=4, rope_rows=99, interleaved=0,
                                                   scale=0.1), **k}.values(), (384, 384, 96))
    dsize = lambda a: lib.atomic_latent_decode_workspace_size(ctypes.byref(a))
    assert dsize(d()) > 0
    for bad in (dict(dc=520), dict(dc=4), dict(page=0), dict(pages=0), dict(table_pages=0), dict(tokens=0),
                dict(heads=4097), dict(batch=65536), dict(table_pages=1 << 27, page=64), dict(interleaved=2)):
        assert dsize(d(**bad)) == 0, bad
    # cos without sin
    assert lib.atomic_latent_decode(ctypes.byref(d()), *[one] * 5, one, null, one, one, 1 << 30, null) == -5
    ap = lambda **k: _lib.LatentAppendArgs(*{**dict(tokens=3, heads=2, dn=64, dr=32, dc=128, dtype=1, page=16, pages=4,
                                                    rope_rows=9, interleaved=0, c_stride=160, k_stride=160),
                                             **k}.values(), (192, 96))
    call = lambda a: lib.atomic_latent_append(ctypes.byref(a), *[null] * 11)
    assert call(ap()) == -5
    for bad in (dict(tokens=0), dict(heads=-1), dict(page=0), dict(dc=12), dict(c_stride=4), dict(rope_rows=0)):
        assert call(ap(**bad)) == -1, bad
    assert call(ap(dtype=7)) == -2


def test_the_host_layer_refuses_what_does_not_fit():
    q, kv, k_pe = torch.zeros(1, 4, 2, 96), torch.zeros(1, 4, 2, 128), torch.zeros(1, 4, 32)
    with pytest.raises(ValueError, match="device"):
        latent.forward(q, kv, k_pe, 1.0)
    with pytest.raises(ValueError, match="device"):
        latent.append(None, None, k_pe[0], None, torch.zeros(4, dtype=torch.int32), torch.zeros(4, 16),
                      torch.zeros(4, 16))
    with pytest.raises(ValueError, match="device"):
        latent.decode(q, torch.zeros(2, 128, 128), torch.zeros(2, 4, 160), torch.zeros(1, 2, dtype=torch.int32),
                      torch.zeros(1, dtype=torch.int32), 1.0)
