"""The C entries of shared prefixes, gathered weights and eviction where no GPU is
needed: their structs' layout and what they refuse before anything is launched."""
import ctypes
import shutil
import subprocess

import pytest

from atomic_ops import _lib

STRUCTS = [(_lib.LatentDecodeArgs, "atomic_latent_decode_args"), (_lib.LatentSharedArgs, "atomic_latent_shared_args"),
           (_lib.LatentEvictArgs, "atomic_latent_evict_args")]


def test_structs_match_the_c_compiler(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("gcc not available")
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "%s"' % _lib.HEADER, "int main(void) {"]
    for struct, name in STRUCTS:
        lines.append('printf("%s %%zu\\n", sizeof(%s));' % (name, name))
        lines += ['printf("%s.%s %%zu\\n", offsetof(%s, %s));' % (name, f[0], name, f[0]) for f in struct._fields_]
    src, exe = tmp_path / "layout.c", tmp_path / "layout"
    src.write_text("\n".join(lines + ["return 0; }"]))
    subprocess.run([gcc, "-std=c11", str(src), "-o", str(exe)], check=True)
    out = dict(x.split() for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.splitlines())
    for struct, name in STRUCTS:
        assert int(out[name]) == ctypes.sizeof(struct)
        for f in struct._fields_:
            assert int(out[f"{name}.{f[0]}"]) == getattr(struct, f[0]).offset, (name, f[0])


def _dec(**kw):
    a = _lib.LatentDecodeArgs(batch=6, tokens=1, heads=4, dn=64, dr=32, dv=64, dc=128, dtype=_lib.ATOMIC_BF16, page=16,
                              pages=9, table_pages=3, rope_rows=0, interleaved=0, scale=0.1)
    a.q_stride[:] = 4 * 96, 4 * 96, 96
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def _shared(prefixes=2, prefix_pages=2, scored=0, stride=48, **kw):
    return _lib.LatentSharedArgs(_dec(**kw), prefixes, prefix_pages, scored, stride)


def test_shared_refusals():
    lib = _lib.load()
    size = lambda a: lib.atomic_latent_decode_shared_workspace_size(ctypes.byref(a))  # noqa: E731
    for a in (_shared(), _shared(prefixes=0), _shared(prefix_pages=0), _shared(table_pages=0), _shared(scored=1),
              _shared(scored=1, prefixes=0), _shared(prefixes=6), _shared(scored=1, table_pages=0, stride=0),
              _shared(batch=1 << 14, heads=64, prefixes=1)):
        assert size(a) > 0
    assert size(_shared(scored=1)) > size(_shared())
    for a in (_shared(prefixes=4), _shared(prefixes=-1), _shared(prefix_pages=-1), _shared(scored=2),
              _shared(scored=1, stride=47), _shared(prefixes=0, table_pages=0), _shared(prefix_pages=0, table_pages=0),
              _shared(prefix_pages=1 << 27), _shared(dn=144), _shared(dtype=3), _shared(table_pages=-1),
              _shared(batch=1 << 14, heads=65, prefixes=1)):
        assert size(a) == 0
    p = ctypes.c_void_p(4096)   # never read: every call below is refused

    def call(a, none=(), odd=(), ws=p, n=1 << 40):
        at = [None if i in none else ctypes.c_void_p(4100) if i in odd else p for i in range(11)]
        return lib.atomic_latent_decode_shared(ctypes.byref(a), *at, ws, n, None)

    names = ("q", "w_kv", "cache", "prefix_table", "prefix_lens", "page_table", "kv_lens", "cos", "sin", "weights", "o")
    for i, name in enumerate(names):
        assert call(_shared(scored=1, rope_rows=4), none=(i,), n=0) == -5, name
    assert call(_shared(rope_rows=4), none=(9,), n=0) == -3                    # unless scored, no weights
    assert call(_shared(prefixes=0, rope_rows=4), none=(3, 4, 9), n=0) == -3
    for i in (0, 1, 2, 7, 8, 10):
        assert call(_shared(rope_rows=4), odd=(i,)) == -1, names[i]
    assert call(_shared(rope_rows=0)) == -1
    assert call(_shared(rope_rows=4), n=16) == -3 and call(_shared(rope_rows=4), ws=None) == -3
    assert call(_shared(prefixes=4, rope_rows=4)) == -1


def _evict(**kw):
    a = _lib.LatentEvictArgs(batch=2, dtype=_lib.ATOMIC_BF16, row=96, page=16, pages=9, table_pages=3, width=50, keep=20,
                             sinks=1, recent=4, weights_stride=50, order_stride=50, weights_out_stride=50,
                             order_out_stride=50)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def test_evict_refusals():
    lib = _lib.load()
    size = lambda a: lib.atomic_latent_evict_workspace_size(ctypes.byref(a))  # noqa: E731
    for kw in ({}, dict(keep=1, sinks=0, recent=1), dict(keep=20, sinks=16), dict(sinks=0, recent=0), dict(keep=1 << 20),
               dict(row=16), dict(row=576), dict(table_pages=1)):
        assert size(_evict(**kw)) > 0, kw
    for kw in (dict(batch=0), dict(batch=65536), dict(row=8), dict(row=92), dict(row=584), dict(page=0), dict(pages=0),
               dict(table_pages=0), dict(table_pages=4), dict(keep=0), dict(keep=4), dict(sinks=-1), dict(recent=-1),
               dict(sinks=17), dict(recent=20), dict(weights_stride=49), dict(order_stride=49), dict(dtype=2),
               dict(weights_out_stride=49), dict(order_out_stride=49), dict(page=1 << 20, table_pages=1 << 12),
               dict(sinks=(1 << 31) - 1, recent=(1 << 31) - 1, keep=1 << 30)):
        assert size(_evict(**kw)) == 0, kw
    p = ctypes.c_void_p(4096)

    def call(a, none=None, odd=None, ws=p, n=1 << 40):
        at = [None if i == none else ctypes.c_void_p(4100) if i == odd else p for i in range(9)]
        return lib.atomic_latent_evict(ctypes.byref(a), *at, ws, n, None)

    for i in range(9):
        assert call(_evict(), none=i, n=0) == -5, i
    assert call(_evict(), odd=0) == -1
    assert call(_evict(), n=16) == -3 and call(_evict(), ws=None) == -3 and call(_evict(), ws=ctypes.c_void_p(4100)) == -3
    assert call(_evict(keep=0)) == -1 and call(_evict(dtype=2)) == -2
