"""Argument checks of the paged KV cache (include/kv_pages.h) that need no GPU: refused with a message
before anything is touched."""

import ctypes

import pytest

import gpu_helpers  # noqa: F401  (puts the package on sys.path)
from gpu_helpers import load_pkg_and_lib


@pytest.fixture(scope="module")
def pl():
    return load_pkg_and_lib()


def _err(pkg, lib):
    msg = pkg.last_error(lib)
    lib.attn_clear_error()
    return msg


GOOD = dict(num_layers=2, num_pages=8, page_size=16, kv_heads=4, head_dim=64, max_seqs=3, max_pages=4, kv_dtype=1)


@pytest.mark.parametrize("field,values", [("num_layers", (0, -1)), ("num_pages", (0, (1 << 20) + 1)), ("page_size", (0, 8, 24, 256)),
                                          ("kv_heads", (0, 1025)), ("head_dim", (32, 96, 256)), ("max_seqs", (0, (1 << 20) + 1)),
                                          ("max_pages", (0, (1 << 20) + 1)), ("kv_dtype", (-1, 2))])
def test_pool_dimensions_are_checked(pl, field, values):
    pkg, lib = pl
    buf = (ctypes.c_char * 64)()
    at = (ctypes.addressof(buf) + 15) & ~15
    for x in values:
        dims = list({**GOOD, field: x}.values())
        assert not lib.kv_pages_alloc(*dims)
        assert field in _err(pkg, lib)
        assert not lib.kv_pages_attach(at, at, at, at, at, *dims)
        assert field in _err(pkg, lib)


def test_rows_beyond_32_bits_are_refused(pl):
    pkg, lib = pl
    dims = {**GOOD, "num_layers": 64, "num_pages": 1 << 19, "page_size": 128, "kv_heads": 8}
    assert not lib.kv_pages_alloc(*dims.values())
    assert "num_layers * num_pages" in _err(pkg, lib)


def test_attach_wants_aligned_addresses(pl):
    pkg, lib = pl
    buf = (ctypes.c_char * 64)()
    at = (ctypes.addressof(buf) + 15) & ~15
    for i, name in enumerate(("k", "v", "table", "len", "ref")):
        args = [at] * 5
        args[i] = None
        # (the addresses before it are host memory, refused as such on a GPU box and uncheckable here)
        if i == 0:
            assert not lib.kv_pages_attach(*args, *GOOD.values())
            assert f"NULL {name}" in _err(pkg, lib)
            args[i] = at + 8
            assert not lib.kv_pages_attach(*args, *GOOD.values())
            assert "aligned" in _err(pkg, lib)


def test_handles_are_checked(pl):
    pkg, lib = pl
    other = (ctypes.c_char * 1024)()
    for h, word in ((None, "NULL"), (ctypes.addressof(other), "not made by")):
        calls = [lambda: lib.kv_pages_extend(h, None, None, 1), lambda: lib.kv_pages_fork(h, None, None, 1),
                 lambda: lib.kv_pages_copy(h, None, None, 1), lambda: lib.kv_pages_free(h, None, 1),
                 lambda: lib.kv_pages_trim(h, None, 1, 1, 0), lambda: lib.kv_pages_compact(h, None),
                 lambda: lib.kv_pages_write(h, 0, None, None, 1, 1, None, None, 1, 64), lambda: lib.kv_pages_import(h, 0, None),
                 lambda: lib.attention_pages_prefix_gqa(None, 0, h, 0, None, 1, 4, 0, 1, None, 1, 1.0),
                 lambda: lib.attention_pages_window_gqa(None, 0, h, 0, None, None, 1, 1, 4, 1, 1, 0, 0, None, 1, 1.0)]
        for call in calls:
            assert call() != 0
            assert word in _err(pkg, lib)
    lib.kv_pages_release(None)
    assert _err(pkg, lib) == ""


def test_attention_arguments_before_the_handle(pl):
    pkg, lib = pl
    assert lib.attention_pages_prefix_gqa(None, 0, None, 0, None, 1, 4, 5, 4, None, 1, 1.0) != 0
    assert "prefix_len" in _err(pkg, lib)
    assert lib.attention_pages_prefix_gqa(None, 0, None, 0, None, 1, 4, 0, 4, None, 7, 1.0) != 0
    assert "element type" in _err(pkg, lib)
    assert lib.attention_pages_window_gqa(None, 0, None, 0, None, None, 1, 1, 4, 1, 1, 0, 0, None, 7, 1.0) != 0
    assert "element type" in _err(pkg, lib)


def test_the_struct_is_the_headers(pl, tmp_path):
    """KVPages of the binding has the size and offsets of include/kv_pages.h."""
    import shutil
    import subprocess
    from pathlib import Path
    pkg, _ = pl
    cc = shutil.which("gcc", path="/usr/bin") or "gcc"
    src, exe = tmp_path / "s.c", tmp_path / "s"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "kv_pages.h"\nint main(void) { printf("%zu %zu %zu %zu %zu\\n", '
                   "sizeof(KVPages), offsetof(KVPages, ref), offsetof(KVPages, num_layers), offsetof(KVPages, max_pages), "
                   "offsetof(KVPages, kv_dtype)); return 0; }\n")
    inc = Path(__file__).resolve().parents[1] / "include"
    subprocess.run([cc, "-Wall", "-Werror", "-I", str(inc), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    s = pkg.KVPages
    assert got == [ctypes.sizeof(s), s.ref.offset, s.num_layers.offset, s.max_pages.offset, s.kv_dtype.offset]
