"""The page functions: what is refused on the host, without a GPU."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

import flash_attention_turing_b200 as fa
from flash_attention_turing_b200 import capi

pytestmark = pytest.mark.skipif(not capi.LIB_PATH.exists(), reason="libfa_b200.so not built")
HEADER = Path(__file__).resolve().parent.parent / "include" / "fa_b200.h"


def _int(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def test_types_are_checked_first():
    table, lens, refs, cache = _int(2, 3), _int(2), _int(4), torch.zeros(4, 32, 64, dtype=torch.float16)
    with pytest.raises(TypeError, match="new_tokens must be an int"):
        fa.kvcache_reserve(table, lens, refs, 1.5, 32)
    with pytest.raises(TypeError, match="page_refs must be"):
        fa.kvcache_reserve(table, lens, [0], 1, 32)
    with pytest.raises(TypeError, match="sequence of tensors"):
        fa.kvcache_copy_pages(cache, lens, lens)
    with pytest.raises(TypeError, match="parents must be"):
        fa.kvcache_fork([cache], table, lens, refs, [0], lens)
    with pytest.raises(TypeError, match="rows must be"):
        fa.kvcache_free(table, lens, refs, 0)
    for call in (lambda: fa.kvcache_reserve(table, lens, refs, 1, 32), lambda: fa.kvcache_free(table, lens, refs, lens),
                 lambda: fa.kvcache_fork([cache], table, lens, refs, lens, lens), lambda: fa.kvcache_compact([cache], table, refs),
                 lambda: fa.kvcache_copy_pages([cache], lens, lens)):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


def test_c_entry_points_check_their_arguments():
    lib, t, c = capi.lib(), capi.FaPageTables(), capi.FaPageCaches()
    at, size = 1 << 20, 1 << 30  # an address that is never read: the calls end before
    assert lib.fa_pages_reserve(None, None, 1, 32, at, at, size, None) == -1
    assert lib.fa_pages_reserve(ctypes.byref(t), None, 1, 32, at, at, size, None) == -1 and b"non-NULL" in lib.fa_last_error()
    t.block_table = t.cache_seqlens = t.page_refs = at
    assert lib.fa_pages_reserve(ctypes.byref(t), None, 1, 32, at, at, size, None) == -1
    t.rows, t.columns, t.num_pages, t.row_stride = 4, 3, 10, 2
    assert lib.fa_pages_free(ctypes.byref(t), at, 1, None) == -1
    t.row_stride = 3
    assert lib.fa_pages_reserve(ctypes.byref(t), None, 1, 0, at, at, size, None) == -1
    need = lib.fa_pages_workspace_bytes(4, 10, 0)
    assert 0 < need < 8192
    assert lib.fa_pages_reserve(ctypes.byref(t), None, 1, 32, at, at, need - 1, None) == -3
    assert lib.fa_pages_reserve(ctypes.byref(t), None, 1, 32, at, at + 16, need, None) == -1 and b"aligned" in lib.fa_last_error()
    assert lib.fa_pages_copy(None, 10, at, at, 1, at, at, size, None) == -1
    c.base, c.page_stride = (ctypes.c_void_p * 1)(at + 8), (ctypes.c_int64 * 1)(4096)
    c.page_bytes, c.count = 4096, 1
    assert lib.fa_pages_copy(ctypes.byref(c), 10, at, at, 1, at, at, size, None) == -1 and b"aligned" in lib.fa_last_error()
    c.base = (ctypes.c_void_p * 1)(at)
    c.page_bytes = 4100
    assert lib.fa_pages_copy(ctypes.byref(c), 10, at, at, 1, at, at, size, None) == -1
    c.page_bytes = 8192  # more than the stride
    assert lib.fa_pages_copy(ctypes.byref(c), 10, at, at, 1, at, at, size, None) == -1
    c.page_bytes = 4096
    assert lib.fa_pages_fork(ctypes.byref(t), ctypes.byref(c), at, at, 2, 512, at, at, size, None) == -1 and b"token" in lib.fa_last_error()
    assert lib.fa_pages_fork(ctypes.byref(t), ctypes.byref(c), at, at, -1, 256, at, at, size, None) == -1
    assert lib.fa_pages_fork(ctypes.byref(t), ctypes.byref(c), at, at, 0, 256, at, at, size, None) == 0
    assert lib.fa_pages_compact(ctypes.byref(t), ctypes.byref(c), None, at, size, None) == -1


def test_struct_layouts_match_the_header(tmp_path):
    names = ("FaPageTables", "FaPageCaches")
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "fa_b200.h"\nint main(void){'
                   + "".join(f'printf("%zu\\n", sizeof({n}));' for n in names) + "return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(getattr(capi, n)) for n in names]
