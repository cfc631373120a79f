"""Differential attention: what is refused on the host, without a GPU."""
import ctypes
import subprocess
from pathlib import Path

import pytest
import torch

import flash_attention_turing_b200 as fa
from flash_attention_turing_b200 import capi

HEADER = Path(__file__).resolve().parent.parent / "include" / "fa_b200.h"
built = pytest.mark.skipif(not capi.LIB_PATH.exists(), reason="libfa_b200.so not built")


def _cache(b=2, n=16, h=4, hk=2, d=64):
    half = lambda *shape: torch.zeros(*shape, dtype=torch.float16)  # noqa: E731
    return half(b, 1, h, d), half(b, n, hk, d), half(b, n, hk, d), torch.zeros(h)


def test_kvcache_arguments_are_checked_as_in_the_plain_call():
    q, k, v, lam = _cache()
    new = torch.zeros(2, 1, 2, 64, dtype=torch.float16)
    with pytest.raises(TypeError, match="lam must be"):
        fa.flash_diff_attn_with_kvcache(q, k, v, None)
    with pytest.raises(ValueError, match="both be provided"):
        fa.flash_diff_attn_with_kvcache(q, k, v, lam, new)
    with pytest.raises(ValueError, match="head_dim 64 or 128"):
        fa.flash_diff_attn_with_kvcache(q[..., :32], k, v, lam)
    with pytest.raises(ValueError, match="cache_seqlens is required"):
        fa.flash_diff_attn_with_kvcache(q, k, v, lam, new, new)
    with pytest.raises(ValueError, match="capacity is insufficient"):
        fa.flash_diff_attn_with_kvcache(q, k, v, lam, new, new, cache_seqlens=16)
    with pytest.raises(ValueError, match="divisible by 256"):
        fa.flash_diff_attn_with_kvcache(q, k, v, lam, cache_seqlens=1, block_table=torch.zeros(2, 1, dtype=torch.int32))
    with pytest.raises(ValueError, match="non-negative"):
        fa.flash_diff_attn_with_kvcache(q, k, v, lam, cache_seqlens=1, num_splits=-1)
    with pytest.raises(RuntimeError, match="must be CUDA tensors"):
        fa.flash_diff_attn_with_kvcache(q, k, v, lam, cache_seqlens=1)


@built
def test_cpu_tensors_are_refused():
    q, k, v, lam = _cache()
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fa.flash_diff_attn_func(q, k, v, lam)
    cu = torch.tensor([0, 1], dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA tensor"):
        fa.flash_diff_attn_varlen_func(q[0], k[0], v[0], lam, cu, cu, 1, 1)


@built
def test_c_entry_points_check_their_arguments():
    lib = capi.lib()
    f, b, k = capi.FaDiffFwdParams(), capi.FaDiffBwdParams(), capi.FaDiffKvcacheParams()
    assert lib.fa_diff_fwd(None, None) == -1 and lib.fa_diff_bwd(None, None) == -1
    assert lib.fa_diff_kvcache(None, None, 0, None) == -1
    assert lib.fa_diff_fwd(ctypes.byref(f), None) == -1 and b"non-NULL" in lib.fa_last_error()
    assert lib.fa_diff_bwd(ctypes.byref(b), None) == -1
    assert lib.fa_diff_kvcache(ctypes.byref(k), None, 0, None) == -2  # d, as fa_kvcache()
    k.base.d = 64
    assert lib.fa_diff_kvcache(ctypes.byref(k), None, 0, None) == -1
    at = 1 << 20  # an address that is never read: the call ends before
    f.base.q = f.base.k = f.base.v = f.base.o = f.base.lse = at
    f.base.d = 96
    assert lib.fa_diff_fwd(ctypes.byref(f), None) == -2 and b"head_dim" in lib.fa_last_error()
    f.base.d, f.base.b, f.base.h, f.base.h_k, f.base.seqlen_q = 64, 1, 4, 3, 8
    assert lib.fa_diff_fwd(ctypes.byref(f), None) == -1
    f.base.h_k = 2
    assert lib.fa_diff_fwd(ctypes.byref(f), None) == -1 and b"lam" in lib.fa_last_error()
    f.weights.lam, f.weights.count = at, 3
    assert lib.fa_diff_fwd(ctypes.byref(f), None) == -1 and b"count" in lib.fa_last_error()


@built
@pytest.mark.parametrize("b,rows,splits", [(1, 70, 0), (1, 4096, 64), (32, 2048, 64), (32, 2048, 0), (3, 200, 3), (2, 200, 0)])
def test_scratch_memory_of_parts_is_bounded(b, rows, splits):
    """Partial rows of a chunk of a prompt: three for 148 tiles of 128 rows of both maps at most, whatever num_splits asks for."""
    p = capi.FaDiffKvcacheParams()
    p.base.b, p.base.seqlen_q, p.base.seqlen_new, p.base.h, p.base.h_k, p.base.d = b, rows, rows, 32, 8, 128
    p.base.cache_batch, p.base.seqlen_cache, p.base.num_splits, p.base.softmax_scale = b, 32768, splits, 0.1
    assert capi.lib().fa_diff_kvcache_workspace_bytes(ctypes.byref(p)) <= 3 * 148 * 128 * 2 * (128 + 1) * 4 + 1024


@built
def test_struct_layouts_match_the_header(tmp_path):
    names = ("FaDiffWeights", "FaDiffFwdParams", "FaDiffBwdParams", "FaDiffKvcacheParams")
    src = tmp_path / "sizes.c"
    src.write_text('#include <stdio.h>\n#include "fa_b200.h"\nint main(void){'
                   + "".join(f'printf("%zu\\n", sizeof({n}));' for n in names) + "return 0;}\n")
    exe = tmp_path / "sizes"
    subprocess.run(["gcc", "-std=c99", "-I", str(HEADER.parent), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(getattr(capi, n)) for n in names]


@built
@pytest.mark.parametrize("b,longest,total,h", [(1000, 8192, 8192 + 999 * 24, 16), (4096, 4096, 200000, 8), (3, 100, 220, 4), (1, 5000, 5000, 32)])
def test_scratch_memory_of_a_packed_backward_follows_the_tokens(b, longest, total, h):
    """Whatever the longest sequence: 148 bytes for each head and row of 64-row tiles, of which a sequence fills all but one."""
    p = capi.FaDiffBwdParams()
    p.base.b, p.base.seqlen_q, p.base.seqlen_k, p.base.h, p.base.h_k, p.base.d = b, longest, longest, h, h, 64
    p.base.total_q = p.base.total_k = total
    p.base.cu_seqlens_q = p.base.cu_seqlens_k = 1 << 20  # never read
    got = capi.lib().fa_diff_bwd_workspace_bytes(ctypes.byref(p))
    assert total * h * 148 <= got <= (total + 64 * (b + 1)) * h * 148 + 1024
