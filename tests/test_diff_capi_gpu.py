"""Differential attention and the page functions through the C interface: raw pointers, strides, scratch memory of exactly the size that the
queries ask for, against the definition in 64 bits."""
import ctypes

import pytest
import torch

import flash_attention_turing_b200 as fa
from diff_oracle import check, check_dlam, sequence, visible
from flash_attention_turing_b200 import capi

pytestmark = pytest.mark.gpu

SHIFT = 2  # FA_CAUSAL_SHIFT
CLEAR_FORWARD, CLEAR_BACKWARD = 1, 2  # FA_FWD_ZERO_UNUSED_ROWS, FA_BWD_ZERO_UNUSED_ROWS


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen).half().cuda()


def _stream():
    return ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)


class Guarded:
    """A buffer of `bytes` at an address aligned to 256 bytes, with known bytes on both sides."""

    def __init__(self, bytes):
        self.bytes = bytes
        self.memory = torch.full((bytes + 1024,), 0x5A, dtype=torch.uint8, device="cuda")
        self.ptr = self.memory.data_ptr() + 512
        assert self.ptr % 256 == 0
        self.inside = self.memory[512:512 + bytes]
        self.inside.fill_(0xFF)  # NaN in every type

    def check(self):
        assert (self.memory[:512] == 0x5A).all() and (self.memory[512 + self.bytes:] == 0x5A).all()


def _strides(p, name, x):
    batch = x.stride(0) if x.dim() == 4 else 0
    for part, value in zip(("batch", "row", "head"), (batch, x.stride(-3), x.stride(-2))):
        setattr(p, f"{name}_{part}_stride", value)


def _weights(lam, h):
    return capi.FaDiffWeights(lam.data_ptr(), lam.stride(0) if lam.dim() else 0, lam.numel(), int(lam.dtype == torch.float16))


def _forward(q, k, v, lam, scale, causal, pitch, shift=0, cu=None, longest=None, keep=True):
    """pitch: lse_row_stride.  (out, o2, lse (b, 2 h, pitch))"""
    p = capi.FaDiffFwdParams()
    b = cu.numel() - 1 if cu is not None else q.shape[0]
    h, d = q.shape[-2:]
    out, o2 = torch.full_like(q, float("nan")), torch.full_like(q, float("nan"))
    lse = Guarded(b * 2 * h * pitch * 4)
    f = p.base
    f.q, f.k, f.v, f.o, f.lse = q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), lse.ptr
    for name, x in (("q", q), ("k", k), ("v", v), ("o", out)):
        _strides(f, name, x)
    f.lse_row_stride, f.b, f.h, f.h_k, f.d = pitch, b, h, k.shape[-2], d
    f.softmax_scale, f.is_causal, f.causal_shift = scale, causal, shift
    if cu is None:
        f.seqlen_q, f.seqlen_k, f.k_batch = q.shape[1], k.shape[1], b
    else:
        f.seqlen_q = f.seqlen_k = longest
        f.total_q, f.total_k = q.shape[0], k.shape[0]
        f.cu_seqlens_q = f.cu_seqlens_k = cu.data_ptr()
        f.flags = CLEAR_FORWARD
    p.weights = _weights(lam, h)
    if keep:
        p.o2 = o2.data_ptr()
        _strides(p, "o2", o2)
    capi.check(capi.lib().fa_diff_fwd(ctypes.byref(p), _stream()))
    lse.check()
    return out, o2, lse.inside.view(torch.float32).view(b, 2 * h, pitch)


def _backward(q, k, v, lam, out, o2, lse, dout, scale, causal, shift=0, cu=None, longest=None):
    p = capi.FaDiffBwdParams()
    h, d = q.shape[-2:]
    grads = [torch.full_like(t, float("nan")) for t in (q, k, v)]
    dlam = torch.full((lam.numel(),), float("nan"), dtype=lam.dtype, device="cuda")
    f = p.base
    f.q, f.k, f.v, f.o, f.dout, f.lse = (t.data_ptr() for t in (q, k, v, out, dout, lse))
    f.dq, f.dk, f.dv = (t.data_ptr() for t in grads)
    for name, x in (("q", q), ("k", k), ("v", v), ("o", out), ("do", dout), *zip(("dq", "dk", "dv"), grads)):
        _strides(f, name, x)
    f.lse_row_stride, f.b, f.h, f.h_k, f.d = lse.shape[2], lse.shape[0], h, k.shape[-2], d
    f.softmax_scale, f.is_causal, f.causal_shift = scale, causal, shift
    if cu is None:
        f.seqlen_q, f.seqlen_k = q.shape[1], k.shape[1]
    else:
        f.seqlen_q = f.seqlen_k = longest
        f.total_q, f.total_k = q.shape[0], k.shape[0]
        f.cu_seqlens_q = f.cu_seqlens_k = cu.data_ptr()
        f.flags = CLEAR_BACKWARD
    p.weights, p.o2, p.dlam = _weights(lam, h), o2.data_ptr(), dlam.data_ptr()
    _strides(p, "o2", o2)
    lib = capi.lib()
    scratch = Guarded(lib.fa_diff_bwd_workspace_bytes(ctypes.byref(p)))
    f.workspace, f.workspace_bytes = scratch.ptr, scratch.bytes - 1
    assert lib.fa_diff_bwd(ctypes.byref(p), _stream()) == -3
    f.workspace_bytes = scratch.bytes
    capi.check(lib.fa_diff_bwd(ctypes.byref(p), _stream()))
    scratch.check()
    return (*grads, dlam)


def _check_lse(got, q, k, scale, seen):
    """One sequence: got (2 h, sq).  The scores' and the exponentials' errors: 2^-21 (1 + |s|) and 2.7e-6, the sum and the logarithm less."""
    if q.shape[0] == 0:
        return
    q, k = q.double(), k.double().repeat_interleave(q.shape[1] // k.shape[1], 1)
    for m in (0, 1):
        s = torch.einsum("ihd,jhd->hij", q.chunk(2, -1)[m], k.chunk(2, -1)[m]) * scale
        bound = 2.0 ** -18 * (1 + s.abs().amax(-1))
        want = torch.logsumexp(torch.where(seen, s, -torch.inf), -1)
        want = torch.where(seen.any(-1), want, 0.0)
        assert ((got[m::2].double() - want).abs() <= bound).all()


@pytest.mark.parametrize("b,sq,sk,h,hk,d,causal,shift,one", [
    (2, 70, 200, 4, 2, 64, 0, 0, False), (1, 130, 130, 2, 1, 128, 1, 0, True),
    (2, 150, 300, 4, 2, 64, SHIFT, 0, False), (2, 150, 300, 2, 2, 128, SHIFT, 77, False), (1, 200, 150, 4, 1, 64, SHIFT, -60, False),
    (1, 257, 140, 2, 2, 128, SHIFT, -130, True), (1, 64, 64, 2, 1, 64, SHIFT, 500, False), (1, 90, 300, 2, 1, 64, SHIFT, -500, False)])
def test_dense(b, sq, sk, h, hk, d, causal, shift, one):
    gen = torch.Generator().manual_seed(1)
    q, dout = (_randn(gen, b, sq, 2 * h, d)[:, :, ::2] for _ in range(2))  # every other head of a wider tensor
    k, v = _randn(gen, b, sk, hk, d), _randn(gen, b, sk + 3, hk, d)[:, 3:]
    lam = torch.tensor([0.45], device="cuda").half() if one else torch.rand(2 * h, generator=gen).cuda()[::2]
    scale, pitch = (d // 2) ** -0.5, sq + 5
    out, o2, lse = _forward(q, k, v, lam, scale, causal, pitch, shift)
    grads = _backward(q, k, v, lam, out, o2, lse, dout, scale, causal, shift)
    assert torch.isnan(lse[:, :, sq:]).all()  # between the rows nothing is written
    lam = lam.float().expand(h)
    # the keys that a call with a diagonal at `shift` has: as many as put it at the bottom right
    n = sk if causal != SHIFT else max(0, min(sk, sq + shift))
    at_corner = causal == 1 or (causal == SHIFT and sq + shift <= sk and n > 0)
    dlam, bound = 0, 0
    for i in range(b):
        if causal == SHIFT and n == 0:
            assert not out[i].any() and all(not g[i].any() for g in grads[:3]) and not lse[i, :, :sq].any()
            continue
        want = sequence(q[i], k[i, :n], v[i, :n], lam, at_corner, dout[i])
        _check_lse(lse[i, :, :sq], q[i], k[i, :n], scale, visible(sq, n, at_corner, "cuda"))
        check(out[i], want["out"], "out")
        check(grads[0][i], want["dq"], "dq")
        check(grads[1][i, :n], want["dk"], "dk")
        check(grads[2][i, :n], want["dv"], "dv")
        assert not grads[1][i, n:].any() and not grads[2][i, n:].any()
        dlam, bound = dlam + want["dlam"][0], bound + want["dlam"][1]
    if torch.is_tensor(dlam):
        check_dlam(grads[3], (dlam, bound))
    else:
        assert not grads[3].any()
    plain, _, _ = _forward(q, k, v, lam if not one else torch.tensor([0.45], device="cuda").half(), scale, causal, pitch, shift, keep=False)
    assert torch.equal(plain, out)
    assert fa.device_status() == 0


@pytest.mark.parametrize("pitch", [300, 384])
def test_packed(pitch):
    """base.lse is (b, 2 h, lse_row_stride): a row of the longest sequence's length at least for each sequence, map and head."""
    gen = torch.Generator().manual_seed(2)
    lens, h, hk, d, spare = [40, 300, 0, 129], 4, 2, 64, 7
    n = sum(lens) + spare
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    q, k, v, dout = (_randn(gen, n, x, d) for x in (h, hk, hk, h))
    lam = torch.rand(h, generator=gen).cuda()
    scale = (d // 2) ** -0.5
    out, o2, lse = _forward(q, k, v, lam, scale, 1, pitch, cu=cu, longest=300)
    grads = _backward(q, k, v, lam, out, o2, lse, dout, scale, 1, cu=cu, longest=300)
    for t in (out, *grads[:3]):
        assert not t[n - spare:].any()
    dlam, bound = 0, 0
    for i, (a, b) in enumerate(zip(cu.tolist(), cu.tolist()[1:])):
        s = slice(a, b)
        want = sequence(q[s], k[s], v[s], lam, True, dout[s])
        _check_lse(lse[i, :, :b - a], q[s], k[s], scale, visible(b - a, b - a, True, "cuda"))
        for x, name in zip((out, *grads[:3]), ("out", "dq", "dk", "dv")):
            check(x[s], want[name], name)
        dlam, bound = dlam + want["dlam"][0], bound + want["dlam"][1]
    check_dlam(grads[3], (dlam, bound))


@pytest.mark.parametrize("b,new,lengths,h,hk,d,page,splits", [
    (2, 1, [700, 63], 4, 2, 64, 0, 0), (2, 1, [1999, 300], 8, 4, 128, 256, 3), (1, 1, [0], 2, 1, 64, 256, 0), (2, 5, [700, 90], 16, 4, 64, 256, 0),
    (2, 130, [300, 77], 4, 2, 64, 256, 1), (1, 70, [4000], 4, 2, 128, 64, 1), (1, 70, [4000], 4, 2, 128, 256, 0),
    (6, 130, [0, 5000, 100, 7, 900, 300], 8, 2, 64, 256, 0)])
@pytest.mark.parametrize("checked", [True, False])
def test_cache_step(b, new, lengths, h, hk, d, page, splits, checked):
    gen = torch.Generator().manual_seed(3)
    unit = max(page, 128)
    capacity = -(-(max(lengths) + new) // unit) * unit
    if page == 64:
        page = 128  # what the tiled kernel takes as well
    rows = (b * capacity // page, page) if page else (b, capacity)
    k_cache, v_cache = _randn(gen, *rows, hk, d), _randn(gen, *rows, hk, d)
    table = torch.randperm(rows[0], generator=gen).int().cuda().view(b, -1) if page else None
    q, k, v = _randn(gen, b, new, h, d), _randn(gen, b, new, hk, d), _randn(gen, b, new, hk, d)
    lam, lens = torch.rand(h, generator=gen).cuda(), torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out, lse = torch.full_like(q, float("nan")), Guarded(b * 2 * h * new * 4)
    p = capi.FaDiffKvcacheParams()
    as_lse = lse.inside.view(torch.float32).view(b, 2 * h, new)
    p.base = capi.kvcache_params(q, k_cache, v_cache, k, v, out, as_lse, lens, table, (d // 2) ** -0.5, True, splits)
    p.weights = _weights(lam, h)
    lib = capi.lib()
    scratch = Guarded(lib.fa_diff_kvcache_workspace_bytes(ctypes.byref(p)))
    p.base.workspace, p.base.workspace_bytes = scratch.ptr if scratch.bytes else None, scratch.bytes
    word = torch.full((1,), -1, dtype=torch.int32).pin_memory()
    capi.check(lib.fa_diff_kvcache(ctypes.byref(p), word.data_ptr() if checked else None, 9, _stream()))
    torch.cuda.synchronize()
    assert word.item() == (18 if checked else -1)
    scratch.check()
    lse.check()
    for i, n in enumerate(lengths):
        keys, values = ((c[table[i].long()].flatten(0, 1) if page else c[i])[:n + new] for c in (k_cache, v_cache))
        assert torch.equal(keys[n:], k[i]) and torch.equal(values[n:], v[i])
        check(out[i], sequence(q[i], keys, values, lam, True)["out"], f"sequence {i}")
        _check_lse(as_lse[i], q[i], keys, (d // 2) ** -0.5, visible(new, n + new, True, "cuda"))
    # new tokens that are only announced are refused, and nothing is launched
    p.base.k_new = p.base.v_new = None
    assert lib.fa_diff_kvcache(ctypes.byref(p), None, 0, _stream()) == -1 and b"without k_new" in lib.fa_last_error()
    assert fa.device_status() == 0


def test_pages():
    """A prompt, two forks of it, one freed, and the pool compacted: the same tables and pages as through the Python functions."""
    lib, rows, columns, pages, page, hk, d = capi.lib(), 40, 5, 30, 64, 2, 64
    new = torch.zeros(rows, dtype=torch.int32, device="cuda")
    new[:2] = torch.tensor([150, 64])
    parents, children, gone = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1, 0, -1], [3, 4, 3, 5], [0, -1, 99]))
    src, dst = (torch.tensor(x, dtype=torch.int32, device="cuda") for x in ([0, 1], [20, 29]))
    base = [torch.randn(pages + 1, page, hk, d, generator=torch.Generator().manual_seed(i)).half().cuda() for i in range(3)]

    def fresh():
        table = torch.full((rows, columns + 2), -1, dtype=torch.int32, device="cuda")[:, :columns]
        return table, *(torch.zeros(n, dtype=torch.int32, device="cuda") for n in (rows, pages)), [t.clone()[:pages] for t in base]

    table, lens, refs, caches = fresh()
    want = [fa.kvcache_reserve(table, lens, refs, new, page)]
    lens += new
    want += [fa.kvcache_fork(caches, table, lens, refs, parents, children), fa.kvcache_copy_pages(caches, src, dst)]
    fa.kvcache_free(table, lens, refs, gone)
    want += [fa.kvcache_compact(caches, table, refs), table, lens, refs, *caches]

    table, lens, refs, caches = fresh()
    t = capi.FaPageTables(table.data_ptr(), lens.data_ptr(), refs.data_ptr(), table.stride(0), rows, columns, pages)
    c = capi.FaPageCaches((ctypes.c_void_p * 3)(*(x.data_ptr() for x in caches)), (ctypes.c_int64 * 3)(*[page * hk * d * 2] * 3), page * hk * d * 2, 3)
    t_, c_ = ctypes.byref(t), ctypes.byref(c)

    def scratch(size):
        g = Guarded(size)
        return g, (g.ptr if size else None), size

    flags = [torch.full((n,), 7, dtype=torch.uint8, device="cuda") for n in (rows, 4, 2)]
    live = torch.full((1,), -1, dtype=torch.int32, device="cuda")
    for always in (False, True):  # scratch memory where it is needed, and the largest size for every call
        if always:
            table, lens, refs, caches = fresh()
            t.block_table, t.cache_seqlens, t.page_refs = table.data_ptr(), lens.data_ptr(), refs.data_ptr()
            c.base = (ctypes.c_void_p * 3)(*(x.data_ptr() for x in caches))
        size = lambda own, n: lib.fa_pages_workspace_bytes(rows, pages, n) if always else own  # noqa: E731
        g, at, bytes = scratch(size(lib.fa_pages_reserve_workspace_bytes(t_), 0))
        capi.check(lib.fa_pages_reserve(t_, new.data_ptr(), 0, page, flags[0].data_ptr(), at, bytes, _stream()))
        lens += new
        g2, at, bytes = scratch(size(lib.fa_pages_fork_workspace_bytes(t_, c_, 4), 4))
        capi.check(lib.fa_pages_fork(t_, c_, parents.data_ptr(), children.data_ptr(), 4, page, flags[1].data_ptr(), at, bytes, _stream()))
        g3, at, bytes = scratch(size(lib.fa_pages_copy_workspace_bytes(c_, pages, 2), 2))
        capi.check(lib.fa_pages_copy(c_, pages, src.data_ptr(), dst.data_ptr(), 2, flags[2].data_ptr(), at, bytes, _stream()))
        capi.check(lib.fa_pages_free(t_, gone.data_ptr(), 3, _stream()))
        g4, at, bytes = scratch(lib.fa_pages_workspace_bytes(rows, pages, 0))
        capi.check(lib.fa_pages_compact(t_, c_, live.data_ptr(), at, bytes, _stream()))
        for guard in (g, g2, g3, g4):
            guard.check()
        for a, b in zip((*(f.bool() for f in flags), live, table, lens, refs, *caches), (want[0], want[1], want[2], *want[3:])):
            assert torch.equal(a, b)
    # 3 + 1 pages, one more for the copy of a tail, and the prompt's own tail is free again
    assert want[1].tolist() == [True, True, False, False] and want[3].item() == 4
