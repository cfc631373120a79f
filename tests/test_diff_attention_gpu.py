"""Differential attention on the GPU against the definition in 64 bits (tests/diff_oracle.py derives the tolerances)."""
import pytest
import torch

import flash_attention_turing_b200 as fa
from diff_oracle import U, batch, check, check_dlam, sequence

pytestmark = pytest.mark.gpu


def _randn(gen, *shape):
    return torch.randn(*shape, generator=gen).half().cuda()


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _lam(gen, h, kind="fp32"):
    lam = torch.rand(h, generator=gen) * 1.2 - 0.2  # negative ones among them
    lam[0] = 0.0 if h > 2 else 0.7
    if kind == "one":
        lam = torch.tensor([0.55])
    return (lam.half() if kind == "fp16" else lam).cuda()


def _heads(lam, h):
    return lam.detach().float().expand(h) if lam.numel() == 1 else lam.detach()


DENSE = [  # b, sq, sk, h, hk, d, causal, lam
    (1, 1, 1, 1, 1, 64, False, "fp32"),
    (2, 1, 70, 4, 2, 128, True, "fp16"),
    (2, 5, 3, 3, 3, 64, True, "fp32"),      # rows without a visible key
    (1, 300, 77, 4, 1, 128, True, "one"),   # a whole tile without one
    (1, 128, 128, 2, 2, 128, False, "fp32"),
    (2, 129, 257, 4, 2, 64, False, "fp16"),
    (3, 257, 129, 2, 1, 128, False, "fp32"),
    (1, 513, 513, 8, 2, 128, True, "fp32"),
    (2, 200, 333, 6, 6, 64, True, "one"),
    (5, 384, 384, 12, 4, 64, True, "fp32"),
    (1, 1100, 1100, 16, 8, 128, True, "fp16"),
    (11, 40, 40, 2, 1, 128, True, "one"),
]


@pytest.mark.parametrize("b,sq,sk,h,hk,d,causal,kind", DENSE)
def test_dense_forward_and_gradients(b, sq, sk, h, hk, d, causal, kind):
    gen = _gen(1)
    q, k, v = _randn(gen, b, sq, h, d), _randn(gen, b, sk, hk, d), _randn(gen, b, sk, hk, d)
    lam, dout = _lam(gen, h, kind), _randn(gen, b, sq, h, d)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    out = fa.flash_diff_attn_func(*leaves, causal=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    want = batch(q, k, v, _heads(lam, h), causal, dout)
    check(out, want["out"], "out")
    for name, g in zip(("dq", "dk", "dv"), grads):
        check(g, want[name], name)
    assert grads[3].shape == lam.shape and grads[3].dtype == lam.dtype
    check_dlam(grads[3], want["dlam"])
    with torch.no_grad():
        assert torch.equal(out, fa.flash_diff_attn_func(*leaves, causal=causal))


def test_softmax_scale_and_large_scores():
    gen = _gen(2)
    q, k, v = _randn(gen, 1, 190, 2, 64) * 6, _randn(gen, 1, 190, 2, 64) * 6, _randn(gen, 1, 190, 2, 64)
    lam = _lam(gen, 2)
    out = fa.flash_diff_attn_func(q, k, v, lam, softmax_scale=0.3, causal=True)
    check(out, batch(q, k, v, lam, True, scale=0.3)["out"], "out")


def test_equal_maps_and_weight_one_cancel():
    gen = _gen(3)
    half = _randn(gen, 2, 150, 4, 64)
    q = torch.cat((half, half), -1)
    half = _randn(gen, 2, 150, 2, 64)
    k = torch.cat((half, half), -1)
    v, lam = _randn(gen, 2, 150, 2, 128), torch.ones(4, device="cuda")
    out = fa.flash_diff_attn_func(q, k, v, lam, causal=True)
    assert out.abs().max().item() <= 2 * U * 6  # the same numbers twice: only their rounding is left, of values below 6


def test_strided_inputs_and_gradient_of_expanded_weight():
    gen = _gen(4)
    qkv = _randn(gen, 2, 140, 3, 4, 64)
    q, k, v = (t.requires_grad_() for t in (qkv[:, :, 0], qkv[:, :, 1].transpose(1, 2).contiguous().transpose(1, 2), qkv[:, :, 2]))
    lam = torch.tensor([0.3, 9.0, 0.6, 9.0, 0.1, 9.0, 0.9, 9.0], device="cuda")[::2].requires_grad_()
    dout = _randn(gen, 2, 4, 140, 64).transpose(1, 2)
    out = fa.flash_diff_attn_func(q, k, v, lam, causal=True)
    got = torch.autograd.grad(out, (q, k, v, lam), dout)
    want = batch(q, k, v, lam, True, dout)
    check(out, want["out"], "out")
    for name, g in zip(("dq", "dk", "dv"), got):
        check(g, want[name], name)
    check_dlam(got[3], want["dlam"])
    one = torch.tensor(0.4, device="cuda", requires_grad=True)
    out = fa.flash_diff_attn_func(q, k, v, one.expand(4), causal=True)
    (g,) = torch.autograd.grad(out, one, dout)
    want = batch(q, k, v, one.detach().expand(4), True, dout)["dlam"]
    check_dlam(g, want)


def test_last_dimension_that_is_not_contiguous():
    gen = _gen(5)
    q, k, v = (_randn(gen, 1, 40, 64, 2).transpose(2, 3) for _ in range(3))
    lam = _lam(gen, 2)
    q.requires_grad_()
    out = fa.flash_diff_attn_func(q, k, v, lam)
    dout = _randn(gen, 1, 40, 64, 2).transpose(2, 3)
    (dq,) = torch.autograd.grad(out, q, dout)
    want = batch(q, k, v, lam, False, dout)
    check(out, want["out"], "out")
    check(dq, want["dq"], "dq")


def test_empty_inputs():
    for b, sq, sk in ((0, 4, 4), (2, 0, 4), (2, 4, 0)):
        q, k = torch.randn(b, sq, 2, 64, device="cuda").half(), torch.randn(b, sk, 2, 64, device="cuda").half()
        leaves = [t.requires_grad_() for t in (q, k, k.clone(), torch.rand(2, device="cuda"))]
        out = fa.flash_diff_attn_func(*leaves)
        assert out.shape == q.shape and not out.any()
        assert not any(g.any() for g in torch.autograd.grad(out.sum(), leaves))


@pytest.mark.parametrize("d,causal", [(64, True), (128, False)])
def test_gradients_against_differences(d, causal):
    """Along a random direction, against the central difference of the 64-bit forward.  The difference is off by its own
    third-order term, of which h = 1e-4 leaves about 1e-8 of the value; the kernel's share are its bounds."""
    gen = _gen(6)
    q, k, v = _randn(gen, 1, 70, 4, d), _randn(gen, 1, 90, 2, d), _randn(gen, 1, 90, 2, d)
    lam, dout = _lam(gen, 4), _randn(gen, 1, 70, 4, d)
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    grads = torch.autograd.grad(fa.flash_diff_attn_func(*leaves, causal=causal), leaves, dout)
    bounds = batch(q, k, v, lam, causal, dout)
    for i, name in enumerate(("dq", "dk", "dv", "dlam")):
        direction = torch.randn(leaves[i].shape, generator=gen).double().cuda()

        def loss(step):
            x = [t.detach().double() for t in leaves]
            x[i] = x[i] + step * direction
            return (batch(*x, causal)["out"][0] * dout.double()).sum().item()

        slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
        got = (grads[i].double() * direction).sum().item()
        bound = (bounds[name][1] * direction.abs()).sum().item()
        assert abs(got - slope) <= bound + 1e-5 * abs(slope) + 1e-5, (name, got, slope, bound)


VARLEN = [  # lengths q, lengths k (None: the same), h, hk, d, causal, spare rows
    ([1, 300, 0, 64, 129], None, 4, 2, 64, True, 0),
    ([200, 77], [130, 0], 4, 4, 128, False, 5),
    ([5, 140, 1], [3, 256, 7], 2, 1, 128, True, 200),
    ([700, 33, 260], None, 8, 2, 128, True, 3),
    ([i * 7 % 41 for i in range(21)], None, 3, 1, 64, True, 0),  # many short ones: dlam goes through them eight at a time
    ([90] + [3] * 8, None, 2, 2, 128, False, 2),
]


@pytest.mark.parametrize("lq,lk,h,hk,d,causal,spare", VARLEN)
def test_packed_sequences(lq, lk, h, hk, d, causal, spare):
    lk = lq if lk is None else lk
    gen = _gen(7)
    tq, tk = sum(lq) + spare, sum(lk) + spare
    q, k, v, dout = _randn(gen, tq, h, d), _randn(gen, tk, hk, d), _randn(gen, tk, hk, d), _randn(gen, tq, h, d)
    for t in (q, dout):
        t[sum(lq):] = float("nan")
    for t in (k, v):
        t[sum(lk):] = float("nan")
    lam = _lam(gen, h)
    ends = [torch.tensor([0] + x).cumsum(0).int().cuda() for x in (lq, lk)]
    leaves = [t.requires_grad_() for t in (q, k, v, lam)]
    out = fa.flash_diff_attn_varlen_func(*leaves, *ends, max(lq), max(lk), causal=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    assert not out[sum(lq):].any() and not grads[0][sum(lq):].any() and not grads[1][sum(lk):].any() and not grads[2][sum(lk):].any()
    dlam, bound = 0, 0
    for i in range(len(lq)):
        a, b = (slice(*e[i:i + 2].tolist()) for e in ends)
        want = sequence(q[a], k[b], v[b], lam, causal, dout[a])
        check(out[a], want["out"], "out")
        check(grads[0][a], want["dq"], "dq")
        check(grads[1][b], want["dk"], "dk")
        check(grads[2][b], want["dv"], "dv")
        dlam, bound = dlam + want["dlam"][0], bound + want["dlam"][1]
    check_dlam(grads[3], (dlam, bound))


@pytest.mark.parametrize("d", [64, 128])
def test_scratch_memory_may_hold_anything(d):
    """NaN wherever torch's allocator hands out memory: statistics of rows that do not exist are not written, and not used."""
    gen = _gen(13)
    lens, h, hk = [1, 65, 0, 127, 24, 200], 4, 2
    n = sum(lens)
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    lam = _lam(gen, h)
    packed = [_randn(gen, n, x, d) for x in (h, hk, hk, h)]
    dense = [_randn(gen, 2, 70, x, d) for x in (h, hk, hk, h)]

    def run(poison):
        out = []
        for x in (packed, dense):
            leaves = [t.detach().requires_grad_() for t in (*x[:3], lam)]
            if poison:
                torch.cuda.empty_cache()
                memory = torch.full((32 << 20,), 255, dtype=torch.uint8, device="cuda")
                del memory
            o = (fa.flash_diff_attn_varlen_func(*leaves, cu, cu, 200, 200, causal=True) if x is packed
                 else fa.flash_diff_attn_func(*leaves, causal=True))
            out += [o, *torch.autograd.grad(o, leaves, x[3])]
        return out

    for a, b in zip(run(True), run(False)):
        assert torch.isfinite(a).all() and torch.equal(a, b)


CACHE = [  # b, new, q rows, lengths, h, hk, d, page (0: contiguous), num_splits
    (1, 1, 1, [0], 2, 1, 64, 0, 0),
    (3, 1, 1, [0, 63, 500], 8, 2, 128, 0, 0),
    (4, 1, 1, [700, 1, 256, 255], 8, 4, 128, 256, 0),
    (2, 1, 1, [1999, 3], 4, 1, 64, 256, 3),
    (2, 2, 2, [300, 511], 16, 4, 64, 256, 0),
    (2, 1, 1, [900, 64], 32, 2, 128, 0, 2),       # 16 rows per KV head for each map
    (2, 0, 1, [900, 0], 4, 2, 128, 256, 0),       # nothing to append, an empty sequence
    (2, 3, 3, [40, 4000], 8, 8, 128, 512, 1),
    (3, 130, 130, [1, 300, 77], 4, 2, 64, 256, 0),  # a chunk of a prompt
    (2, 257, 257, [0, 511], 8, 2, 128, 256, 0),
    (2, 3, 3, [1500, 20], 16, 4, 128, 256, 0),    # 24 rows per KV head: two M tiles
    (1, 7, 7, [3001], 8, 2, 64, 0, 0),            # 56 rows, the last tile half full
    (3, 5, 5, [0, 130, 2], 6, 1, 128, 0, 4),      # 60 rows, groups of three
    (2, 8, 8, [700, 1], 8, 2, 64, 256, 1),        # 64 rows, one split
    (2, 9, 9, [700, 1], 8, 2, 64, 256, 0),        # 72 rows: the tiled kernel
    (1, 4, 4, [50000], 2, 1, 128, 0, 0),          # a long cache, shared out over many CTAs
    (1, 70, 70, [9000], 4, 2, 128, 256, 0),       # few row tiles, a long cache: its keys in parts
    (3, 140, 140, [5, 2500, 0], 4, 1, 64, 0, 3),  # parts that some rows have no key in
    (2, 100, 100, [1000, 3000], 8, 4, 64, 256, 1),
    (6, 130, 130, [0, 5000, 100, 7, 900, 300], 8, 2, 64, 256, 0),   # 96 row tiles, one long sequence: cut by the device's decision
    (4, 256, 200, [4000, 10, 3000, 300], 12, 4, 128, 512, 0),
    (6, 130, 130, [2500, 2000, 2300, 2700, 2100, 2900], 8, 2, 64, 0, 0),  # as many, nearly equal: not cut
    (3, 0, 500, [6000, 500, 0], 8, 8, 64, 256, 0),                  # nothing to append
    (64, 1, 1, list(range(5, 645, 10)), 4, 2, 64, 256, 0),
    (40, 1, 1, list(range(100, 4100, 100)), 8, 4, 128, 256, 0),
]


@pytest.mark.parametrize("b,new,rows,lengths,h,hk,d,page,splits", CACHE)
@pytest.mark.parametrize("check_on_host", [True, False])
def test_kvcache_step(b, new, rows, lengths, h, hk, d, page, splits, check_on_host, monkeypatch):
    from flash_attention_turing_b200 import flash_attention_interface as interface

    monkeypatch.setattr(interface, "HOST_CAPACITY_CHECK", check_on_host)
    gen = _gen(8)
    capacity = -(-(max(lengths) + new) // (page or 64)) * (page or 64)
    shape = (b * capacity // page, page) if page else (b, capacity)
    k_cache, v_cache = (torch.full((*shape, hk, d), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    table = torch.randperm(shape[0], generator=gen).int().cuda().view(b, -1) if page else None
    dense = []
    for i, n in enumerate(lengths):
        dense.append([_randn(gen, n, hk, d), _randn(gen, n, hk, d)])
        for cache, x in zip((k_cache, v_cache), dense[-1]):
            if page:
                for at in range(0, n, page):
                    cache[table[i, at // page], :min(page, n - at)] = x[at:at + page]
            else:
                cache[i, :n] = x
    q, lam = _randn(gen, b, rows, h, d), _lam(gen, h, "fp16")
    k, v = (_randn(gen, b, new, hk, d), _randn(gen, b, new, hk, d)) if new else (None, None)
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = fa.flash_diff_attn_with_kvcache(q, k_cache, v_cache, lam, k, v, cache_seqlens=lens, block_table=table, causal=True,
                                          num_splits=splits)
    for i, n in enumerate(lengths):
        kk, vv = (torch.cat((c, x[i])) if new else c for c, x in zip(dense[i], (k, v) if new else (None, None)))
        check(out[i], sequence(q[i], kk, vv, lam, True)["out"], f"sequence {i}")
        for cache, x in zip((k_cache, v_cache), (kk, vv)):
            whole = cache[table[i].long()].flatten(0, 1) if page else cache[i]
            assert torch.equal(whole[:n + new], x)
    assert fa.device_status() == 0


def test_kvcache_rows_of_a_cache_and_no_mask():
    gen = _gen(9)
    k_cache, v_cache = _randn(gen, 5, 128, 2, 64), _randn(gen, 5, 128, 2, 64)
    q, lam = _randn(gen, 2, 4, 4, 64), _lam(gen, 4, "one")
    idx = torch.tensor([3, 1], dtype=torch.int32, device="cuda")
    lens = torch.tensor([100, 17], dtype=torch.int32, device="cuda")
    out = fa.flash_diff_attn_with_kvcache(q, k_cache, v_cache, lam, cache_seqlens=lens, cache_batch_idx=idx)
    for i, (r, n) in enumerate(((3, 100), (1, 17))):
        check(out[i], sequence(q[i], k_cache[r, :n], v_cache[r, :n], _heads(lam, 4), False)["out"])
    with pytest.raises(ValueError, match="capacity"):
        fa.flash_diff_attn_with_kvcache(q, k_cache[:2], v_cache[:2], lam, cache_seqlens=lens + 29, causal=True)


def test_steps_equal_the_whole_sequence():
    """A prompt in chunks and single tokens against the cache, and the whole in one call."""
    gen = _gen(10)
    n, h, hk, d = 300, 8, 2, 128
    q, k, v, lam = _randn(gen, 1, n, h, d), _randn(gen, 1, n, hk, d), _randn(gen, 1, n, hk, d), _lam(gen, h)
    k_cache, v_cache = (torch.zeros(1, 512, hk, d, dtype=torch.float16, device="cuda") for _ in range(2))
    at, parts = 0, []
    for size in (200, 64, 30, 1, 1, 1, 2, 1):
        s = slice(at, at + size)
        parts.append(fa.flash_diff_attn_with_kvcache(q[:, s], k_cache, v_cache, lam, k[:, s], v[:, s], cache_seqlens=at, causal=True))
        at += size
    want = sequence(q[0], k[0], v[0], lam, True)["out"]
    check(torch.cat(parts, 1)[0], want, "steps")
    check(fa.flash_diff_attn_func(q, k, v, lam, causal=True)[0], want, "whole")


def test_on_a_host_thread_of_its_own():
    """Its first call of all is the operator's."""
    from concurrent.futures import ThreadPoolExecutor

    gen = _gen(15)
    q, k, v, lam = _randn(gen, 1, 140, 4, 64), _randn(gen, 1, 140, 2, 64), _randn(gen, 1, 140, 2, 64), _lam(gen, 4)
    want = fa.flash_diff_attn_func(q, k, v, lam)
    with ThreadPoolExecutor(1) as pool:
        assert torch.equal(pool.submit(fa.flash_diff_attn_func, q, k, v, lam).result(), want)
    with ThreadPoolExecutor(4) as pool:  # and several at once
        got = list(pool.map(lambda _: fa.flash_diff_attn_func(q, k, v, lam), range(16)))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)


def _training_step(gen):
    leaves = [t.requires_grad_() for t in (_randn(gen, 2, 260, 8, 64), _randn(gen, 2, 260, 2, 64), _randn(gen, 2, 260, 2, 64), _lam(gen, 8))]
    return leaves, _randn(gen, 2, 260, 8, 64)


def test_bitwise_reproducible_and_on_a_stream_of_its_own():
    leaves, dout = _training_step(_gen(11))
    out = fa.flash_diff_attn_func(*leaves, causal=True)
    first = [out.detach(), *torch.autograd.grad(out, leaves, dout)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams * 3:  # two calls in flight at once
        with torch.cuda.stream(s):
            out = fa.flash_diff_attn_func(*leaves, causal=True)
            results.append([out.detach(), *torch.autograd.grad(out, leaves, dout)])
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(a, b) for a, b in zip(first, r))


def test_training_step_in_a_cuda_graph():
    gen = _gen(12)
    leaves, dout = _training_step(gen)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out = fa.flash_diff_attn_func(*leaves, causal=True)
        torch.autograd.grad(out, leaves, dout)
    torch.cuda.current_stream().wait_stream(side)
    alive = fa.flash_diff_attn_func(*leaves, causal=True)  # an eager graph of the same leaves
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fa.flash_diff_attn_func(*leaves, causal=True)
        grads = torch.autograd.grad(out, leaves, dout)
    with torch.no_grad():
        for t in (*leaves[:3], dout):
            t.copy_(_randn(gen, *t.shape))
    for _ in range(3):
        graph.replay()
    want = batch(*leaves, True, dout)
    check(out, want["out"], "out")
    for name, g in zip(("dq", "dk", "dv"), grads):
        check(g, want[name], name)
    check_dlam(grads[3], want["dlam"])
    del alive


def test_decode_in_a_cuda_graph(monkeypatch):
    from flash_attention_turing_b200 import flash_attention_interface as interface

    monkeypatch.setattr(interface, "HOST_CAPACITY_CHECK", False)
    gen = _gen(13)
    k_cache, v_cache, lam = _randn(gen, 2, 512, 2, 64), _randn(gen, 2, 512, 2, 64), _lam(gen, 4)
    q, k, v = _randn(gen, 2, 1, 4, 64), _randn(gen, 2, 1, 2, 64), _randn(gen, 2, 1, 2, 64)
    lens = torch.tensor([400, 77], dtype=torch.int32, device="cuda")

    def step():
        return fa.flash_diff_attn_with_kvcache(q, k_cache, v_cache, lam, k, v, cache_seqlens=lens, causal=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
        lens.add_(1)
    for _ in range(3):
        for t in (q, k, v):
            t.copy_(_randn(gen, *t.shape))
        n = lens.tolist()
        graph.replay()
        for i in range(2):
            check(out[i], sequence(q[i], k_cache[i, :n[i] + 1], v_cache[i, :n[i] + 1], lam, True)["out"])
            assert torch.equal(k_cache[i, n[i]], k[i, 0])


def test_chunks_in_a_cuda_graph_with_other_lengths(monkeypatch):
    """96 row tiles: whether the keys are cut is decided on the device, at every replay anew."""
    from flash_attention_turing_b200 import flash_attention_interface as interface

    monkeypatch.setattr(interface, "HOST_CAPACITY_CHECK", False)
    gen = _gen(14)
    b, rows, h, hk, d, capacity = 6, 130, 8, 2, 64, 5376
    k_cache, v_cache, lam = _randn(gen, b, capacity, hk, d), _randn(gen, b, capacity, hk, d), _lam(gen, h)
    q, k, v = _randn(gen, b, rows, h, d), _randn(gen, b, rows, hk, d), _randn(gen, b, rows, hk, d)
    lens = torch.zeros(b, dtype=torch.int32, device="cuda")

    def step():
        return fa.flash_diff_attn_with_kvcache(q, k_cache, v_cache, lam, k, v, cache_seqlens=lens, causal=True)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for lengths in ([0] * 6, [5200, 10, 0, 700, 300, 90], [2000, 2100, 1900, 2050, 1800, 2200], [3, 4000, 8, 100, 5246, 60]):
        lens.copy_(torch.tensor(lengths, dtype=torch.int32))
        graph.replay()
        for i, n in enumerate(lengths):
            check(out[i], sequence(q[i], k_cache[i, :n + rows], v_cache[i, :n + rows], lam, True)["out"], f"{lengths} {i}")


def test_parameter_and_the_class_behind_the_native_node():
    gen = _gen(14)
    q, k, v, lam = _randn(gen, 1, 40, 2, 64), _randn(gen, 1, 40, 2, 64), _randn(gen, 1, 40, 2, 64), _lam(gen, 2)
    p = torch.nn.Parameter(lam)
    out = fa.flash_diff_attn_func(q, k, v, p, 64 ** -1)  # a scale that is a float
    out.sum().backward()
    check_dlam(p.grad, batch(q, k, v, lam, False, torch.ones_like(q), 64 ** -1)["dlam"])
    scale = torch.tensor(0.2).item()
    a = fa.flash_diff_attn_func(q, k, v, lam, scale)
    b = fa.diff_attention_interface.FlashDiffAttnFunc.apply(q, k, v, lam, scale, False, True)
    assert torch.equal(a, b)


@pytest.mark.parametrize("packed", [False, True])
def test_transforms_and_modes_go_to_the_class(packed):
    """functorch transforms and forward-mode AD are refused, a mode and a tensor subclass reach the class; saved tensors are guarded."""
    from torch.overrides import TorchFunctionMode

    gen, module = _gen(16), fa.diff_attention_interface
    shape = (40,) if packed else (1, 40)
    inputs = [_randn(gen, *shape, 2, 64), _randn(gen, *shape, 2, 64), _randn(gen, *shape, 2, 64), _lam(gen, 2)]
    cu = torch.tensor([0, 15, 40], dtype=torch.int32, device="cuda")
    cls = module.FlashDiffAttnVarlenFunc if packed else module.FlashDiffAttnFunc

    def call(*x):
        return fa.flash_diff_attn_varlen_func(*x, cu, cu, 25, 25, causal=True) if packed else fa.flash_diff_attn_func(*x, causal=True)

    with pytest.raises(RuntimeError, match="functorch transforms"):
        torch.func.vmap(call)(*(x[None] for x in inputs))
    with torch.autograd.forward_ad.dual_level():
        for i in (0, 3):
            dual = [torch.autograd.forward_ad.make_dual(x, torch.ones_like(x)) if i == j else x for j, x in enumerate(inputs)]
            with pytest.raises((RuntimeError, NotImplementedError)):
                call(*dual)
    want, applied, real = call(*inputs), [], cls.apply
    try:
        cls.apply = classmethod(lambda c, *a: applied.append(1) or real(*a))

        class Mode(TorchFunctionMode):
            def __torch_function__(self, func, types, args=(), kwargs=None):
                return func(*args, **(kwargs or {}))

        with Mode():
            assert torch.equal(call(*inputs), want)
        sub = call(inputs[0].as_subclass(type("Sub", (torch.Tensor,), {})), *inputs[1:])
        assert torch.equal(sub.as_subclass(torch.Tensor), want) and len(applied) == 2
    finally:
        del cls.apply
    leaves, dout = [x.clone().requires_grad_() for x in inputs], _randn(gen, *inputs[0].shape)
    out = call(*leaves)
    native = torch.autograd.grad(out, leaves, dout, retain_graph=True)
    extra = (cu, cu, 25, 25) if packed else ()
    by_class = torch.autograd.grad(cls.apply(*leaves, *extra, None, True, True), leaves, dout)
    assert all(torch.equal(a, b) for a, b in zip(native, by_class))
    with torch.no_grad():
        leaves[3].add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, dout)


def test_refusals():
    q, k, lam = torch.zeros(1, 4, 4, 64, device="cuda").half(), torch.zeros(1, 4, 2, 64, device="cuda").half(), torch.zeros(4, device="cuda")
    for args, text in (
        ((q.float(), k, k, lam), "float16"),
        ((q, k, k, lam.cpu()), "lam must be a CUDA tensor"),
        ((q, k, k, lam.double()), "lam must be a float32 or float16"),
        ((q, k, k, lam[:3]), "one element or shape"),
        ((q, k, k, lam.view(2, 2)), "one element or shape"),
        ((q[..., :32], k[..., :32], k[..., :32], lam), "head_dim"),
        ((q[:, :, :3], k, k, lam[:3]), "divisible"),
        ((q, k, k[:, :3], lam), "seqlen_k"),
        ((q.cpu(), k, k, lam), "CUDA"),
    ):
        with pytest.raises(RuntimeError, match=text):
            fa.flash_diff_attn_func(*args)
    for scale in (0.0, -0.1, float("nan")):
        with pytest.raises(RuntimeError, match="softmax_scale"):
            fa.flash_diff_attn_func(q, k, k, lam, softmax_scale=scale)
        with pytest.raises(RuntimeError, match="softmax_scale"):
            fa.flash_diff_attn_with_kvcache(q, k, k, lam, cache_seqlens=2, softmax_scale=scale)
    with pytest.raises(RuntimeError, match="same number of rows"):
        fa.flash_diff_attn_with_kvcache(q, k, k.expand(2, -1, -1, -1), lam, cache_seqlens=2)
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="int32"):
        fa.flash_diff_attn_varlen_func(q[0], k[0], k[0], lam, cu.long(), cu, 4, 4)
    with pytest.raises(TypeError, match="lam"):
        fa.flash_diff_attn_with_kvcache(q, k, k, 0.5)
    with pytest.raises(RuntimeError, match="lam must be"):
        fa.flash_diff_attn_with_kvcache(q, k, k, lam.double(), cache_seqlens=2)
    assert fa.device_status() == 0


@pytest.mark.parametrize("lens,longest,d,causal", [([150, 40], 100, 64, True), ([70, 400, 3], 130, 128, False), ([129], 128, 128, True), ([300, 300], 1, 64, False)])
def test_sequences_longer_than_the_given_maximum(lens, longest, d, causal):
    """Rows past max_seqlen_q have no place in the LSE: they are zero and count for nothing, whatever the memory held before."""
    gen = _gen(17)
    n, h, hk = sum(lens), 4, 2
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    leaves = [t.requires_grad_() for t in (_randn(gen, n, h, d), _randn(gen, n, hk, d), _randn(gen, n, hk, d), _lam(gen, h))]
    dout = _randn(gen, n, h, d)
    torch.cuda.empty_cache()
    memory = torch.full((32 << 20,), 255, dtype=torch.uint8, device="cuda")
    del memory
    out = fa.flash_diff_attn_varlen_func(*leaves, cu, cu, longest, max(lens), causal=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    dlam, bound = 0, 0
    for a, b in zip(cu.tolist(), cu.tolist()[1:]):
        s, past = slice(a, b), slice(min(a + longest, b), b)
        counted = dout[s].clone()
        counted[longest:] = 0
        want = sequence(leaves[0][s], leaves[1][s], leaves[2][s], leaves[3], causal, counted)
        check(out[a:past.start], tuple(t[:longest] for t in want["out"]), "out")
        assert not out[past].any() and not grads[0][past].any()
        check(grads[0][a:past.start], tuple(t[:longest] for t in want["dq"]), "dq")
        check(grads[1][s], want["dk"], "dk")
        check(grads[2][s], want["dv"], "dv")
        dlam, bound = dlam + want["dlam"][0], bound + want["dlam"][1]
    check_dlam(grads[3], (dlam, bound))
    assert fa.device_status() == 0


@pytest.mark.parametrize("h,hk,d,causal", [(3, 1, 64, True), (2, 2, 128, False)])
def test_one_long_sequence_among_many_short_ones(h, hk, d, causal):
    """Sequences that begin anywhere in the 64-row tiles of the scratch memory, in the middle of a batch and at its ends."""
    gen = _gen(18)
    lens = [3, 0, 61, 64, 1] + [i * 5 % 23 for i in range(60)] + [1500] + [(i * 7 + 1) % 90 for i in range(60)] + [128, 0, 65]
    n = sum(lens)
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    leaves = [t.requires_grad_() for t in (_randn(gen, n, h, d), _randn(gen, n, hk, d), _randn(gen, n, hk, d), _lam(gen, h))]
    dout = _randn(gen, n, h, d)
    torch.cuda.empty_cache()
    memory = torch.full((64 << 20,), 255, dtype=torch.uint8, device="cuda")
    del memory
    out = fa.flash_diff_attn_varlen_func(*leaves, cu, cu, 1500, 1500, causal=causal)
    grads = torch.autograd.grad(out, leaves, dout)
    dlam, bound = 0, 0
    for a, b in zip(cu.tolist(), cu.tolist()[1:]):
        s = slice(a, b)
        want = sequence(leaves[0][s], leaves[1][s], leaves[2][s], leaves[3], causal, dout[s])
        for x, name in zip((out, *grads[:3]), ("out", "dq", "dk", "dv")):
            check(x[s], want[name], name)
        dlam, bound = dlam + want["dlam"][0], bound + want["dlam"][1]
    check_dlam(grads[3], (dlam, bound))


def test_no_key_heads():
    """Refused by every entry point, plain and differential: the number of query heads is not divided by zero."""
    q, k, lam = torch.zeros(1, 4, 4, 64, device="cuda").half(), torch.zeros(1, 4, 0, 64, device="cuda").half(), torch.zeros(4, device="cuda")
    cu = torch.tensor([0, 4], dtype=torch.int32, device="cuda")
    for more in ((), (lam,)):
        names = ("flash_diff_attn_func", "flash_diff_attn_varlen_func", "flash_diff_attn_with_kvcache") if more else (
            "flash_attn_func", "flash_attn_varlen_func", "flash_attn_with_kvcache")
        dense, packed, cached = (getattr(fa, n) for n in names)
        for call in (lambda: dense(q, k, k, *more), lambda: packed(q[0], k[0], k[0], *more, cu, cu, 4, 4),
                     lambda: cached(q, k, k, *more, cache_seqlens=2), lambda: cached(q, k, k, *more, k, k, cache_seqlens=0)):
            with pytest.raises((RuntimeError, ValueError)):
                call()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="a tensor on another device")
def test_a_cache_index_on_another_device_is_refused():
    q, k, lam = torch.zeros(1, 1, 4, 64, device="cuda:0").half(), torch.zeros(1, 64, 2, 64, device="cuda:0").half(), torch.zeros(4, device="cuda:0")
    idx = torch.zeros(1, dtype=torch.int32, device="cuda:1")
    with pytest.raises(RuntimeError, match="device of q"):
        fa.flash_diff_attn_with_kvcache(q, k, k, lam, cache_seqlens=2, cache_batch_idx=idx)


def test_keys_past_the_given_maximum():
    """They are attended, and have no gradients from the next whole tile on."""
    gen = _gen(19)
    lens, h, hk, d = [300, 40], 4, 2, 64
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    leaves = [t.requires_grad_() for t in (_randn(gen, 340, h, d), _randn(gen, 340, hk, d), _randn(gen, 340, hk, d), _lam(gen, h))]
    dout = _randn(gen, 340, h, d)
    torch.cuda.empty_cache()
    memory = torch.full((32 << 20,), 255, dtype=torch.uint8, device="cuda")
    del memory
    out = fa.flash_diff_attn_varlen_func(*leaves, cu, cu, 300, 100, causal=True)
    grads = torch.autograd.grad(out, leaves, dout)
    for a, b in zip(cu.tolist(), cu.tolist()[1:]):
        s, n = slice(a, b), min(b - a, 128)
        want = sequence(leaves[0][s], leaves[1][s], leaves[2][s], leaves[3], True, dout[s])
        check(out[s], want["out"], "out")
        check(grads[0][s], want["dq"], "dq")
        for i, name in ((1, "dk"), (2, "dv")):
            check(grads[i][a:a + n], tuple(t[:n] for t in want[name]), name)
            assert not grads[i][a + n:b].any()
