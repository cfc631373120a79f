"""NaN and infinities in q, k and v of differential attention: what they reach by the definition is not finite, whichever kernel runs, and
everything else has the bits that it has without them."""
import math

import pytest
import torch

import flash_attention_turing_b200 as fa

pytestmark = pytest.mark.gpu

NAN, INF = float("nan"), float("inf")


def _rand(gen, *shape):
    """Queries and keys of one sign, so that an infinite element of a key is an infinite score of every query."""
    return (torch.rand(*shape, generator=gen) + 0.1).half().cuda()


def _definition(q, k, v, lam, causal):
    """One sequence in 64 bits: q (sq, h, d), k, v (sk, hk, d).  Only rows without a visible key are zero."""
    q, k, v = (t.double() for t in (q, k, v))
    (sq, h, d), (sk, hk) = q.shape, k.shape[:2]
    i, j = torch.arange(sq, device=q.device)[:, None], torch.arange(sk, device=q.device)[None]
    seen = j <= i + sk - sq if causal else torch.ones(sq, sk, dtype=torch.bool, device=q.device)
    k, v = (t.repeat_interleave(h // hk, 1) for t in (k, v))
    out = 0
    for m, f in ((0, torch.ones_like(lam)), (1, -lam)):
        a, b = q.chunk(2, -1)[m], k.chunk(2, -1)[m]
        s = torch.einsum("ihd,jhd->hij", a, b) * (d // 2) ** -0.5
        p = torch.softmax(torch.where(seen, s, -math.inf), -1)
        p = torch.where(seen.any(-1, keepdim=True), p, 0.0)
        out = out + torch.einsum("hij,jhd->ihd", p, v) * f.double()[:, None]
    return out


def _compare(got, clean, want, name):
    reached = ~torch.isfinite(want)
    assert reached.any(), f"{name}: nothing is reached"
    assert torch.equal(~torch.isfinite(got), reached), f"{name}: {(torch.isfinite(got) & reached).sum()} hidden, " \
                                                       f"{(~torch.isfinite(got) & ~reached).sum()} too many"
    assert torch.equal(got[~reached], clean[~reached]), name


def _places(sq, sk, d, causal):
    """(tensor, position, element, value); keys 6 and 7 of eight have another exponential in the tiled kernels than the others."""
    for value in (NAN, INF):
        for column in (3, d // 2 + 5):
            yield "q", sq // 2, column, value
            for key in {k for k in (0, 5, 6, sk // 2 // 8 * 8 + 7, sk - 1) if k < sk}:
                yield "k", key, column, value
        if not causal:  # by the definition 0 * NaN reaches every row
            yield "v", sk // 2, 9, value


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("sq,sk", [(300, 300), (40, 500), (200, 70), (1, 1)])
def test_dense(sq, sk, d, causal):
    gen = torch.Generator().manual_seed(1)
    h, hk, lam = 4, 2, torch.tensor([0.4, 0.0, -0.3, 1.0], device="cuda")
    x = {"q": _rand(gen, 2, sq, h, d), "k": _rand(gen, 2, sk, hk, d), "v": _rand(gen, 2, sk, hk, d)}
    clean = fa.flash_diff_attn_func(*x.values(), lam, causal=causal)
    for name, at, column, value in _places(sq, sk, d, causal):
        bad = {n: t.clone() for n, t in x.items()}
        bad[name][1, at, 1, column] = value
        want = torch.stack([_definition(*(t[i] for t in bad.values()), lam, causal) for i in range(2)])
        if torch.isfinite(want).all():  # a key that no query sees
            continue
        _compare(fa.flash_diff_attn_func(*bad.values(), lam, causal=causal), clean, want, f"{name} {at} {column} {value}")


def test_packed():
    gen = torch.Generator().manual_seed(2)
    lens, h, hk, d, lam = [150, 1, 300], 4, 2, 64, torch.tensor([0.4, 0.2, -0.3, 1.0], device="cuda")
    cu = torch.tensor([0] + lens).cumsum(0).int().cuda()
    x = [_rand(gen, sum(lens), n, d) for n in (h, hk, hk)]
    clean = fa.flash_diff_attn_varlen_func(*x, lam, cu, cu, 300, 300, causal=True)
    for which, at, value in ((0, 20, NAN), (0, 150, INF), (1, 149, NAN), (1, 6, INF), (1, 150, NAN), (1, 300, NAN)):
        for column in (0, 63):
            bad = [t.clone() for t in x]
            bad[which][at, 1, column] = value
            want = torch.cat([_definition(*(t[a:b] for t in bad), lam, True) for a, b in zip(cu.tolist(), cu.tolist()[1:])])
            _compare(fa.flash_diff_attn_varlen_func(*bad, lam, cu, cu, 300, 300, causal=True), clean, want, f"{which} {at} {value} {column}")


@pytest.mark.parametrize("d", [64, 128])
def test_gradients_of_rows_that_are_reached_are_not_finite(d):
    gen = torch.Generator().manual_seed(3)
    h, lam = 2, torch.tensor([0.4, 0.3], device="cuda")
    x = [_rand(gen, 1, 200, h, d) for _ in range(3)]
    for which, at in ((0, 70), (1, 6), (1, 150)):
        for column in (1, d - 1):
            leaves = [t.clone() for t in x]
            leaves[which][0, at, 1, column] = NAN
            leaves = [t.requires_grad_() for t in (*leaves, lam.clone())]
            out = fa.flash_diff_attn_func(*leaves, causal=True)
            dq, dk, dv, dlam = torch.autograd.grad(out, leaves, torch.ones_like(out))
            rows = ~torch.isfinite(out[0, :, 1]).all(-1)
            assert rows.tolist() == [(i == at if which == 0 else i >= at) for i in range(200)]
            half = slice(0, d // 2) if column < d // 2 else slice(d // 2, d)  # of the map that holds it
            assert not torch.isfinite(dq[0, rows, 1, half]).any()
            assert not torch.isfinite(dv[0, rows.nonzero()[0, 0], 1]).any()
            assert torch.isfinite(dlam[1]) == (column < d // 2)  # it is that of map 2's output
            for g in (dq, dk, dv):
                assert torch.isfinite(g[0, :, 0]).all()  # the other head
            assert torch.isfinite(dlam[0])


STEPS = [  # b, new, lengths, h, hk, d, page, num_splits: the kernels that a step may take
    (1, 1, [0], 4, 2, 64, 0, 1),
    (2, 1, [700, 63], 4, 2, 64, 0, 0),                # even shares
    (2, 1, [1999, 300], 8, 4, 128, 256, 3),           # parts, merged
    (2, 1, [300, 90], 8, 2, 128, 256, 1),             # one part
    (2, 5, [700, 90], 16, 4, 64, 256, 0),
    (2, 130, [300, 77], 4, 2, 64, 256, 1),            # a chunk of a prompt, its keys whole
    (1, 70, [4000], 4, 2, 128, 256, 0),               # ... and in parts
    (6, 130, [0, 5000, 100, 7, 900, 300], 8, 2, 64, 256, 0),  # cut by the device's decision
]


def _step(fn, x, lens, table, splits, caches, lam):
    k_cache, v_cache = (t.clone() for t in caches)
    args = (x["q"], k_cache, v_cache) + (() if lam is None else (lam,))
    return fn(*args, x["k"], x["v"], cache_seqlens=lens, block_table=table, causal=True, num_splits=splits)


@pytest.mark.parametrize("b,new,lengths,h,hk,d,page,splits", STEPS)
def test_cache_step(b, new, lengths, h, hk, d, page, splits):
    gen = torch.Generator().manual_seed(4)
    capacity = -(-(max(lengths) + new) // (page or 64)) * (page or 64)
    lam = torch.rand(h, generator=gen).cuda() + 0.1
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    table = torch.arange(b * capacity // page, dtype=torch.int32, device="cuda").view(b, -1) if page else None
    caches = [_rand(gen, b, capacity, hk, d) for _ in range(2)]
    x = {"q": _rand(gen, b, new, h, d), "k": _rand(gen, b, new, hk, d), "v": _rand(gen, b, new, hk, d)}

    def run(x, caches):
        shaped = [t.view(-1, page, hk, d) if page else t for t in caches]
        return _step(fa.flash_diff_attn_with_kvcache, x, lens, table, splits, shaped, lam)

    clean = run(x, caches)
    long = max(range(b), key=lambda i: lengths[i])
    n = lengths[long]
    places = [("q", new // 2), ("k", new - 1)] + [("cache", at) for at in ((6, n // 2, n - 1) if n else ())]
    for name, at in places:
        for column in (1, d - 2):
            for value in (NAN, INF):
                bad, dirty = {m: t.clone() for m, t in x.items()}, [t.clone() for t in caches]
                (dirty[0] if name == "cache" else bad[name])[long, at, hk - 1, column] = value
                want = torch.zeros_like(clean, dtype=torch.float64)
                for i, length in enumerate(lengths):
                    keys, values = (torch.cat((c[i, :length], bad[m][i])) for c, m in zip(dirty, ("k", "v")))
                    want[i] = _definition(bad["q"][i], keys, values, lam, True)
                _compare(run(bad, dirty), clean, want, f"{name} {at} {column} {value}")
    assert fa.device_status() == 0


@pytest.mark.parametrize("length,splits,h", [(0, 1, 4), (700, 0, 4), (1999, 3, 8), (300, 1, 8), (2500, 4, 32)])
def test_plain_cache_step_with_a_query_that_is_not_a_number(length, splits, h):
    """Every score of the query is NaN, so that no part has a maximum: the plain decode kernels and the merges are the same code."""
    gen = torch.Generator().manual_seed(5)
    x = {"q": _rand(gen, 2, 1, h, 64), "k": _rand(gen, 2, 1, 2, 64), "v": _rand(gen, 2, 1, 2, 64)}
    caches = [_rand(gen, 2, length + 64, 2, 64) for _ in range(2)]
    lens = torch.full((2,), length, dtype=torch.int32, device="cuda")
    clean = _step(fa.flash_attn_with_kvcache, x, lens, None, splits, caches, None)
    x["q"][1, 0, 1, 5] = NAN
    got = _step(fa.flash_attn_with_kvcache, x, lens, None, splits, caches, None)
    assert torch.isnan(got[1, 0, 1]).all()
    got[1, 0, 1] = clean[1, 0, 1]
    assert torch.equal(got, clean)


@pytest.mark.parametrize("b,new,lengths,h,hk,d,page,splits", STEPS)
def test_a_score_of_minus_infinity_is_a_weight_of_zero(b, new, lengths, h, hk, d, page, splits):
    """The map that sees it goes by the other keys, the other map by all: the bits are those of an element whose weight underflows."""
    gen = torch.Generator().manual_seed(6)
    capacity = -(-(max(lengths) + new) // (page or 64)) * (page or 64)
    lam = torch.rand(h, generator=gen).cuda() + 0.1
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    table = torch.arange(b * capacity // page, dtype=torch.int32, device="cuda").view(b, -1) if page else None
    caches = [_rand(gen, b, capacity, hk, d) for _ in range(2)]
    x = {"q": _rand(gen, b, new, h, d), "k": _rand(gen, b, new, hk, d), "v": _rand(gen, b, new, hk, d)}
    long = max(range(b), key=lambda i: lengths[i])
    n = lengths[long]
    for at in {0, 6, n // 2, n - 1} if n else ():
        for column in (1, d - 2):
            outs = []
            for value in (-INF, -60000.0):
                keys = caches[0].clone()
                keys[long, at, 0, column] = value
                shaped = [t.view(-1, page, hk, d) if page else t for t in (keys, caches[1])]
                outs.append(_step(fa.flash_diff_attn_with_kvcache, x, lens, table, splits, shaped, lam))
                dense = [torch.cat((c[long, :n], x[m][long]))[None] for c, m in zip((keys, caches[1]), ("k", "v"))]
                outs.append(fa.flash_diff_attn_func(x["q"][long:long + 1], *dense, lam, causal=True))
            assert torch.isfinite(outs[0]).all() and torch.isfinite(outs[1]).all()
            assert torch.equal(outs[0], outs[2]) and torch.equal(outs[1], outs[3])
