"""Inputs and gradients of outputs in layouts that tensor maps do not take: expanded, sliced, not aligned to 16 bytes."""
import pytest
import torch

import flash_attention_turing_b200 as fa
from flash_attention_turing_b200 import diff_attention_interface, flash_attention_interface

pytestmark = pytest.mark.gpu


def _layouts(shape, gen):
    """Gradients of `shape` (rows.., heads, d)."""
    rand = lambda *s: torch.randn(*s, generator=gen).half().cuda()  # noqa: E731
    *rows, h, d = shape
    yield "sum over rows", rand(1, h, d).expand(*rows, h, d) if len(rows) == 1 else rand(rows[0], 1, h, d).expand(shape)
    yield "sum over everything in front", rand(*[1] * len(rows), h, d).expand(shape)
    yield "one for all heads", rand(*rows, 1, d).expand(shape)
    yield "sum over all", rand(1).expand(shape)
    yield "slice of wider heads", rand(*rows, h, d + 3)[..., 3:]
    yield "slice at an odd element", rand(*rows, h * d + 1)[..., 1:].unflatten(-1, (h, d))
    yield "transposed", rand(*rows, d, h).transpose(-1, -2)
    yield "whole", rand(*shape)


@pytest.mark.parametrize("differential", [True, False])
@pytest.mark.parametrize("packed", [True, False])
@pytest.mark.parametrize("by_class", [True, False])
def test_gradient_layouts(differential, packed, by_class):
    gen = torch.Generator().manual_seed(1)
    shape = (90, 4, 64) if packed else (2, 45, 4, 64)
    leaves = [torch.randn(*shape[:-2], n, 64, generator=gen).half().cuda().requires_grad_() for n in (4, 2, 2)]
    if differential:
        leaves.append(torch.rand(4, generator=gen).cuda().requires_grad_())
    cu = torch.tensor([0, 50, 90], dtype=torch.int32, device="cuda")
    more = (cu, cu, 50, 50) if packed else ()
    module = diff_attention_interface if differential else flash_attention_interface
    if by_class:  # what the native node leaves to it
        name = "Flash" + ("Diff" if differential else "") + "Attn" + ("Varlen" if packed else "") + "Func"
        out = getattr(module, name).apply(*leaves, *more, None, True, True)
    else:
        name = "flash_" + ("diff_" if differential else "") + "attn_" + ("varlen_" if packed else "") + "func"
        out = getattr(fa, name)(*leaves, *more, causal=True)
    out = out[0] if isinstance(out, tuple) else out
    for name, dout in _layouts(shape, gen):
        want = torch.autograd.grad(out, leaves, dout.clone(memory_format=torch.contiguous_format), retain_graph=True)
        got = torch.autograd.grad(out, leaves, dout, retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), name
    pooled = out.sum(0 if packed else 1)
    assert torch.isfinite(torch.autograd.grad((pooled * torch.arange(4, device="cuda")[:, None]).sum(), leaves)[0]).all()


@pytest.mark.parametrize("differential", [True, False])
@pytest.mark.parametrize("packed", [True, False])
def test_input_layouts(differential, packed):
    """Keys and values that are broadcast over heads or batch, slices at odd places: output and gradients as of copies."""
    gen = torch.Generator().manual_seed(2)
    rand = lambda *s: torch.randn(*s, generator=gen).half().cuda()  # noqa: E731
    rows, cu = ((90,) if packed else (2, 45)), torch.tensor([0, 50, 90], dtype=torch.int32, device="cuda")
    more = (cu, cu, 50, 50) if packed else ()
    lam = (torch.rand(4, generator=gen).cuda(),) if differential else ()
    fn = getattr(fa, "flash_" + ("diff_" if differential else "") + "attn_" + ("varlen_" if packed else "") + "func")
    dout = rand(*rows, 4, 64)
    for name, base, view in (
        ("one key head", (rand(*rows, 4, 64), rand(*rows, 1, 64), rand(*rows, 1, 64)), lambda q, k, v: (q, k.expand(*rows, 4, 64), v.expand(*rows, 4, 64))),
        ("one for all rows", (rand(*[1] * len(rows), 4, 64), rand(*rows, 2, 64), rand(*rows, 2, 64)), lambda q, k, v: (q.expand(*rows, 4, 64), k, v)),
        ("odd slices", [rand(*rows, n, 67) for n in (4, 2, 2)], lambda *x: [t[..., 3:] for t in x]),
        ("odd rows", [rand(*rows, n * 64 + 1) for n in (4, 2, 2)], lambda *x: [t[..., 1:].unflatten(-1, (-1, 64)) for t in x]),
    ):
        results = []
        for copied in (False, True):
            leaves = [t.clone().requires_grad_() for t in base]
            out = fn(*((t.contiguous() if copied else t) for t in view(*leaves)), *lam, *more, causal=True)
            results.append([out, *torch.autograd.grad(out, leaves, dout)])
        assert all(torch.equal(a, b) for a, b in zip(*results)), name


@pytest.mark.parametrize("differential", [True, False])
def test_one_row_with_an_odd_stride(differential):
    """The stride of a dimension of one element, which no address depends on."""
    gen = torch.Generator().manual_seed(3)
    leaves = [torch.randn(1, 1, n, 64, generator=gen).half().cuda().requires_grad_() for n in (4, 2, 2)]
    if differential:
        leaves.append(torch.rand(4, generator=gen).cuda().requires_grad_())
    dout = torch.randn(257, generator=gen).half().cuda().as_strided((1, 1, 4, 64), (257, 257, 64, 1))
    assert dout.stride() == (257, 257, 64, 1) and dout.is_contiguous()
    for cls in (None, diff_attention_interface.FlashDiffAttnFunc if differential else flash_attention_interface.FlashAttnFunc):
        fn = fa.flash_diff_attn_func if differential else fa.flash_attn_func
        out = cls.apply(*leaves, None, False, True) if cls else fn(*leaves)
        out = out[0] if isinstance(out, tuple) else out
        want = torch.autograd.grad(out, leaves, dout.clone(memory_format=torch.contiguous_format), retain_graph=True)
        assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(out, leaves, dout), want))
