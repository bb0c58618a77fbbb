"""embedding(scale=) against 64 bits, both directions, and beside the unscaled one."""

from __future__ import annotations

import math

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu


def make(tokens, hidden, vocab, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randn(vocab, hidden, generator=g).to(dtype).to(device)
    ids = (torch.rand(tokens, generator=g) ** 3 * vocab).long().clamp_max(vocab - 1)  # few ids many times
    return w, ids.to(device), torch.randn(tokens, hidden, generator=g).to(dtype).to(device)


def run(w, ids, grad, scale, tie=None):
    w = w.detach().requires_grad_(True)
    out = Fn.embedding(w, ids, tie, scale=scale)
    return out.detach(), *torch.autograd.grad(out, w, grad)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,hidden,vocab", [
    (1, 8, 1), (2, 64, 5), (64, 256, 1000), (65, 264, 50257), (700, 72, 33), (8193, 768, 8192), (3000, 1024, 3),
])
@pytest.mark.parametrize("scale", [math.sqrt(768), 0.125, -3.0, 0.0])
def test_scaled_embedding(device, tokens, hidden, vocab, scale, dtype) -> None:
    """One rounding (u) of each row; the gradient's fp32 sum of n rows is off by n 2^-24
    of the sum of their magnitudes, its product with the scale (itself rounded to fp32)
    by 2^-23, and it is rounded once (u)."""
    w, ids, grad = make(tokens, hidden, vocab, dtype, device)
    out, dw = run(w, ids, grad, scale)
    u = torch.finfo(dtype).eps / 2
    want = w.double()[ids] * scale
    assert ((out.double() - want).abs() <= (u + 2.0**-23) * want.abs()).all()
    sums = torch.zeros(vocab, hidden, dtype=torch.float64, device=device).index_add_(0, ids, grad.double())
    mags = torch.zeros_like(sums).index_add_(0, ids, grad.double().abs())
    n = torch.bincount(ids, minlength=vocab)[:, None]
    assert ((dw.double() - sums * scale).abs() <= abs(scale) * (n * 2.0**-24 * mags + (u + 2.0**-22) * sums.abs())).all()
    assert all(torch.equal(a, b) for a, b in zip((out, dw), run(w, ids, grad, scale)))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_scale_one_and_powers_of_two(device, dtype) -> None:
    """A scale of 1 is the unscaled lookup, one of 4 exactly four times it."""
    w, ids, grad = make(500, 128, 300, dtype, device)
    plain = run(w, ids, grad, None)
    assert all(torch.equal(a, b) for a, b in zip(plain, run(w, ids, grad, 1.0)))
    assert all(torch.equal(4 * a, b) for a, b in zip(plain, run(w, ids, grad, 4.0)))


def test_ids_outside_views_and_shapes(device) -> None:
    w, ids, grad = make(60, 64, 40, torch.bfloat16, device)
    ids = ids.clone()
    ids[::7] = torch.tensor([-1, 40, 1 << 40], device=device).repeat(3)
    out, dw = run(w, ids, grad, 2.0)
    inside = (ids >= 0) & (ids < 40)
    assert (out[~inside] == 0).all() and torch.equal(out[inside], 2 * w[ids[inside]])
    kept = run(w, ids[inside], grad[inside], 2.0)[1]
    assert torch.equal(dw, kept)
    # a table that is a view (of a wider one, of a misaligned start), ids of another type and shape
    wide = torch.randn(40, 100, device=device).bfloat16()
    flat = torch.randn(40 * 64 + 1, device=device).bfloat16()
    for t in (wide[:, 3:67], flat[1:].view(40, 64)):
        a = run(t, ids.clamp(0, 39).int().view(6, 10), grad.view(6, 10, 64), 3.0)
        b = run(t.clone(memory_format=torch.contiguous_format), ids.clamp(0, 39), grad, 3.0)
        assert a[0].shape == (6, 10, 64) and torch.equal(a[0].view(60, 64), b[0]) and torch.equal(a[1], b[1])
    assert run(w, ids[:0], grad[:0], 2.0)[1].abs().sum() == 0


def test_tied_gradient_is_not_scaled(device) -> None:
    w, ids, grad = make(90, 64, 50, torch.float32, device)
    head = torch.randn_like(w)
    tie = Fn.TiedGrad()
    w2 = w.detach().requires_grad_(True)
    out = Fn.embedding(w2, ids, tie, scale=5.0)
    tie.grad = head
    (dw,) = torch.autograd.grad(out, w2, grad)
    assert torch.equal(dw, head + run(w, ids, grad, 5.0)[1])


def test_refusals(device) -> None:
    w, ids, _ = make(4, 64, 8, torch.bfloat16, device)
    for scale in (float("nan"), float("inf"), 1e39):
        with pytest.raises(ValueError, match="scale"):
            Fn.embedding(w, ids, scale=scale)
    with pytest.raises(TypeError, match="integer"):
        Fn.embedding(w, ids.float(), scale=2.0)
    with pytest.raises(ValueError, match="GPU only"):
        Fn.embedding(w.cpu(), ids.cpu(), scale=2.0)
