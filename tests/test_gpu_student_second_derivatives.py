"""Gradients of layer_norm, rotary_positions and lm_head_distillation that are differentiated again
raise, also where the gradient that came in was a constant; what has no second derivative stays."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu


def calls(device):
    g = torch.Generator().manual_seed(1)
    x, r, table = (torch.randn(n, 64, generator=g).to(device) for n in (4, 4, 50))
    w, b = torch.ones(64, device=device), torch.zeros(64, device=device)
    values, ids = torch.randn(4, 3, generator=g).to(device), torch.randint(0, 50, (4, 3), generator=g).to(device)
    targets = torch.tensor([1, 2, 3, -100], device=device)

    def head(t, tbl, reduction="none"):
        return Fn.lm_head_distillation(t, tbl, values, ids, targets, validate=False, reduction=reduction)

    return {
        "norm": (x, lambda t: Fn.layer_norm(t, w, b)),
        "norm weight": (w, lambda t: Fn.layer_norm(x, t, b)),
        "norm residual": (r, lambda t: Fn.layer_norm(x, w, b, residual=t)[0]),
        "norm and sum": (x, lambda t: sum(Fn.layer_norm(t, w, b, residual=r))),
        "head": (x, lambda t: head(t, table)),
        "head sum": (x, lambda t: head(t, table, "sum")),
        "head mean": (x, lambda t: head(t, table, "mean")),
        "head table": (table, lambda t: head(x, t, "mean")),
    }


NAMES = ["norm", "norm weight", "norm residual", "norm and sum", "head", "head sum", "head mean", "head table"]


@pytest.mark.parametrize("name", NAMES)
def test_a_constant_came_in(device, name) -> None:
    t, f = calls(device)[name]
    t = t.requires_grad_(True)
    up = torch.linspace(0.5, 1.5, f(t).numel(), device=device).view(f(t).shape)
    plain, = torch.autograd.grad(f(t), t, up)
    assert not plain.requires_grad
    first, = torch.autograd.grad(f(t), t, up, create_graph=True)
    assert torch.equal(first, plain)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        torch.autograd.grad(first.square().sum(), t)
    # a penalty on the gradient, added to the loss
    for differentiate in (lambda loss: loss.backward(), lambda loss: torch.autograd.grad(loss, t)):
        first, = torch.autograd.grad(f(t), t, up, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            differentiate(f(t).sum() + first.square().sum())


def test_through_a_model(device) -> None:
    """The parameter before the norm and the head is what the penalty is differentiated by."""
    made = calls(device)
    for name in ("norm", "norm residual", "head mean"):
        x, f = made[name]
        p = torch.ones(64, device=device, requires_grad=True)
        h = x * p
        first, = torch.autograd.grad(f(h).sum(), h, create_graph=True)
        with pytest.raises(RuntimeError, match="once_differentiable"):
            torch.autograd.grad(f(h).sum() + first.square().sum(), p)


def test_linear_ones(device) -> None:
    """A rotation's gradient and that of the sum before a norm do not depend on the inputs."""
    q = torch.randn(1, 2, 4, 64, device=device, requires_grad=True)
    f = Fn.rotary_frequencies(64, device=device)
    up = torch.randn(1, 2, 4, 64, device=device)
    first, = torch.autograd.grad(Fn.rotary_positions(q, None, f), q, up, create_graph=True)
    assert not first.requires_grad
    (q.sum() + first.square().sum()).backward()
    assert torch.equal(q.grad, torch.ones_like(q))
    # but on what comes in they do
    scale = torch.ones((), device=device, requires_grad=True)
    first, = torch.autograd.grad(Fn.rotary_positions(q, None, f), q, up * scale, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()

    x, r = (torch.randn(4, 64, device=device, requires_grad=True) for _ in range(2))
    h = Fn.layer_norm(x, torch.ones(64, device=device), residual=r)[1]
    up = torch.randint(-8, 9, (4, 64), device=device).float()  # whose sums are exact
    first, = torch.autograd.grad(h, x, up, create_graph=True)
    assert torch.equal(first, up) and not first.requires_grad
    h = Fn.layer_norm(x, torch.ones(64, device=device), residual=r)[1]
    first, = torch.autograd.grad(h, x, up * scale, create_graph=True)
    second, = torch.autograd.grad(first.sum(), scale)
    assert torch.equal(second, up.sum())
