"""Derivatives that layer_norm, rotary_positions and lm_head_distillation do not have are
refused, never dropped: forward mode, function transforms, and a batch of calls at once."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu


def calls(device):
    x = torch.randn(4, 64, device=device)
    w, b = torch.ones(64, device=device), torch.zeros(64, device=device)
    q = torch.randn(1, 2, 4, 64, device=device)
    f = Fn.rotary_frequencies(64, device=device)
    table = torch.randn(50, 64, device=device)
    values, ids = torch.randn(4, 3, device=device), torch.zeros(4, 3, dtype=torch.int32, device=device)
    return {
        "norm": (x, lambda t: Fn.layer_norm(t, w, b)),
        "norm weight": (w, lambda t: Fn.layer_norm(x, t, b)),
        "norm bias": (b, lambda t: Fn.layer_norm(x, w, t)),
        "norm residual": (x, lambda t: Fn.layer_norm(x, w, b, residual=t)[0]),
        "rotary": (q, lambda t: Fn.rotary_positions(t, None, f)),
        "rotary key": (q, lambda t: Fn.rotary_positions(q, t, f)[1]),
        "head": (x, lambda t: Fn.lm_head_distillation(t, table, values, ids, validate=False)),
        "head table": (table, lambda t: Fn.lm_head_distillation(x, t, values, ids, validate=False)),
    }


NAMES = ["norm", "norm weight", "norm bias", "norm residual", "rotary", "rotary key", "head", "head table"]


@pytest.mark.parametrize("name", NAMES)
def test_forward_mode(device, name) -> None:
    t, f = calls(device)[name]
    for grads in (True, False):
        with torch.set_grad_enabled(grads), forward_ad.dual_level():
            with pytest.raises(RuntimeError):
                f(forward_ad.make_dual(t, torch.ones_like(t)))


@pytest.mark.parametrize("name", NAMES)
def test_transforms(device, name) -> None:
    t, f = calls(device)[name]
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda a: f(a).sum())(t)
    with pytest.raises(RuntimeError):
        torch.func.vmap(f)(torch.stack((t, t)))


@pytest.mark.parametrize("kw", [dict(values=True), dict(frequencies=True)])
def test_what_gets_no_gradient(device, kw) -> None:
    """Tangents and gradients of a teacher's logits and of frequencies."""
    x, table = torch.randn(4, 64, device=device), torch.randn(50, 64, device=device)
    values, ids = torch.randn(4, 3, device=device), torch.zeros(4, 3, dtype=torch.int32, device=device)
    f = Fn.rotary_frequencies(64, device=device)
    q = torch.randn(1, 2, 4, 64, device=device)
    if "values" in kw:
        call, t = (lambda v: Fn.lm_head_distillation(x, table, v, ids)), values
    else:
        call, t = (lambda v: Fn.rotary_positions(q, None, v)), f
    with pytest.raises(ValueError, match="no gradient"):
        call(t.clone().requires_grad_(True))
    with torch.no_grad():
        call(t.clone().requires_grad_(True))
    with forward_ad.dual_level(), pytest.raises(ValueError, match="no gradient"):
        call(forward_ad.make_dual(t, torch.ones_like(t)))
