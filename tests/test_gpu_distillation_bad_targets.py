"""lm_head_distillation with unchecked targets outside the vocabulary: such a token's loss is NaN and so
is every gradient that it enters, and no other token's."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu

BAD = {3: 1 << 40, 7: 301, 8: 300, 11: -5, 30: -1}


def make(dtype, device):
    g = torch.Generator().manual_seed(5)
    x, w = (torch.randn(n, 64, generator=g).to(dtype).to(device) for n in (40, 300))
    values, ids = torch.randn(40, 6, generator=g).to(device), torch.randint(0, 300, (40, 6), generator=g)
    ids[5:9] = -1  # rows with and without a teacher's entry
    targets = torch.randint(0, 300, (40,), generator=g)
    targets[20:24] = -100
    return x, w, values, ids.to(device), targets.to(device), torch.randn(40, generator=g).to(device)


def step(x, w, values, ids, targets, up, reduction="none", **kw):
    x, w = (t.detach().requires_grad_(True) for t in (x, w))
    loss = Fn.lm_head_distillation(x, w, values, ids, targets, validate=False, reduction=reduction, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), up if reduction == "none" else None))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [1.0, 2.0])
@pytest.mark.parametrize("weight", [0.7, 0.0])
@pytest.mark.parametrize("chunk", [None, 16])
def test_bad_targets(device, dtype, temperature, weight, chunk) -> None:
    x, w, values, ids, targets, up = make(dtype, device)
    kw = dict(temperature=temperature, target_weight=weight, chunk=chunk)
    want = step(x, w, values, ids, targets, up, **kw)
    assert all(t.isfinite().all() for t in want)
    bad = targets.clone()
    for row, target in BAD.items():
        bad[row] = target
    rows = torch.zeros(40, dtype=torch.bool, device=device)
    rows[list(BAD)] = True
    for reduction in ("none", "sum", "mean"):
        loss, dx, dw = step(x, w, values, ids, bad, up, reduction, **kw)
        if reduction == "none":
            assert loss[rows].isnan().all() and torch.equal(loss[~rows], want[0][~rows])
            assert torch.equal(dx[~rows], want[1][~rows])
        else:
            assert loss.isnan() and dx[~rows].isfinite().all()
        assert dx[rows].isnan().all() and dw.isnan().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("ignore", [-5, 300, 1 << 40, 17])
def test_an_ignored_target_is_not_bad(device, dtype, ignore) -> None:
    """Wherever ignore_index lies, its tokens have no second term."""
    x, w, values, ids, targets, up = make(dtype, device)
    targets = torch.where(targets == 17, 18, targets)
    want = step(x, w, values, ids, targets, up)
    got = step(x, w, values, ids, torch.where(targets == -100, ignore, targets), up, ignore_index=ignore)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
