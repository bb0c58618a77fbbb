"""Several heads that share one TiedGrad: the table's gradient is that of all of them."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu


def heads(device):
    g = torch.Generator().manual_seed(6)
    values, ids = torch.randn(40, 4, generator=g).to(device), torch.randint(0, 300, (40, 4), generator=g).to(device)
    targets = torch.randint(0, 300, (40,), generator=g).to(device)
    return {
        "teacher": lambda h, w, tie: Fn.lm_head_distillation(h, w, values, ids, targets, tie=tie),
        "capped": lambda h, w, tie: Fn.lm_head_cross_entropy(h, w, targets, logit_cap=30.0, z_loss=1e-3, tie=tie),
        "plain": lambda h, w, tie: Fn.lm_head_cross_entropy(h, w, targets, tie=tie),
    }


def table_of(device, dtype):
    g = torch.Generator().manual_seed(7)
    return torch.randn(300, 64, generator=g).to(dtype).to(device), torch.randint(0, 300, (40,), generator=g).to(device)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("names", [("teacher", "teacher"), ("teacher", "plain"), ("capped", "teacher"), ("plain", "capped"),
                                   ("teacher", "capped", "plain")])
def test_heads_add_up(device, dtype, names) -> None:
    made = heads(device)
    table, tokens = table_of(device, dtype)

    def gradient(tied, names):
        w = table.detach().requires_grad_(True)
        tie = Fn.TiedGrad() if tied else None
        h = Fn.embedding(w, tokens, tie)
        loss = sum(made[name](h, w, tie) for name in names)
        grad, = torch.autograd.grad(loss, w)
        assert tie is None or tie.grad is None
        return grad

    got, want = gradient(True, names), gradient(False, names)
    # the same parts, rounded one by one and as sums, at most one more of each a head
    half = torch.finfo(dtype).eps / 2
    size = sum(gradient(False, (name,)).double().abs() for name in names)
    # (and of the embedding's part, which is in each of them, both ways)
    assert ((got.double() - want.double()).abs() <= 4 * len(names) * half * (size + want.double().abs())).all()
    for name in names:  # far from losing any
        assert (got - gradient(False, (name,))).double().norm() > 0.1 * gradient(False, (name,)).double().norm()


@pytest.mark.parametrize("name", ["teacher", "capped", "plain"])
def test_what_never_came_to_the_embedding_is_dropped(device, name) -> None:
    head = heads(device)[name]
    table, tokens = table_of(device, torch.float32)
    w = table.detach().requires_grad_(True)
    tie = Fn.TiedGrad()
    h = Fn.embedding(w, tokens, tie)
    loss = head(h, w, tie)
    torch.autograd.grad(loss, h, retain_graph=True)
    got, = torch.autograd.grad(loss, w, retain_graph=True)
    again, = torch.autograd.grad(loss, w)
    fresh = Fn.TiedGrad()
    want, = torch.autograd.grad(head(Fn.embedding(w, tokens, fresh), w, fresh), w)
    assert torch.equal(got, want) and torch.equal(again, want)
