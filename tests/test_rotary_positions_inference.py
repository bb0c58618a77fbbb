"""RotaryPositions in inference mode first, then in training."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import RotaryPositions


@pytest.mark.parametrize("how", ["called", "moved", "built"])
def test_frequencies_are_ordinary_tensors(how) -> None:
    if how == "built":
        with torch.inference_mode():
            m = RotaryPositions(64)
    else:
        m = RotaryPositions(64)
    meta = torch.device("meta")
    with torch.inference_mode():
        if how == "moved":
            m._bring(meta)
        m.frequencies(meta)
    assert not m.frequencies(meta).is_inference()


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["called", "moved", "built"])
def test_training_after_inference(device, how) -> None:
    q = torch.randn(2, 3, 5, 64, device=device)
    if how == "built":
        with torch.inference_mode():
            m = RotaryPositions(64)
    else:
        m = RotaryPositions(64)
    with torch.inference_mode():
        if how == "moved":
            m.to(device)
        value = m(q)
    leaf = q.detach().requires_grad_(True)
    out = m(leaf)
    out.sum().backward()
    assert torch.equal(out, value)
    other = q.detach().requires_grad_(True)
    Fn.rotary_positions(other, None, Fn.rotary_frequencies(64, device=device)).sum().backward()
    assert torch.equal(leaf.grad, other.grad)
