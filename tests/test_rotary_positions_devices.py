"""RotaryPositions built under a default device: its frequencies are there, in 64 bits, wherever it goes."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import RotaryPositions

CPU = torch.device("cpu")


def test_built_on_meta() -> None:
    want = Fn.rotary_frequencies(32, scaling="parts", factor=8.0, original_length=4096)
    with torch.device("meta"):
        m = RotaryPositions(64, rotary_dim=32, scaling="parts", factor=8.0, original_length=4096)
        assert torch.equal(m.frequencies(CPU), want)
        m.to(CPU)
    m.to_empty(device="cpu")
    assert torch.equal(m.frequencies(CPU), want) and m.frequencies(CPU).dtype == torch.float64


def test_frequencies_follow_the_default_device() -> None:
    with torch.device("meta"):
        assert Fn.rotary_frequencies(32).is_meta
        assert torch.equal(Fn.rotary_frequencies(32, device="cpu"), Fn.rotary_frequencies(32, device=CPU))
    assert Fn.rotary_frequencies(32).device == CPU


def built(how, device):
    if how == "meta":
        with torch.device("meta"):
            return RotaryPositions(64).to_empty(device=device)
    if how == "default":
        torch.set_default_device("cuda")
        try:
            return RotaryPositions(64)
        finally:
            torch.set_default_device(None)
    with torch.device(how):
        return RotaryPositions(64)


@pytest.mark.gpu
@pytest.mark.parametrize("how", ["meta", "default", "cuda", "cuda:0"])
def test_first_call_captured(device, how) -> None:
    q = torch.randn(2, 3, 5, 64, device=device)
    want = Fn.rotary_positions(q, None, Fn.rotary_frequencies(64, device=device))
    m = built(how, device)
    assert set(m._frequencies) == {CPU, device}
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = m(q)
    for _ in range(3):
        graph.replay()
        assert torch.equal(m(q), want)
        torch.cuda.synchronize()
        assert torch.equal(got, want)
