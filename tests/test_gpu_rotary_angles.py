"""rotary_positions' angles: the nearest 2^-32 of a turn."""

from __future__ import annotations

import math

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("sign", [1, -1])
def test_small_angles(device, sign) -> None:
    """(1, 0) turned by it is (cos, sin): of angles up to 64 parts of 2^-32 turns the sine is fp32's
    (relative to its size), and off by half a part and the roundings alone: 2^-52 of the angle
    before it is cut, three of fp32 after."""
    pairs = 512
    parts = torch.arange(1, pairs + 1, dtype=torch.float64) / 8 + 1 / 64
    angles = sign * parts * (2 * math.pi / 2**32)
    q = torch.cat((torch.ones(1, 1, 1, pairs), torch.zeros(1, 1, 1, pairs)), -1).to(device)
    out = Fn.rotary_positions(q, None, angles.to(device), sequence_offset=1)[0, 0, 0].cpu()
    assert (out[:pairs] == 1).all()
    part = 2 * math.pi / 2**32
    bound = part / 2 * (1 + 2.0**-20) + 4 * 2.0**-24 * angles.abs()
    assert ((out[pairs:].double() - torch.sin(angles)).abs() <= bound).all()


def test_just_below_a_whole_turn(device) -> None:
    """What rounds up to a turn is none, on both sides of it."""
    turns = torch.tensor([1 - 2.0**-34, 1 - 2.0**-40, 1 + 2.0**-34, -(2.0**-35), 3 - 2.0**-36, 1 - 2.0**-32],
                         dtype=torch.float64)
    n = len(turns)
    q = torch.cat((torch.ones(1, 1, 1, n), torch.full((1, 1, 1, n), 2.0)), -1).to(device)
    out = Fn.rotary_positions(q, None, (turns * (2 * math.pi)).to(device), sequence_offset=1)[0, 0, 0].cpu()
    assert torch.equal(out[:n - 1], torch.ones(n - 1)) and torch.equal(out[n:-1], torch.full((n - 1,), 2.0))
    # one part before a turn: (1 + 2 x, 2 - x) for the angle -x of 1.5e-9, which fp32 rounds to (1, 2)
    assert out[n - 1] == 1 and out[-1] == 2
