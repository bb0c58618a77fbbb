"""Derivatives that scored_attention does not have are refused, never left out."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import nano_megatron_amd.functional as Fn


def test_slopes_with_a_tangent() -> None:
    q, k, v = (torch.zeros(2, n, 5, 64, dtype=torch.bfloat16) for n in (4, 2, 2))
    with forward_ad.dual_level():
        slopes = forward_ad.make_dual(torch.zeros(4), torch.ones(4))
        with pytest.raises(ValueError, match="no gradient"):
            Fn.scored_attention(q, k, v, distance_slopes=slopes)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("sq", [3, 40])
def test_forward_mode(device, dtype, which, sq) -> None:
    """As ``attention``: an error, not a value whose tangent is missing."""
    args = [torch.randn(2, s, n, 64, device=device).to(dtype).transpose(1, 2) for n, s in ((4, sq), (2, 40), (2, 40))]
    with forward_ad.dual_level():
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(NotImplementedError):
            Fn.scored_attention(*args, sequence_offset=40 - sq, score_cap=20.0)
        # without a tangent in the level: a value without one
        plain = [forward_ad.unpack_dual(t).primal for t in args]
        o = Fn.scored_attention(*plain, sequence_offset=40 - sq, score_cap=20.0)
        assert forward_ad.unpack_dual(o).tangent is None and o.isfinite().all()
