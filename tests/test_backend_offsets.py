"""The query offset of the backend's attention: one number, also held by a tensor, or one
per sequence."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import HipKernelBackend


@pytest.mark.parametrize("offset", [torch.tensor(3), torch.tensor(3, dtype=torch.int32), torch.tensor([3])])
@pytest.mark.parametrize("more", [{}, {"dropout_p": 0.1}, {"score_cap": 20.0}])
def test_one_number(monkeypatch, offset, more) -> None:
    seen = []
    for name in ("attention", "masked_attention", "scored_attention"):
        monkeypatch.setattr(Fn, name, lambda *a, sequence_offset, **kw: seen.append(sequence_offset))
    HipKernelBackend().local_attention(*(torch.zeros(2, 2, 5, 64) for _ in range(3)), sequence_offset=offset, **more)
    assert seen == [3] and isinstance(seen[0], int)


def test_one_sequence(monkeypatch) -> None:
    """Of a batch of one: still the number where a mask or dropout takes only that."""
    seen = []
    monkeypatch.setattr(Fn, "masked_attention", lambda *a, sequence_offset, **kw: seen.append(sequence_offset))
    monkeypatch.setattr(Fn, "scored_attention", lambda *a, sequence_offset, **kw: seen.append(sequence_offset))
    offset = torch.tensor([3], dtype=torch.int32)
    args = [torch.zeros(1, 2, 5, 64) for _ in range(3)]
    HipKernelBackend().local_attention(*args, sequence_offset=offset, dropout_p=0.1)
    HipKernelBackend().local_attention(*args, sequence_offset=offset, attention_mask=torch.ones(5, 5).bool())
    HipKernelBackend().local_attention(*args, sequence_offset=offset)
    assert seen[:2] == [3, 3] and seen[2] is offset


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_result(device, dtype) -> None:
    q, k, v = (torch.randn(2, s, 2, 64, device=device).to(dtype).transpose(1, 2) for s in (5, 30, 30))
    backend = HipKernelBackend()
    want = backend.local_attention(q, k, v, sequence_offset=25)
    assert torch.equal(backend.local_attention(q, k, v, sequence_offset=torch.tensor(25, device=device)), want)
