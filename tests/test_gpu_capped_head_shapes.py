"""The LM head with capped logits at layouts and sizes where its kernels' strides end."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn
from tests.test_gpu_capped_head import check, make, reference, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("tokens,hidden", [(30, 64), (70_000, 64), (3, 72)])
def test_one_row_of_a_sequence(device, tokens, hidden, dtype) -> None:
    """The last token of one long sequence, and a table of one row out of a wider one: the
    stride of a dimension of size 1 says nothing."""
    x, w, t, up = make(1, hidden, 50, dtype, device, ignored=0.0)
    states = torch.zeros(1, tokens, hidden, dtype=dtype, device=device)
    states[0, -1] = x[0]
    got = run(states[:, -1], w, t, up, logit_cap=20.0, z_loss=1e-2)
    check(got, reference(x, w, t, up, 20.0, 1e-2))
    wide = torch.zeros(4, hidden + 4, dtype=dtype, device=device)
    wide[2, :hidden] = w[0]
    one = torch.zeros_like(t)
    got = run(x, wide[2:3, :hidden], one, up, logit_cap=20.0, z_loss=1e-2)
    check(got, reference(x, w[:1], one, up, 20.0, 1e-2))
