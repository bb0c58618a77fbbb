"""What lm_head_distillation's ``validate`` looks at: present entries' ids and targets."""

from __future__ import annotations

import math

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu

VOCAB = 300


def make(device, ids_type=torch.int32, logits_type=torch.float32):
    g = torch.Generator().manual_seed(2)
    x, w = (torch.randn(n, 64, generator=g).to(device) for n in (20, VOCAB))
    values = torch.randn(20, 5, generator=g).to(device, logits_type)
    ids = torch.randint(0, VOCAB, (20, 5), generator=g).to(device, ids_type)
    return x, w, values, ids, torch.randint(0, VOCAB, (20,), generator=g).to(device)


@pytest.mark.parametrize("ids_type,past", [(torch.int32, VOCAB), (torch.int32, (1 << 31) - 1), (torch.int64, VOCAB),
                                           (torch.int64, 1 << 40)])
@pytest.mark.parametrize("logits_type", [torch.float32, torch.bfloat16])
def test_absent_entries_hold_any_id(device, ids_type, past, logits_type) -> None:
    """As the padding of a teacher's larger vocabulary: logits of minus infinity."""
    x, w, values, ids, targets = make(device, ids_type, logits_type)
    mask = torch.rand(20, 5, generator=torch.Generator().manual_seed(3)).to(device) < 0.4
    mask[:2] = True
    hidden = torch.where(mask, -math.inf, values)
    want = Fn.lm_head_distillation(x, w, hidden, torch.where(mask, -1, ids), targets)
    assert torch.equal(Fn.lm_head_distillation(x, w, hidden, torch.where(mask, past, ids), targets), want)
    # present ones do not
    for value in (0.0, torch.finfo(logits_type).min, math.nan, math.inf):
        values[3, 1], ids[3, 1] = value, past
        with pytest.raises(ValueError, match="teacher_ids"):
            Fn.lm_head_distillation(x, w, values, ids, targets)


def test_a_target_check_checks_the_targets_alone(device) -> None:
    """And the call that is given one waits for nothing else."""
    x, w, values, ids, targets = make(device)
    check = Fn.TargetCheck(targets, VOCAB)
    ids[3, 1] = VOCAB
    Fn.lm_head_distillation(x, w, values, ids, targets, reduction="none", validate=False)  # kernels are loaded
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode("error")
    try:
        loss = Fn.lm_head_distillation(x, w, values, ids, targets, reduction="none", validate=check)
    finally:
        torch.cuda.set_sync_debug_mode("default")
    assert loss[3].isnan() and loss.isnan().sum() == 1
    targets[4] = VOCAB
    with pytest.raises(ValueError, match="targets"):
        Fn.lm_head_distillation(x, w, values, ids, targets, validate=Fn.TargetCheck(targets, VOCAB))
    with pytest.raises(ValueError, match="teacher_ids"):
        Fn.lm_head_distillation(x, w, values, ids, targets)
