"""lm_head_distillation: what is refused, before any device work."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from nano_megatron_amd import _lib
from nano_megatron_amd import functional as Fn

FAKE = 256  # a non-null address that is never dereferenced


@pytest.mark.parametrize("kw,message", [
    (dict(reduction="max"), "reduction"), (dict(weight=torch.ones(9, 7)), "hidden size"),
    (dict(weight=torch.ones(9, 8).bfloat16()), "one dtype"), (dict(weight=torch.ones(8)), "hidden size"),
    (dict(hidden=torch.ones(3, 8).half(), weight=torch.ones(9, 8).half()), "float16"),
    (dict(teacher_logits=torch.ones(3, 4).double()), "float32 or bfloat16"),
    (dict(teacher_ids=torch.ones(3, 4)), "int32 or int64"), (dict(teacher_ids=torch.ones(3, 4, dtype=torch.int16)), "int32"),
    (dict(teacher_ids=torch.ones(3, 5, dtype=torch.int32)), "both be"),
    (dict(teacher_logits=torch.ones(2, 4), teacher_ids=torch.ones(2, 4, dtype=torch.int32)), "both be"),
    (dict(teacher_logits=torch.ones(3), teacher_ids=torch.ones(3, dtype=torch.int32)), "both be"),
    (dict(teacher_logits=torch.ones(3, 0), teacher_ids=torch.ones(3, 0, dtype=torch.int32)), "1 to 1024"),
    (dict(teacher_logits=torch.ones(3, 1025), teacher_ids=torch.ones(3, 1025, dtype=torch.int32)), "1 to 1024"),
    (dict(targets=torch.ones(4, dtype=torch.int64)), "targets"), (dict(targets=torch.ones(3)), "targets"),
    (dict(temperature=0.0), "temperature"), (dict(temperature=101.0), "temperature"),
    (dict(temperature=math.nan), "temperature"), (dict(target_weight=-1.0), "target_weight"),
    (dict(target_weight=math.inf), "target_weight"), (dict(chunk=0), "chunk"),
    (dict(teacher_logits=torch.ones(3, 4, requires_grad=True)), "no gradient"),
    (dict(hidden=torch.ones(3, 12).bfloat16(), weight=torch.ones(9, 12).bfloat16()), "multiple of 8"),
    (dict(), "GPU only"),
])
def test_refusals(kw, message) -> None:
    args = {"hidden": torch.ones(3, 8), "weight": torch.ones(9, 8), "teacher_logits": torch.ones(3, 4),
            "teacher_ids": torch.ones(3, 4, dtype=torch.int32), **kw}
    with pytest.raises(ValueError, match=message):
        Fn.lm_head_distillation(**args)


def teacher(**kw) -> "_lib.Teacher":
    return _lib.Teacher(**{**dict(logits=FAKE, ld=4, ids=FAKE, ldi=4, targets=FAKE, ignore_index=-100, top=4,
                                  logits_dtype=_lib.NMB_F32, id_bytes=4, temperature=1.0, target_weight=1.0), **kw})


BAD_TEACHERS = [
    (dict(logits=None), "null"), (dict(ids=None), "null"), (dict(top=0), "1 to 1024"), (dict(top=1025), "1 to 1024"),
    (dict(id_bytes=2), "4 or 8"), (dict(logits_dtype=3), "fp32 or bf16"), (dict(ld=-1), "strides"),
    (dict(temperature=0.001), "temperature"), (dict(temperature=math.nan), "temperature"),
    (dict(target_weight=-1.0), "weight"), (dict(target_weight=math.inf), "weight"),
]


@pytest.mark.parametrize("change,message", BAD_TEACHERS + [
    (dict(x=None), "null"), (dict(ldx=12), "multiples of 8"), (dict(hidden=72), "leading dimension"),
    (dict(w=FAKE + 8), "aligned"), (dict(rows=-1), "shape"), (dict(vocab=0), "shape"), (dict(loss=None), "null"),
    (dict(picked=None), "null"), (dict(stats_ld=3), "null"), (dict(ws=None), "workspace"), (dict(nbytes=8), "workspace"),
    (dict(ws=FAKE + 2), "workspace"), (dict(ldx=1 << 30), "2 GiB"),
])
def test_forward_entry(change, message) -> None:
    a = dict(x=FAKE, ldx=64, w=FAKE, ldw=64, rows=4, vocab=100, hidden=64, teacher=None, loss=FAKE, stats=FAKE, stats_ld=4,
             picked=FAKE, ws=FAKE, nbytes=1 << 20)
    t = teacher(**{k: v for k, v in change.items() if k not in a})
    a.update({k: v for k, v in change.items() if k in a})
    if a["ldx"] == 12:
        a["hidden"] = 8
    a["teacher"] = ctypes.byref(t)
    with pytest.raises(ValueError, match=message):
        _lib.call("nmb_distill_fwd", *a.values(), None)


@pytest.mark.parametrize("change,message", BAD_TEACHERS + [
    (dict(stats=None), "null"), (dict(grad=None), "null"), (dict(g=None), "null"), (dict(g=FAKE + 8), "aligned"),
    (dict(ldg=100), "whole 8"), (dict(ldg=96), "whole 8"), (dict(kept=FAKE + 8), "aligned"),
])
def test_gradient_entry(change, message) -> None:
    a = dict(x=FAKE, ldx=64, w=FAKE, ldw=64, rows=4, vocab=100, hidden=64, teacher=None, stats=FAKE, stats_ld=4,
             picked=FAKE, grad=FAKE, g=FAKE, ldg=104, kept=FAKE)
    t = teacher(**{k: v for k, v in change.items() if k not in a})
    a.update({k: v for k, v in change.items() if k in a})
    a["teacher"] = ctypes.byref(t)
    with pytest.raises(ValueError, match=message):
        _lib.call("nmb_distill_grad", *a.values(), None)


@pytest.mark.parametrize("change,message", BAD_TEACHERS + [
    (dict(s=None), "null"), (dict(ld=99), "overlap"), (dict(stats_ld=3), "null"),
])
def test_row_entries(change, message) -> None:
    a = dict(s=FAKE, ld=100, rows=4, vocab=100, teacher=None)
    kept = dict(stats=FAKE, stats_ld=4, picked=FAKE)
    # "ld" is the products' here: the teacher's is changed to a negative one only
    own = {k: v for k, v in change.items() if k in a and v != -1 or k in kept}
    t = teacher(**{k: v for k, v in change.items() if k not in own})
    a.update({k: v for k, v in own.items() if k in a})
    kept.update({k: v for k, v in own.items() if k in kept})
    a["teacher"] = ctypes.byref(t)
    with pytest.raises(ValueError, match=message):
        _lib.call("nmb_distill_rows_fwd", *a.values(), FAKE, *kept.values(), FAKE, 1 << 20, None)
    with pytest.raises(ValueError, match=message):
        _lib.call("nmb_distill_rows_grad", *a.values(), *kept.values(), FAKE, FAKE, 8, 8, FAKE, None)


@pytest.mark.parametrize("x,ldx,hidden", [(None, 8, 8), (FAKE, 7, 8), (FAKE, 8, 0)])
def test_kept_needs_its_x(x, ldx, hidden) -> None:
    with pytest.raises(ValueError, match="kept"):
        _lib.call("nmb_distill_rows_grad", FAKE, 100, 4, 100, ctypes.byref(teacher()), FAKE, 4, FAKE, FAKE, x, ldx, hidden,
                  FAKE, None)


def test_no_rows_and_null() -> None:
    _lib.call("nmb_distill_fwd", None, 0, None, 0, 0, 100, 64, ctypes.byref(teacher(logits=None, ids=None)), None, None, 0,
              None, None, 0, None)
    with pytest.raises(ValueError, match="null"):
        _lib.call("nmb_distill_fwd", FAKE, 64, FAKE, 64, 4, 100, 64, None, FAKE, FAKE, 4, FAKE, FAKE, 1 << 20, None)


def test_workspace_bytes() -> None:
    nbytes = ctypes.c_int64()
    _lib.call("nmb_distill_workspace_bytes", 100, 1000, _lib.NMB_F32, ctypes.byref(nbytes))
    assert nbytes.value == 3 * 100 * 4
    _lib.call("nmb_distill_workspace_bytes", 100, 1000, _lib.NMB_BF16, ctypes.byref(nbytes))
    assert nbytes.value % (3 * 100 * 4) == 0 and nbytes.value >= 3 * 100 * 4 * (1000 // 256)
    with pytest.raises(ValueError, match="dtype"):
        _lib.call("nmb_distill_workspace_bytes", 100, 1000, 9, ctypes.byref(nbytes))


@pytest.mark.parametrize("change,message", [
    (dict(total=None), "null"), (dict(over=None), "null"), (dict(loss=None), "null"), (dict(stats=None), "null"),
    (dict(stats_ld=3), "null"), (dict(rows=-1), "bad args"), (dict(rows=1 << 30), "bad args"),
    (dict(rows=8193, stats_ld=8193, ws=None), "workspace"), (dict(rows=8193, stats_ld=8193, nbytes=4095), "workspace"),
    (dict(rows=8193, stats_ld=8193, ws=FAKE + 4), "workspace"),
])
def test_total_entry(change, message) -> None:
    a = dict(loss=FAKE, stats=FAKE, stats_ld=4, targets=FAKE, ignore=-100, rows=4, mean=1, total=FAKE, over=FAKE,
             ws=FAKE, nbytes=4096)
    a.update(change)
    with pytest.raises(ValueError, match=message):
        _lib.call("nmb_distill_total", *a.values(), None)


def test_more_rows_than_a_launch_takes() -> None:
    """A launch has fewer than 2^32 threads."""
    t = ctypes.byref(teacher())
    many = 1 << 26
    size = ctypes.c_int64()
    _lib.call("nmb_distill_workspace_bytes", many, 8, _lib.NMB_BF16, ctypes.byref(size))
    with pytest.raises(ValueError, match="too many rows"):
        _lib.call("nmb_distill_fwd", FAKE, 64, FAKE, 64, many, 8, 64, t, FAKE, FAKE, many, FAKE, FAKE, size.value, None)
    with pytest.raises(ValueError, match="too many rows"):
        _lib.call("nmb_distill_grad", FAKE, 64, FAKE, 64, many, 8, 64, t, FAKE, many, FAKE, FAKE, FAKE, 8, None, None)
    many = 1 << 22
    with pytest.raises(ValueError, match="too many rows"):
        _lib.call("nmb_distill_rows_fwd", FAKE, 8, many, 8, t, FAKE, FAKE, many, FAKE, FAKE, 1 << 40, None)
    with pytest.raises(ValueError, match="too many rows"):
        _lib.call("nmb_distill_rows_grad", FAKE, 8, many, 8, t, FAKE, many, FAKE, FAKE, None, 0, 0, None, None)


def test_rows_of_a_first_call() -> None:
    """Whole tiles of rows, fewer than all, none where one round holds every tile."""
    first = ctypes.c_int64()
    for la, lb in ((0, 0), (0, 1), (1, 1)):
        for m, n, k in ((50304, 768, 8192), (8192, 768, 50304), (3000, 2048, 32000), (50264, 1024, 709), (257, 64, 64)):
            _lib.call("nmb_gemm_bf16_first_rows", la, lb, m, n, k, ctypes.byref(first))
            assert 0 <= first.value < m and first.value % 256 == 0
            again = ctypes.c_int64(-1)
            _lib.call("nmb_gemm_bf16_first_rows", la, lb, m, n, k, ctypes.byref(again))
            assert again.value == first.value
    for m, n, k in ((0, 8, 8), (8, 0, 8), (1, 8, 8), (256, 128, 768), (512, 64, 0)):
        _lib.call("nmb_gemm_bf16_first_rows", 1, 1, m, n, k, ctypes.byref(first))
        assert first.value == 0
    for bad in ((-1, 8, 8), (8, 1 << 30, 8), (8, 8, -1)):
        with pytest.raises(ValueError, match="shape"):
            _lib.call("nmb_gemm_bf16_first_rows", 0, 0, *bad, ctypes.byref(first))
    with pytest.raises(ValueError, match="null"):
        _lib.call("nmb_gemm_bf16_first_rows", 0, 0, 8, 8, 8, None)
