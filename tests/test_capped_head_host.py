"""What the LM head with capped logits refuses, before any device work (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import _lib

FAKE = 256  # a non-null, 16-byte aligned address that is never dereferenced


@pytest.mark.parametrize("kw,message", [
    (dict(logit_cap=0.0), "logit_cap"), (dict(logit_cap=float("nan")), "logit_cap"),
    (dict(logit_cap=float("inf")), "logit_cap"), (dict(z_loss=-1e-4), "z_loss"), (dict(z_loss=float("nan")), "z_loss"),
    (dict(logit_cap=30.0, reduction="max"), "reduction"), (dict(logit_cap=30.0), "GPU only"),
    (dict(z_loss=1e-4), "GPU only"),
])
def test_refused_arguments(kw, message) -> None:
    with pytest.raises(ValueError, match=message):
        Fn.lm_head_cross_entropy(torch.zeros(4, 16), torch.zeros(10, 16), torch.zeros(4, dtype=torch.long), **kw)


def test_refused_tensors() -> None:
    t = torch.zeros(4, dtype=torch.long)
    for x, w, message in ((torch.zeros(4, 16), torch.zeros(10, 8), "one hidden size"),
                          (torch.zeros(4, 16).bfloat16(), torch.zeros(10, 16), "one dtype"),
                          (torch.zeros(4, 12).bfloat16(), torch.zeros(10, 12).bfloat16(), "multiple of 8"),
                          (torch.zeros(3, 16), torch.zeros(10, 16), "targets must match")):
        with pytest.raises(ValueError, match=message):
            Fn.lm_head_cross_entropy(x, w, t, logit_cap=30.0)


def test_c_entries_refuse() -> None:
    lib = _lib.load()
    need = ctypes.c_int64()
    assert lib.nmb_head_loss_workspace_bytes(300, 1000, ctypes.byref(need)) == 0 and need.value > 0
    assert lib.nmb_head_loss_workspace_bytes(-1, 1000, ctypes.byref(need)) == _lib.NMB_EINVAL

    def fwd(ldx=64, ldw=64, vocab=100, hidden=64, cap=30.0, z=0.0, x=FAKE, ws=1 << 20):
        return lib.nmb_head_loss_fwd(x, ldx, FAKE, ldw, FAKE, 4, vocab, hidden, -100, cap, z, FAKE, FAKE, FAKE, ws, None)

    def grad(ldg=104, g=FAKE, **kw):
        return lib.nmb_head_loss_grad(FAKE, 64, FAKE, 64, FAKE, 4, 100, 64, -100, 30.0, 0.0, FAKE, FAKE, g, ldg, None)

    for status, text, got in (
        (_lib.NMB_EINVAL, b"leading", lambda: fwd(ldx=32)), (_lib.NMB_EINVAL, b"cap and z", lambda: fwd(cap=-1.0)),
        (_lib.NMB_EINVAL, b"cap and z", lambda: fwd(z=float("nan"))), (_lib.NMB_EINVAL, b"null", lambda: fwd(x=None)),
        (_lib.NMB_EUNSUPPORTED, b"multiples of 8", lambda: fwd(hidden=60)),
        (_lib.NMB_EINVAL, b"aligned", lambda: fwd(x=FAKE + 8)), (_lib.NMB_EINVAL, b"workspace", lambda: fwd(ws=16)),
        (_lib.NMB_EINVAL, b"shape", lambda: fwd(vocab=0)), (_lib.NMB_EINVAL, b"whole 8", lambda: grad(ldg=100)),
        (_lib.NMB_EINVAL, b"whole 8", lambda: grad(ldg=96)), (_lib.NMB_EINVAL, b"null", lambda: grad(g=None)),
        (_lib.NMB_EINVAL, b"shape", lambda: lib.nmb_head_rows_fwd(FAKE, 99, FAKE, 4, 100, -100, 1.0, 0.0, FAKE, FAKE, None)),
        (_lib.NMB_EINVAL, b"cap and z", lambda: lib.nmb_head_rows_bwd(FAKE, 100, FAKE, 4, 100, -100, float("inf"), 0.0,
                                                                     FAKE, FAKE, None)),
    ):
        assert got() == status and text in lib.nmb_last_error(), lib.nmb_last_error()


@pytest.mark.parametrize("cap", [1e-4, 1e-300, 2e4])
def test_refuses_caps_that_float32_cannot_hold(cap) -> None:
    with pytest.raises(ValueError, match="logit_cap"):
        Fn.lm_head_cross_entropy(torch.zeros(4, 16), torch.zeros(10, 16), torch.zeros(4, dtype=torch.long), logit_cap=cap)
    if cap < 1e-100:
        return  # 0 to the library: no cap
    lib = _lib.load()
    got = lib.nmb_head_rows_fwd(FAKE, 100, FAKE, 4, 100, -100, cap, 0.0, FAKE, FAKE, None)
    assert got == _lib.NMB_EINVAL and b"cap and z" in lib.nmb_last_error()


def test_dx_refuses() -> None:
    lib = _lib.load()

    def dx(g=FAKE, ldg=104, w=FAKE, ldw=64, vocab=97, hidden=64, out=FAKE, ldo=64, rows=4):
        return lib.nmb_head_loss_dx(g, ldg, w, ldw, rows, vocab, hidden, out, ldo, None, 0, None)

    for status, got in (
        (_lib.NMB_EINVAL, lambda: dx(g=None)), (_lib.NMB_EINVAL, lambda: dx(vocab=0)),
        (_lib.NMB_EINVAL, lambda: dx(ldg=96)), (_lib.NMB_EUNSUPPORTED, lambda: dx(ldg=100)),
        (_lib.NMB_EUNSUPPORTED, lambda: dx(hidden=60)), (_lib.NMB_EINVAL, lambda: dx(out=FAKE + 8)),
        (_lib.NMB_EINVAL, lambda: dx(ldo=56)), (_lib.NMB_EINVAL, lambda: dx(rows=4096, vocab=50257, ldg=50264)),
    ):
        assert got() == status, lib.nmb_last_error()
    assert dx(rows=0) == _lib.NMB_OK


def test_one_device() -> None:
    x, w, t = torch.zeros(4, 16), torch.zeros(10, 16), torch.zeros(4, dtype=torch.long)
    with pytest.raises(ValueError, match="one device"):
        Fn.lm_head_cross_entropy(x, w, t.to("meta"), logit_cap=30.0)
    with pytest.raises(ValueError, match="one device"):
        Fn.embedding(w, t.to("meta"), scale=2.0)
