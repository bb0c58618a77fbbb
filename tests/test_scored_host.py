"""What scored_attention refuses, before any device work (CPU)."""

from __future__ import annotations

import ctypes

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import HipKernelBackend, _lib

FAKE = 256  # a non-null, 16-byte aligned address that is never dereferenced


def qkv(b=2, hq=4, hkv=2, sq=5, sk=5, d=64, dtype=torch.bfloat16):
    return torch.zeros(b, hq, sq, d, dtype=dtype), *(torch.zeros(b, hkv, sk, d, dtype=dtype) for _ in range(2))


def i32(*v):
    return torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("kw,message", [
    (dict(score_cap=0.0), "score_cap"), (dict(score_cap=-1.0), "score_cap"), (dict(score_cap=float("nan")), "score_cap"),
    (dict(score_cap=float("inf")), "score_cap"), (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(window=0), "window"), (dict(window=-3), "window"),
    (dict(distance_slopes=torch.zeros(2)), "distance_slopes"),
    (dict(distance_slopes=torch.zeros(4, dtype=torch.bfloat16)), "distance_slopes"),
    (dict(distance_slopes=torch.zeros(4, requires_grad=True)), "no gradient"),
    (dict(sequence_offset=torch.zeros(2, dtype=torch.int64)), "sequence_offset"),
    (dict(sequence_offset=i32(1)), "sequence_offset"),
    (dict(prefix=i32(1, 2, 3)), "prefix"), (dict(prefix=torch.zeros(2)), "prefix"),
    (dict(prefix=i32(1, 2), causal=False), "prefix needs causal"),
    (dict(documents=torch.zeros(2, 4, dtype=torch.int32)), "key tokens"),
    (dict(documents=torch.zeros(2, 5, dtype=torch.int64)), "int32"),
    (dict(documents=torch.zeros(2, 5, dtype=torch.int32), sequence_offset=1), "lie outside"),
    (dict(documents=torch.zeros(2, 5, dtype=torch.int32), sequence_offset=-1), "lie outside"),
    (dict(), "GPU only"),
])
def test_refused_arguments(kw, message) -> None:
    with pytest.raises(ValueError, match=message):
        Fn.scored_attention(*qkv(), **kw)


def test_refused_tensors() -> None:
    q, k, v = qkv()
    for args, message in (((q[0], k, v), "must have"), ((q, k, v[:, :, :3]), "identical"), ((q[:1], k, v), "batch"),
                          ((q[:, :3], k, v), "divisible"), ((q, k.float(), v.float()), "one dtype"),
                          (qkv(d=136), "up to 128"), (qkv(dtype=torch.float16), "float16")):
        with pytest.raises(ValueError, match=message):
            Fn.scored_attention(*args)
    with pytest.raises(ValueError, match="int32"):
        Fn.document_runs(torch.zeros(5, dtype=torch.int32))


def call(fn, scores, *, sk=16, d=64, hq=4, dtype=_lib.NMB_BF16, strides=(1024, 64, 64), ws=0):
    st = _lib.i64x3(strides)
    head = [FAKE] * (6 if fn == "nmb_attn_scored_fwd" else 10)
    tail = [st] * (4 if fn == "nmb_attn_scored_fwd" else 5)
    return getattr(_lib.load(), fn)(*head, 1, hq, 4, 16, sk, d, *tail, ctypes.byref(scores) if scores else None, dtype,
                                    FAKE if ws else None, ws, None)


@pytest.mark.parametrize("fn", ["nmb_attn_scored_fwd", "nmb_attn_scored_bwd"])
def test_c_entries_refuse(fn) -> None:
    ok = _lib.Scores(0.0, 0.0, 1, 0, 0)
    lib = _lib.load()
    for status, text, kw in (
        (_lib.NMB_EINVAL, b"null", dict(scores=None)),
        (_lib.NMB_EINVAL, b"cap", dict(scores=_lib.Scores(0.0, -1.0, 1, 0, 0))),
        (_lib.NMB_EINVAL, b"cap", dict(scores=_lib.Scores(0.0, float("nan"), 1, 0, 0))),
        (_lib.NMB_EINVAL, b"window", dict(scores=_lib.Scores(0.0, 0.0, 1, -1, 0))),
        (_lib.NMB_EINVAL, b"prefix", dict(scores=_lib.Scores(0.0, 0.0, 0, 0, 0, None, None, FAKE))),
        (_lib.NMB_EINVAL, b"runs", dict(scores=_lib.Scores(0.0, 0.0, 0, 0, 0, None, None, None, FAKE + 4))),
        (_lib.NMB_EINVAL, b"divisible", dict(scores=ok, hq=6)),
        (_lib.NMB_EINVAL, b"stride", dict(scores=ok, strides=(1024, -64, 64))),
        (_lib.NMB_EUNSUPPORTED, b"head_dim", dict(scores=ok, d=136)),
        (_lib.NMB_EUNSUPPORTED, b"dtype", dict(scores=ok, dtype=5)),
    ):
        assert call(fn, **kw) == status and text in lib.nmb_last_error(), (kw, lib.nmb_last_error())
    if fn == "nmb_attn_scored_bwd":
        assert call(fn, ok) == _lib.NMB_EINVAL and b"workspace" in lib.nmb_last_error()


def test_document_runs_refuses() -> None:
    lib = _lib.load()
    assert lib.nmb_document_runs(None, 4, 1, 4, FAKE, None) == _lib.NMB_EINVAL
    assert lib.nmb_document_runs(FAKE, 4, 1, 4, FAKE + 4, None) == _lib.NMB_EINVAL
    assert lib.nmb_document_runs(FAKE, -4, 1, 4, FAKE, None) == _lib.NMB_EINVAL


@pytest.mark.parametrize("kw,message", [
    (dict(score_cap=1e-4), "score_cap"), (dict(score_cap=1e-300), "score_cap"), (dict(score_cap=2e4), "score_cap"),
    (dict(scale=1e-50), "scale"), (dict(scale=1e39), "scale"), (dict(sequence_offset=1 << 41), "sequence_offset"),
    (dict(sequence_offset=(1 << 64) + 3), "sequence_offset"),
])
def test_refuses_what_float32_or_positions_cannot_hold(kw, message) -> None:
    with pytest.raises(ValueError, match=message):
        Fn.scored_attention(*qkv(), **kw)
    for cap in (1e-4, 2e4):
        status = call("nmb_attn_scored_fwd", _lib.Scores(0.0, cap, 1, 0, 0))
        assert status == _lib.NMB_EINVAL and b"cap" in _lib.load().nmb_last_error()
    scores = _lib.Scores(0.0, 0.0, 1, 0, 0, FAKE)
    assert call("nmb_attn_scored_fwd", scores, sk=(1 << 24) + 1) == _lib.NMB_EUNSUPPORTED
    assert b"2^24 keys" in _lib.load().nmb_last_error()


@pytest.mark.parametrize("kw", [dict(score_cap=30.0), dict(window=4), dict(documents=torch.zeros(2, 5, dtype=torch.int32)),
                                dict(sequence_offset=i32(0, 0))])
def test_backend_refuses_masks_and_dropout(kw) -> None:
    backend = HipKernelBackend()
    for more in (dict(attention_mask=torch.ones(5, 5, dtype=torch.bool)), dict(dropout_p=0.1)):
        with pytest.raises(ValueError, match="cannot be combined"):
            backend.local_attention(*qkv(), **kw, **more)
    with pytest.raises(ValueError, match="GPU only"):  # scored_attention's own
        backend.local_attention(*qkv(), **kw)


def test_runs_of_other_tensors_are_refused() -> None:
    for t in (torch.zeros(2, 5, 2, dtype=torch.int64), torch.zeros(2, 5, dtype=torch.int32),
              torch.zeros(2, 5, 4, dtype=torch.int32)[..., ::2], torch.zeros(2, 5, 3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="runs must be"):
            Fn.DocumentRuns(t)
