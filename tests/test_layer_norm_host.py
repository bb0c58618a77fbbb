"""layer_norm: what is refused, before any device work."""

from __future__ import annotations

import ctypes

import pytest
import torch

from nano_megatron_amd import LayerNorm, _lib
from nano_megatron_amd import functional as Fn

FAKE = 256  # a non-null address that is never dereferenced


@pytest.mark.parametrize("kw,message", [
    (dict(weight=torch.ones(7)), "last dimension"),
    (dict(weight=torch.ones(1, 8)), "last dimension"),
    (dict(x=torch.ones(3, 0), weight=torch.ones(0)), "last dimension"),
    (dict(x=torch.tensor(1.0), weight=torch.ones(1)), "last dimension"),
    (dict(bias=torch.ones(9)), "does not match the weight"),
    (dict(residual=torch.ones(1, 8)), "does not match x"),
    (dict(residual=torch.ones(3, 8).bfloat16()), "one dtype"),
    (dict(weight=torch.ones(8).bfloat16()), "one dtype"),
    (dict(eps=0.0), "eps"),
    (dict(eps=float("nan")), "eps"),
    (dict(eps=float("inf")), "eps"),
    (dict(x=torch.ones(3, 8).half(), weight=torch.ones(8).half()), "float16"),
    (dict(), "GPU only"),
])
def test_refusals(kw, message) -> None:
    args = {"x": torch.ones(3, 8), "weight": torch.ones(8), **kw}
    with pytest.raises(ValueError, match=message):
        Fn.layer_norm(**args)


def test_module_checks() -> None:
    with pytest.raises(ValueError, match="positive"):
        LayerNorm(0)
    with pytest.raises(ValueError, match="positive"):
        LayerNorm(8, eps=0.0)
    with pytest.raises(ValueError, match="last dimension"):
        LayerNorm(8)(torch.ones(3, 9))
    assert LayerNorm(8, bias=False).bias is None


@pytest.mark.parametrize("change,message", [
    (dict(cols=0), "invalid shape"), (dict(rows=-1), "invalid shape"), (dict(rows=1 << 31), "invalid shape"),
    (dict(cols=16385), "maximum"), (dict(x=None), "null"), (dict(w=None), "null"), (dict(ldx=-8), "stride"),
    (dict(res=FAKE, h=None), "missing"), (dict(res=None, h=FAKE), "missing"), (dict(y=None), "missing"),
    (dict(eps=0.0), "eps"), (dict(dtype=7), "dtype"),
])
def test_forward_entry(change, message) -> None:
    a = {**dict(x=FAKE, ldx=8, res=FAKE, ldr=8, w=FAKE, b=FAKE, y=FAKE, h=FAKE, stats=FAKE, rows=4, cols=8, eps=1e-5,
                dtype=_lib.NMB_F32), **change}
    with pytest.raises(ValueError, match=message):
        _lib.call("nmb_layernorm_fwd", *a.values(), None)


@pytest.mark.parametrize("change,message", [
    (dict(ws=None), "workspace"), (dict(nbytes=0), "workspace"), (dict(ws=FAKE + 2), "workspace"),
    (dict(stats=None), "null"), (dict(dy=None), "null"), (dict(dx=None), "null"), (dict(lddy=-1), "stride"),
    (dict(cols=1 << 20), "maximum"),
])
def test_backward_entry(change, message) -> None:
    a = {**dict(h=FAKE, ldh=8, stats=FAKE, w=FAKE, dy=FAKE, lddy=8, dh=FAKE, lddh=8, dx=FAKE, dw=FAKE, db=FAKE, ws=FAKE,
                nbytes=1 << 20, rows=4, cols=8, dtype=_lib.NMB_BF16), **change}
    with pytest.raises(ValueError, match=message):
        _lib.call("nmb_layernorm_bwd", *a.values(), None)


def test_workspace_holds_two_sums_a_workgroup() -> None:
    nbytes = ctypes.c_size_t()
    for rows, cols in ((0, 5), (1, 1), (100_000, 768), (1 << 30, 16384)):
        _lib.call("nmb_layernorm_bwd_workspace_bytes", rows, cols, _lib.NMB_BF16, ctypes.byref(nbytes))
        assert nbytes.value % (8 * cols) == 0 and 1 <= nbytes.value // (8 * cols) <= 512


def test_more_rows_than_a_launch_takes() -> None:
    """A launch has fewer than 2^32 threads, eight to a row of eight elements."""
    with pytest.raises(ValueError, match="too many"):
        _lib.call("nmb_layernorm_fwd", FAKE, 8, None, 0, FAKE, None, FAKE, None, None, 1 << 29, 8, 1e-5, _lib.NMB_F32, None)
