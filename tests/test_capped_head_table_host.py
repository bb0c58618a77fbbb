"""The workspace of dx = G W of the capped head, and tables it refuses (CPU)."""

from __future__ import annotations

import ctypes

from nano_megatron_amd import _lib

FAKE = 256  # a non-null, 16-byte aligned address that is never dereferenced


def test_workspace_and_refusals() -> None:
    lib = _lib.load()
    need, plain = ctypes.c_int64(), ctypes.c_int64()
    for rows, vocab, hidden in ((8192, 50304, 768), (709, 50257, 1024), (1, 8, 8), (64, 262136, 4096)):
        assert lib.nmb_head_loss_dx_workspace_bytes(rows, vocab, hidden, hidden, ctypes.byref(need)) == _lib.NMB_OK
        assert lib.nmb_gemm_bf16_workspace_bytes(0, 1, rows, hidden, vocab, ctypes.byref(plain)) == _lib.NMB_OK
        assert need.value == plain.value
    # parts of a larger table are added up from fp32 partials, a whole number of them
    assert lib.nmb_head_loss_dx_workspace_bytes(2096, 256128, 4608, 4608, ctypes.byref(need)) == _lib.NMB_OK
    assert need.value >= 2 * 2096 * 4608 * 4 and need.value % (2096 * 4608 * 4) == 0
    assert lib.nmb_head_loss_dx_workspace_bytes(4, 100, 64, 64, None) == _lib.NMB_EINVAL
    assert lib.nmb_head_loss_dx_workspace_bytes(4, 100, 64, 56, ctypes.byref(need)) == _lib.NMB_EINVAL
    assert lib.nmb_head_loss_dx_workspace_bytes(4, 100, 64, 1 << 22, ctypes.byref(need)) == _lib.NMB_EUNSUPPORTED
    assert lib.nmb_head_loss_dx(FAKE, 256128, FAKE, 4608, 8, 256128, 4608, FAKE, 4608, None, 0, None) == _lib.NMB_EINVAL
    assert b"workspace" in lib.nmb_last_error()
