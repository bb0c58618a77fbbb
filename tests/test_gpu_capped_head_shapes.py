"""The LM head with capped logits at layouts and sizes where its kernels' strides end."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import _lib
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


@pytest.mark.parametrize("vocab", [262_153, 262_144])
def test_table_past_2_30_elements(device, vocab) -> None:
    """Its bytes pass what 32-bit offsets reach: dx is formed by parts of the vocabulary."""
    g = torch.Generator(device=device).manual_seed(0)
    rows, hidden = 40, 4096
    x = torch.randn(rows, hidden, generator=g, device=device).bfloat16()
    w = torch.empty(vocab, hidden, dtype=torch.bfloat16, device=device)
    w.normal_(generator=g).mul_(4 / 64)
    t = torch.randint(0, vocab, (rows,), generator=g, device=device)
    t[0], t[1], t[2] = vocab - 1, 0, -100
    up = torch.randn(rows, generator=g, device=device)
    got = run(x, w, t, up, logit_cap=30.0)
    check(got, reference(x, w, t, up, 30.0, 0.0))


@pytest.mark.parametrize("rows,hidden,vocab,chunk", [
    (17_000, 8, 66_001, 17_000),     # gradients of the whole chunk would pass 2^30 elements
    (131_200, 8192, 8, None),        # the chunk's hidden states would
])
def test_chunks_past_2_30_elements(device, rows, hidden, vocab, chunk) -> None:
    """(Nearly all rows are ignored, whose gradients are zeros, so that the others are
    compared alone.)"""
    g = torch.Generator(device=device).manual_seed(0)
    x = torch.empty(rows, hidden, dtype=torch.bfloat16, device=device).normal_(generator=g)
    w = torch.randn(vocab, hidden, generator=g, device=device).mul_(4 / hidden**0.5).bfloat16()
    used = torch.cat([torch.randperm(rows, generator=g, device=device)[:120],
                      torch.tensor([0, rows - 1], device=device)]).unique()
    t = torch.full((rows,), -100, device=device)
    t[used] = torch.randint(0, vocab, (len(used),), generator=g, device=device)
    up = torch.randn(rows, generator=g, device=device)
    loss, dx, dw = run(x, w, t, up, logit_cap=30.0, chunk=chunk)
    value = reference(x[used], w, t[used], up[used], 30.0, 0.0)
    check((loss[used], dx[used], dw), value)
    rest = torch.ones(rows, dtype=torch.bool, device=device)
    rest[used] = False
    assert (dx[rest] == 0).all() and (loss[rest] == 0).all()


def test_parts_of_the_product(device) -> None:
    """dx through the library's entry alone, from gradients that end inside a part."""
    g = torch.Generator(device=device).manual_seed(1)
    for rows, hidden, vocab, ldw in ((3, 64, 300_001, 3600), (300, 128, 70_001, 16_000)):
        cols = (vocab + 7) // 8 * 8
        grad = torch.zeros(rows, cols, dtype=torch.bfloat16, device=device)
        grad[:, :vocab].normal_(generator=g)
        store = torch.empty(vocab, ldw, dtype=torch.bfloat16, device=device)
        store.fill_(float("nan"))
        w = store[:, :hidden]
        w.normal_(generator=g)
        need = _lib.ctypes.c_int64()
        _lib.call("nmb_head_loss_dx_workspace_bytes", rows, vocab, hidden, ldw, _lib.ctypes.byref(need))
        ws = torch.empty(need.value, dtype=torch.uint8, device=device)
        dx = torch.empty(rows, hidden, dtype=torch.bfloat16, device=device)
        _lib.call("nmb_head_loss_dx", grad.data_ptr(), cols, w.data_ptr(), ldw, rows, vocab, hidden, dx.data_ptr(),
                  hidden, ws.data_ptr(), need.value, _lib.stream_of(dx))
        a, b = grad[:, :vocab].double(), w.double()
        want = a @ b
        # fp32 sums, and half a step of the result
        bound = (vocab + 64) ** 0.5 * 2.0**-22 * (a.abs() @ b.abs()) + 2.0**-8 * want.abs()
        assert ((dx.double() - want).abs() <= bound).all()


@pytest.mark.parametrize("rows,hidden,vocab", [
    (65, 72, 66_001), (128, 64, 32_000), (257, 64, 16_001), (200, 136, 33_001), (1025, 64, 33_001),
])
@pytest.mark.parametrize("cap,z", [(100.0, 0.0), (60.0, 1e-2)])
def test_caps_that_need_a_maximum(device, rows, hidden, vocab, cap, z) -> None:
    """Past 80 / log2 e = 55 the exponentials' sums follow a running maximum: every tile size."""
    x, w, t, up = make(rows, hidden, vocab, torch.bfloat16, device)
    check(run(x * 4, w, t, up, logit_cap=cap, z_loss=z), reference(x * 4, w, t, up, cap, z))


def test_vocabularies_past_2_22(device) -> None:
    """What the gradient of the hidden states cannot address is refused before the loss, not
    in the backward; the loss alone, and the table's gradient, are formed."""
    g = torch.Generator(device=device).manual_seed(0)
    vocab, hidden = (1 << 22) + 3, 8
    x = torch.randn(3, hidden, generator=g, device=device).bfloat16()
    w = torch.randn(vocab, hidden, generator=g, device=device).bfloat16()
    t = torch.tensor([vocab - 1, 5, -100], device=device)
    up = torch.randn(3, generator=g, device=device)
    with pytest.raises(ValueError, match="below 2\\^22"):
        Fn.lm_head_cross_entropy(x.requires_grad_(True), w, t, logit_cap=30.0)
    with pytest.raises(ValueError, match="at most 4194240"):
        Fn.lm_head_cross_entropy(x.detach().float(), w.float().requires_grad_(True), t, logit_cap=30.0)
    x, w = x.detach(), w.requires_grad_(True)
    loss = Fn.lm_head_cross_entropy(x, w, t, reduction="none", logit_cap=30.0)
    (dw,) = torch.autograd.grad(loss, w, up)
    want = reference(x, w.detach(), t, up, 30.0, 0.0)
    for got, (value, bound) in ((loss.detach(), want[0]), (dw, want[2])):
        assert ((got.double() - value).abs() <= bound * 1.01 + 1e-37).all()
