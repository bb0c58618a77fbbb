"""lm_head_cross_entropy with capped logits and the log-normaliser's penalty
against 64 bits, both directions."""

from __future__ import annotations

import math

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu


def make(rows, hidden, vocab, dtype, device, seed=0, ignored=0.2):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hidden, generator=g).to(dtype).to(device)
    w = (torch.randn(vocab, hidden, generator=g) * 4 / math.sqrt(hidden)).to(dtype).to(device)
    t = torch.randint(0, vocab, (rows,), generator=g)
    t[torch.rand(rows, generator=g) < ignored] = -100
    up = torch.randn(rows, generator=g).to(device)
    return x, w, t.to(device), up


def reference(x, w, t, up, cap, z):
    """(loss, dx, dw) in 64 bits with a bound for each: a logit is off by e =
    (hidden + 8) 2^-24 sum |x w| (times the cap's slope) and by 2^-20 cap; the loss by
    2 max e, z's term by 2 z lse that, and by 2^-21 of its parts; the gradient G by the
    factor exp(2 e) of its exponentials and, in bf16, by half a step (u) before the next
    product, whose fp32 sums add (n + 8) 2^-24 of their terms; results by u."""
    f = torch.float64
    u = torch.finfo(x.dtype).eps / 2
    bf16 = x.dtype == torch.bfloat16
    xd, wd = x.to(f), w.to(f)
    s = xd @ wd.t()
    e = (x.shape[1] + 8) * 2.0**-24 * (xd.abs() @ wd.abs().t())
    bent = torch.ones_like(s)
    y = s
    if cap:
        th = torch.tanh(s / cap)
        y, bent = cap * th, 1 - th * th
        e = e * bent + 2.0**-20 * cap
    lse = torch.logsumexp(y, 1)
    used = t != -100
    at = t.clamp_min(0)
    picked = y.gather(1, at[:, None])[:, 0]
    loss = torch.where(used, lse - picked + z * lse**2, 0.0)
    row = e.amax(1)
    loss_bound = used * (2 * row * (1 + z * lse.abs()) + 2.0**-21 * (lse.abs() + picked.abs() + 16 + z * lse**2))
    p = torch.exp(y - lse[:, None])
    hot = torch.zeros_like(p).scatter_(1, at[:, None], 1.0)
    upd = torch.where(used, up.to(f), 0.0)[:, None]
    fac = (1 + 2 * z * lse)[:, None]
    g = (p * fac - hot) * bent * upd
    off = (2 * row[:, None] + (w.shape[0] + 64) ** 0.5 * 2.0**-23 + 2.0**-20)
    off_bent = (2.0**-20 + 2 * e / cap) if cap else 0.0
    g_bound = u * bf16 * g.abs() + off * (p * fac.abs()) * bent * upd.abs() + (p * fac.abs() + hot) * upd.abs() * off_bent \
        + 2.0**-22 * (p * fac.abs() + hot) * bent * upd.abs()
    n = lambda k: (k + 8) * 2.0**-24  # noqa: E731
    dx, dw = g @ wd, g.t() @ xd
    dx_bound = (g_bound + n(w.shape[0]) * g.abs()) @ wd.abs() + u * dx.abs()
    dw_bound = (g_bound + n(x.shape[0]) * g.abs()).t() @ xd.abs() + u * dw.abs()
    return (loss, loss_bound), (dx, dx_bound), (dw, dw_bound)


def run(x, w, t, up, **kw):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = Fn.lm_head_cross_entropy(x, w, t, reduction="none", **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), up))


def check(got, want):
    for name, a, (value, bound) in zip(("loss", "dx", "dw"), got, want):
        off = (a.double() - value).abs()
        assert (off <= bound * 1.01 + 1e-37).all(), (name, float((off - bound).max()), float(off.max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden,vocab", [
    (1, 64, 8), (3, 8, 17), (63, 72, 1001), (64, 256, 320), (65, 64, 257), (129, 128, 1000), (200, 200, 515),
    (257, 64, 777), (513, 136, 300), (300, 1024, 50257),
])
@pytest.mark.parametrize("cap,z", [(30.0, 0.0), (5.0, 1e-2), (None, 1e-3), (200.0, 0.1)])
def test_capped_head(device, rows, hidden, vocab, cap, z, dtype) -> None:
    x, w, t, up = make(rows, hidden, vocab, dtype, device)
    got = run(x, w, t, up, logit_cap=cap, z_loss=z)
    check(got, reference(x, w, t, up, cap, z))
    again = run(x, w, t, up, logit_cap=cap, z_loss=z)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("rows,hidden,vocab", [
    (65, 72, 66001),  # few rows, a long table
    (257, 64, 16001), (200, 136, 33001), (1025, 64, 33001),
    (4100, 8, 33001),  # a gradient larger than the last-level cache
])
@pytest.mark.parametrize("cap,z", [(30.0, 1e-3), (None, 1e-3)])
def test_every_tile_size(device, rows, hidden, vocab, cap, z) -> None:
    """(With neither cap nor penalty it is the plain head that runs, whose logits are
    rounded to bf16: those of 20 by up to 20 * 2^-8 = 0.08, past these bounds.)"""
    x, w, t, up = make(rows, hidden, vocab, torch.bfloat16, device)
    check(run(x, w, t, up, logit_cap=cap, z_loss=z), reference(x, w, t, up, cap, z))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_chunks_and_reductions(device, dtype) -> None:
    x, w, t, up = make(300, 64, 500, dtype, device)
    check(run(x, w, t, up, logit_cap=10.0, chunk=128), reference(x, w, t, up, 10.0, 0.0))
    none = Fn.lm_head_cross_entropy(x.view(3, 100, 64), w, t.view(3, 100), reduction="none", logit_cap=10.0)
    assert none.shape == (3, 100)
    total = Fn.lm_head_cross_entropy(x, w, t, reduction="sum", logit_cap=10.0)
    mean = Fn.lm_head_cross_entropy(x, w, t, logit_cap=10.0)
    assert torch.allclose(total, none.sum(), rtol=1e-6) and torch.allclose(mean, none.sum() / (t != -100).sum(), rtol=1e-6)
    with pytest.raises(ValueError, match="targets contain ids"):
        Fn.lm_head_cross_entropy(x, w, t.clamp_min(0) + 500, logit_cap=10.0)


def test_edges(device) -> None:
    """No rows; nothing but ignored targets; views; hidden states of any magnitude."""
    for dtype in (torch.bfloat16, torch.float32):
        x, w, t, up = make(5, 64, 100, dtype, device)
        loss, dx, dw = run(x[:0], w, t[:0], up[:0], logit_cap=30.0)
        assert loss.shape == (0,) and dx.shape == (0, 64) and (dw == 0).all()
        loss, dx, dw = run(x, w, torch.full_like(t, -100), up, logit_cap=30.0, z_loss=0.1)
        assert (loss == 0).all() and (dx == 0).all() and (dw == 0).all()
        wide = torch.randn(100, 200, device=device).to(dtype)
        got = run(x, wide[:, 8:72], t, up, logit_cap=30.0)
        check(got, reference(x, wide[:, 8:72], t, up, 30.0, 0.0))
        # logits far beyond the cap: its value and no slope
        loss, dx, dw = run(x * 1e4, w, t, up, logit_cap=30.0)
        assert loss.isfinite().all() and dx.isfinite().all() and dw.isfinite().all()
        check((loss, dx, dw), reference(x * 1e4, w, t, up, 30.0, 0.0))


@pytest.mark.parametrize("rows,vocab", [(5, 97), (300, 1003), (129, 20001)])
def test_rows_behind_the_table(device, rows, vocab) -> None:
    """A table that is the front of a larger one, whose other rows are not numbers."""
    x, w, t, up = make(rows, 64, vocab, torch.bfloat16, device)
    wide = torch.full((vocab + 9, 64), math.nan, dtype=w.dtype, device=device)
    wide[:vocab] = w
    got = run(x, wide[:vocab], t, up, logit_cap=20.0)
    check(got, reference(x, w, t, up, 20.0, 0.0))


def test_tied_with_the_embedding(device) -> None:
    """The table's two gradients meet in the embedding's backward, as without a cap."""
    g = torch.Generator().manual_seed(3)
    w = (torch.randn(96, 64, generator=g) * 0.3).bfloat16().to(device).requires_grad_(True)
    ids = torch.randint(0, 96, (40,), generator=g).to(device)
    t = torch.randint(0, 96, (40,), generator=g).to(device)
    tie = Fn.TiedGrad()
    h = Fn.embedding(w, ids, tie)
    (tied,) = torch.autograd.grad(Fn.lm_head_cross_entropy(h, w, t, logit_cap=8.0, tie=tie), w)
    v = w.detach().requires_grad_(True)
    h = Fn.embedding(v, ids)
    loss = Fn.lm_head_cross_entropy(h, v, t, logit_cap=8.0)
    (both,) = torch.autograd.grad(loss, v)
    assert torch.equal(tied, both)


def test_gradient_against_differences(device) -> None:
    x, w, t, up = make(7, 16, 33, torch.float32, device)
    got = run(x, w, t, up, logit_cap=3.0, z_loss=0.05)
    g = torch.Generator().manual_seed(5)
    f = lambda a, b: float((reference(a, b, t, up, 3.0, 0.05)[0][0] * up.double()).sum())  # noqa: E731
    for k in (0, 1):
        leaves = [x.double(), w.double()]
        step = torch.randn(leaves[k].shape, generator=g, dtype=torch.float64).to(device)
        up_, down = list(leaves), list(leaves)
        up_[k], down[k] = leaves[k] + 1e-4 * step, leaves[k] - 1e-4 * step
        slope = (f(*up_) - f(*down)) / 2e-4
        # h^2 times a third derivative of order 10, and the fp32 sums of the gradient
        assert abs(float((got[1 + k].double() * step).sum()) - slope) < 1e-5 * (float(step.norm()) + abs(slope))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_mean_of_a_batch(device, dtype) -> None:
    """[batch, tokens, hidden] states, the mean's gradient, and a table that needs none."""
    x, w, t, _ = make(60, 64, 333, dtype, device)
    leaves = x.view(3, 20, 64).requires_grad_(True), w.requires_grad_(True)
    loss = Fn.lm_head_cross_entropy(*leaves, t.view(3, 20), logit_cap=10.0, z_loss=1e-2)
    dx, dw = torch.autograd.grad(loss, leaves)
    n = int((t != -100).sum())
    up = torch.full((60,), 1.0 / n, device=device)
    (value, bound), (dx64, dx_bound), (dw64, dw_bound) = reference(x.detach(), w.detach(), t, up, 10.0, 1e-2)
    # the weights 1 / n are rounded, and the mean adds 60 terms in fp32
    eps = 2.0**-23
    assert abs(float(loss.detach()) - float(value.sum()) / n) <= float(bound.sum()) / n + 70 * eps * float(value.sum()) / n
    for got, want, b in ((dx.view(60, 64), dx64, dx_bound), (dw, dw64, dw_bound)):
        assert ((got.double() - want).abs() <= b * 1.01 + eps * want.abs() + 1e-37).all()
    (alone,) = torch.autograd.grad(Fn.lm_head_cross_entropy(leaves[0], w.detach(), t.view(3, 20), logit_cap=10.0, z_loss=1e-2),
                                   leaves[0])
    assert torch.equal(alone, dx)
    (alone,) = torch.autograd.grad(Fn.lm_head_cross_entropy(x.detach(), leaves[1], t, logit_cap=10.0, z_loss=1e-2), leaves[1])
    assert torch.equal(alone, dw)
