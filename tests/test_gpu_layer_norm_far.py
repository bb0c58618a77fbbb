"""layer_norm of fp32 rows that lie far from zero for their spread, against 64 bits."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu

U = 2.0**-24
EPS = 1e-5


def bounds(h, w):
    """n in 64 bits, how far the forward's may be off it and how far the backward's, and s.

    A sum of up to 16,384 fp32 terms, added at most 32 in a row and then pairwise, divided, is off by
    46 u of the mean of their sizes (u = 2^-24): the mean by e = 46 u mean|h|.  The differences d from
    it are off by u |d| each, their mean by 46 u mean|d| more, and taking it off them is a rounding.
    The variance is off by 50 u of mean d^2 = var + e^2 and by what the square of the second mean,
    at most e, is: s is by half of that relative to var + eps, and by 6 u for root, quotient
    and products.  The backward's mean is rounded once: u of it."""
    h = h.double()
    mean = h.mean(1, keepdim=True)
    var = h.var(1, correction=0, keepdim=True)
    s = 1 / torch.sqrt(var + EPS)
    n = (h - mean) * s
    e = 46 * U * h.abs().mean(1, keepdim=True)
    d = (h - mean).abs() + e
    size = d.mean(1, keepdim=True)
    r = (50 * U * (var + e * e) + 2 * e * 46 * U * size + U * e * e) / (2 * (var + EPS)) + 6 * U
    off = s * (48 * U * size + 3 * U * d) + n.abs() * r
    return n, off * 1.01, (off + s * U * mean.abs()) * 1.01


def make(cols, center, spread, device, rows=12):
    g = torch.Generator().manual_seed(cols)
    x = (torch.randn(rows, cols, generator=g) * spread + center).to(device)
    w, b = (torch.randn(cols, generator=g).to(device) for _ in range(2))
    return x, w, b, torch.randn(rows, cols, generator=g).to(device)


@pytest.mark.parametrize("cols", [3, 64, 768, 1001, 2736, 5000, 9000, 16384])
@pytest.mark.parametrize("center,spread", [(0.0, 1.0), (1000.0, 1.0), (-1e6, 3.0), (1234.567, 0.0), (0.37, 0.0), (-1e8, 0.0)])
@pytest.mark.parametrize("residual", [False, True])
def test_far_rows(device, cols, center, spread, residual) -> None:
    x, w, b, dy = make(cols, center, spread, device)
    r = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).to(device) * spread if residual else None
    x, w, b = (t.requires_grad_(True) for t in (x, w, b))
    y = Fn.layer_norm(x, w, b, EPS, residual=r)
    y, h = y if residual else (y, x)
    n, forward, backward = bounds(h.detach(), w)
    wd = w.detach().double()
    want = n * wd + b.detach().double()
    assert ((y.detach().double() - want).abs() <= forward * wd.abs() + 2 * U * (n * wd).abs() + 2 * U * want.abs()).all()
    dw, db = torch.autograd.grad(y, (w, b), dy)
    d = dy.double()
    # sums over the 12 rows: at most 40 added in a row
    off = (d.abs() * backward).sum(0) + 42 * U * (d * n).abs().sum(0)
    assert ((dw.double() - (d * n).sum(0)).abs() <= off).all()
    assert ((db.double() - d.sum(0)).abs() <= 42 * U * d.abs().sum(0)).all()
