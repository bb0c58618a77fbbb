"""The operators of a model with capped scores together, with inputs on which every option
changes the result well beyond the roundings: none may be lost between a model and its
kernels, in either type."""

from __future__ import annotations

import functools
import math

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import HipKernelBackend

B, S, HIDDEN, HEADS, KV, VOCAB = 2, 140, 128, 4, 2, 331
D = HIDDEN // HEADS
OPTIONS = dict(scale=6.0, score_cap=3.0, slopes=(0.2, 0.05, 0.1, 0.02), window=25, documents=True, prefix=(30, 0),
               logit_cap=2.0, z=0.1)
OFF = dict(scale=7.0, score_cap=None, slopes=None, window=None, documents=False, prefix=None, logit_cap=None, z=0.0)


def make(dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std: (torch.randn(*s, generator=g) * std).to(dtype)  # noqa: E731
    weights = [n(VOCAB, HIDDEN, std=0.15)]
    for _ in range(2):
        weights += [n(HIDDEN, HIDDEN, std=1.6 * HIDDEN**-0.5), n(KV * D, HIDDEN, std=1.6 * HIDDEN**-0.5),
                    n(KV * D, HIDDEN, std=HIDDEN**-0.5), n(HIDDEN, HIDDEN, std=HIDDEN**-0.5)]
    ids = torch.randint(0, VOCAB, (B, S), generator=g)
    targets = torch.roll(ids, -1, 1)
    targets[:, -1] = -100
    docs = torch.cumsum(torch.rand(B, S, generator=g) < 1 / 40, 1).to(torch.int32)
    docs[1, S - 20:] = -1
    targets[1, S - 20:] = -100
    return weights, ids, targets, docs, torch.rand(B, S, generator=g) / (B * S)


def step(weights, ids, targets, docs, up, o):
    """The tokens' losses and the weights' gradients by this library."""
    dev = ids.device
    leaves = [w.detach().requires_grad_(True) for w in weights]
    backend, tie = HipKernelBackend(), Fn.TiedGrad()
    x = Fn.embedding(leaves[0], ids, tie, scale=o["scale"])
    kw = dict(score_cap=o["score_cap"], window=o["window"],
              distance_slopes=torch.tensor(o["slopes"], device=dev) if o["slopes"] else None,
              documents=Fn.document_runs(docs) if o["documents"] else None,
              prefix=torch.tensor(o["prefix"], dtype=torch.int32, device=dev) if o["prefix"] else None)
    for wq, wk, wv, wo in (leaves[1:5], leaves[5:]):
        q, k, v = (Fn.linear(x, w).view(B, S, -1, D).transpose(1, 2) for w in (wq, wk, wv))
        x = x + Fn.linear(backend.local_attention(q, k, v, **kw).transpose(1, 2).reshape(B, S, HIDDEN), wo)
    loss = Fn.lm_head_cross_entropy(x, leaves[0], targets, reduction="none", validate=False, tie=tie,
                                    logit_cap=o["logit_cap"], z_loss=o["z"])
    return [loss.detach(), *torch.autograd.grad(loss, leaves, up)]


class Rounded(torch.autograd.Function):
    """A value, and its gradient, held in bf16."""

    @staticmethod
    def forward(ctx, x):
        return x.bfloat16().double()

    @staticmethod
    def backward(ctx, grad):
        return grad.bfloat16().double()


def step64(weights, ids, targets, docs, up, o, keep=lambda t: t):
    """The same from the formulas, in 64 bits on the CPU; keep: what an operator does to its
    output (and to the gradient that comes back)."""
    leaves = [w.detach().double().requires_grad_(True) for w in weights]
    x = keep(leaves[0][ids] * o["scale"])
    pos = torch.arange(S)
    far = pos[:, None] - pos
    seen = (far >= 0)[None].expand(B, S, S)
    if o["prefix"]:
        seen = seen | (pos[None, None] < torch.tensor(o["prefix"])[:, None, None])
    if o["window"]:
        seen = seen & (far.abs() < o["window"])
    if o["documents"]:
        run = torch.cumsum(torch.nn.functional.pad(docs[:, 1:] != docs[:, :-1], (1, 0)), 1)
        seen = seen & (run[:, :, None] == run[:, None]) & (docs >= 0)[:, :, None]
    for wq, wk, wv, wo in (leaves[1:5], leaves[5:]):
        q, k, v = (keep(x @ w.t()).view(B, S, -1, D).transpose(1, 2) for w in (wq, wk, wv))
        k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
        s = q @ k.transpose(2, 3) / math.sqrt(D)
        if o["score_cap"]:
            s = o["score_cap"] * torch.tanh(s / o["score_cap"])
        if o["slopes"]:
            s = s - torch.tensor(o["slopes"], dtype=torch.float64)[None, :, None, None] * far.abs()
        p = torch.softmax(s.masked_fill(~seen[:, None], -1e300), 3) * seen[:, None]
        x = keep(x + keep(keep(keep(p) @ v).transpose(1, 2).reshape(B, S, HIDDEN) @ wo.t()))
    y = keep(x @ leaves[0].t())  # (its gradient is an operand of the next products)
    if o["logit_cap"]:
        y = o["logit_cap"] * torch.tanh(y / o["logit_cap"])
    lse = torch.logsumexp(y, 2)
    loss = (lse - y.gather(2, targets.clamp_min(0)[:, :, None])[:, :, 0] + o["z"] * lse**2) * (targets != -100)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, up.double())]


def distance(a, b) -> list[float]:
    return [float((x.cpu().double() - y).norm() / y.norm()) for x, y in zip(a, b)]


@functools.lru_cache
def bounds(dtype) -> tuple:
    """(the 64-bit result, how far each part of this library's may be from it).  bf16: three
    times what rounding every operator's output and gradient once does to the formulas (the
    same count of roundings, at other places, and other sums).  fp32: that scaled by the
    ratio of the two types' steps, times the length of the sums, at most 512 terms."""
    args = make(dtype)
    want = step64(*args, OPTIONS)
    bf16 = make(torch.bfloat16)
    off = distance(step64(*bf16, OPTIONS, Rounded.apply), step64(*bf16, OPTIONS))
    return want, [3 * x if dtype == torch.bfloat16 else 3 * x * 2.0**-16 * 512**0.5 for x in off]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("option", list(OPTIONS))
def test_every_option_shows(option, dtype) -> None:
    """In 64 bits, on the CPU: a result without one of the options is told from the right one."""
    want, bound = bounds(dtype)
    other = distance(step64(*make(dtype), {**OPTIONS, option: OFF[option]}), want)
    assert any(x > 2 * b for x, b in zip(other, bound)), (other, bound)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_against_64_bits(device, dtype) -> None:
    want, bound = bounds(dtype)
    got = step(*([w.to(device) for w in t] if isinstance(t, list) else t.to(device) for t in make(dtype)), OPTIONS)
    off = distance(got, want)
    assert all(x <= b for x, b in zip(off, bound)), list(zip(off, bound))


@pytest.mark.gpu
@pytest.mark.parametrize("option", list(OPTIONS))
def test_every_option_alone(device, option) -> None:
    """Without one option, as the formulas without it: none stands in for another."""
    options = {**OPTIONS, option: OFF[option]}
    args = make(torch.bfloat16)
    want = step64(*args, options)
    bound = [3 * x for x in distance(step64(*args, options, Rounded.apply), want)]
    got = step(*([w.to(device) for w in t] if isinstance(t, list) else t.to(device) for t in args), options)
    off = distance(got, want)
    assert all(x <= b for x, b in zip(off, bound)), list(zip(off, bound))
