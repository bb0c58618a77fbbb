"""Layer norm, rotary positions and the head against a teacher together, as a small decoder
uses them: norms with the residual addition, a stretched rotary half of each head, and the
tied head on a teacher's largest logits beside the targets; against 64 bits, captured and
replayed, on several streams, recomputed, and token by token over a cache."""

from __future__ import annotations

import functools
import math

import pytest
import torch
import torch.utils.checkpoint

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import HipKernelBackend

pytestmark = pytest.mark.gpu

B, S, HIDDEN, HEADS, KV, VOCAB, TOP, LAYERS = 2, 150, 128, 2, 1, 331, 9, 2
D = HIDDEN // HEADS
OPTIONS = dict(rotary_dim=32, interleaved=True, magnitude=1.1, first=70_000, temperature=2.0, target_weight=0.5)


def make(dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std, mean=0.0: (torch.randn(*s, generator=g) * std + mean).to(dtype).to(device)  # noqa: E731
    weights = [n(VOCAB, HIDDEN, std=0.5)]
    for _ in range(LAYERS):
        weights += [n(HIDDEN, std=0.1, mean=1.0), n(HIDDEN, std=0.1),
                    n((HEADS + 2 * KV) * D, HIDDEN, std=1.5 * HIDDEN**-0.5), n(HIDDEN, HIDDEN, std=HIDDEN**-0.5)]
    weights += [n(HIDDEN, std=0.1, mean=1.0), n(HIDDEN, std=0.1)]
    ids = torch.randint(0, VOCAB, (B, S), generator=g).to(device)
    targets = torch.roll(ids, -1, 1)
    targets[:, -1] = -100
    values = torch.randn(B, S, TOP, generator=g).sort(2, descending=True).values * 3
    top = torch.argsort(torch.rand(B, S, VOCAB, generator=g), 2)[:, :, :TOP].to(torch.int32)
    top[:, :, 5:][torch.rand(B, S, TOP - 5, generator=g) < 0.5] = -1
    top[1, S - 20:] = -1  # padding, which trains nothing
    targets[1, S - 20:] = -100
    up = (torch.rand(B, S, generator=g) / (B * S)).to(device)
    return weights, ids, targets, values.to(device), top.to(device), up


@functools.lru_cache
def frequencies(device, rotary_dim):
    return Fn.rotary_frequencies(rotary_dim, scaling="parts", factor=16.0, original_length=512, device=device)


def hidden_states(weights, ids, tie=None, o=OPTIONS, attend=None):
    f = frequencies(ids.device, o["rotary_dim"])
    b, s = ids.shape
    branch, x = Fn.embedding(weights[0], ids, tie), None
    for n in range(LAYERS):
        w, bias, qkv, out = weights[1 + 4 * n:5 + 4 * n]
        if x is None:
            y, x = Fn.layer_norm(branch, w, bias), branch
        else:
            y, x = Fn.layer_norm(branch, w, bias, residual=x)
        q, k, v = Fn.linear(y, qkv).view(b, s, HEADS + 2 * KV, D).transpose(1, 2).split((HEADS, KV, KV), 1)
        if attend is None:
            q, k = Fn.rotary_positions(q, k, f, sequence_offset=o["first"], interleaved=o["interleaved"],
                                       magnitude=o["magnitude"])
            a = HipKernelBackend().local_attention(q, k, v)
        else:
            a = attend(n, q, k, v, f)
        branch = Fn.linear(a.transpose(1, 2).reshape(b, s, HIDDEN), out)
    return Fn.layer_norm(branch, weights[-2], weights[-1], residual=x)[0]


def forward(weights, ids, targets, values, top, o=OPTIONS):
    tie = Fn.TiedGrad()
    x = hidden_states(weights, ids, tie, o)
    return Fn.lm_head_distillation(x, weights[0], values, top, targets, temperature=o["temperature"],
                                   target_weight=o["target_weight"], reduction="none", validate=False, tie=tie)


def step(weights, ids, targets, values, top, up, o=OPTIONS, forward=forward):
    leaves = [w.detach().requires_grad_(True) for w in weights]
    loss = forward(leaves, ids, targets, values, top, o)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, up)]


def step64(weights, ids, targets, values, top, up, o=OPTIONS):
    """The same from the formulas, in 64 bits on the CPU."""
    f = torch.float64
    leaves = [w.detach().cpu().to(f).requires_grad_(True) for w in weights]
    ids, targets, values, top, up = (t.cpu() for t in (ids, targets, values, top, up))
    r = o["rotary_dim"]
    angle = (torch.arange(S, dtype=f) + o["first"])[:, None] * frequencies("cpu", r)
    cos, sin = torch.cos(angle) * o["magnitude"], torch.sin(angle) * o["magnitude"]

    def norm(x, w, b):
        d = x - x.mean(2, keepdim=True)
        return d / torch.sqrt((d * d).mean(2, keepdim=True) + 1e-5) * w + b

    def turn(x):
        if o["interleaved"]:
            a, b = x[..., 0:r:2], x[..., 1:r:2]
            both = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = x[..., :r // 2], x[..., r // 2:r]
            both = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        return torch.cat((both, x[..., r:]), -1)

    x = leaves[0][ids]
    hidden = torch.triu(torch.ones(S, S, dtype=torch.bool), 1)
    for n in range(LAYERS):
        w, b, qkv, out = leaves[1 + 4 * n:5 + 4 * n]
        q, k, v = (norm(x, w, b) @ qkv.t()).view(B, S, -1, D).transpose(1, 2).split((HEADS, KV, KV), 1)
        q, k = turn(q), turn(k)
        k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
        p = torch.softmax((q @ k.transpose(2, 3) / math.sqrt(D)).masked_fill(hidden, -1e300), 3)
        x = x + (p @ v).transpose(1, 2).reshape(B, S, HIDDEN) @ out.t()
    z = norm(x, leaves[-2], leaves[-1]) @ leaves[0].t()
    t = o["temperature"]
    p = torch.softmax((values.to(f) / t).masked_fill(top < 0, -1e300), 2) * (top >= 0)
    log_q = torch.log_softmax(z / t, 2).gather(2, top.clamp_min(0).long())
    loss = t * t * (torch.special.xlogy(p, p) - p * log_q).sum(2)
    ce = torch.nn.functional.cross_entropy(z.flatten(0, 1), targets.flatten(), reduction="none", ignore_index=-100)
    loss = loss + o["target_weight"] * ce.view(B, S)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, up.to(f))]


def distance(got, want):
    return [float((a.cpu().double() - b).norm() / b.norm()) for a, b in zip(got, want)]


def bound_of(dtype):
    """From a leaf to its gradient lie at most 40 operators (20 forward, 20 back).  In bf16 each
    rounds its outputs, and attention and the head their operands, by half a step at most: the
    norm of the error is below 2 * 40 half steps of the result's, where the errors of later
    operators' inputs pass on unamplified (scores and logits of a few units, norms of rows of
    unit spread).  In fp32 each sum of n <= 512 terms adds n + 8 half steps."""
    half = torch.finfo(dtype).eps / 2
    return 80 * half if dtype == torch.bfloat16 else 40 * 520 * half


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_against_64_bits(device, dtype) -> None:
    args = make(dtype, device)
    off = distance(step(*args), step64(*args))
    assert max(off) <= bound_of(dtype), off
    # tokens that train nothing have no loss
    assert not step(*args)[0][1, S - 20:].any()


@pytest.mark.parametrize("change", [
    dict(interleaved=False), dict(rotary_dim=64), dict(magnitude=1.0), dict(first=0), dict(temperature=1.0),
    dict(target_weight=0.0),
])
def test_every_option_matters(device, change) -> None:
    """Left out, each option moves the result well past the fp32 bound, the library's and the
    formulas' alike.  (The angles at 70,000 differ from those at 0 by rounding alone: a shift of
    all positions changes nothing.)"""
    args = make(torch.float32, device)
    without = {**OPTIONS, **change}
    got, want = step(*args, without), step64(*args, without)
    assert max(distance(got, want)) <= bound_of(torch.float32)
    moved = max(distance(step(*args), want))
    if "first" in change:
        assert moved <= 2 * bound_of(torch.float32)
    else:
        assert moved > 2 * bound_of(torch.float32)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_and_replayed(device, dtype) -> None:
    """Two graphs of the step, replayed in turn on new inputs with eager steps between, give
    the eager step's bits."""
    weights, *rest = make(dtype, device)
    step(weights, *rest)  # loads what the first call loads
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        fixed = [t.clone() for t in rest]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(weights, *fixed)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(weights, *fixed)
        graphs.append((graph, fixed, out))
    for turn in range(4):
        for n, (graph, fixed, out) in enumerate(graphs):
            _, *new = make(dtype, device, seed=10 * turn + n)
            for a, b in zip(fixed, new):
                a.copy_(b)
            want = step(weights, *new)
            graph.replay()
            noise = step(weights, *make(dtype, device, seed=99)[1:])  # eager work behind the replay
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (turn, n)
            assert all(t.isfinite().all() for t in noise)


def test_on_two_streams_at_once(device) -> None:
    args = [make(torch.bfloat16, device, seed) for seed in range(2)]
    want = [step(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(5):
        for n, (stream, a) in enumerate(zip(streams, args)):
            with torch.cuda.stream(stream):
                got[n].append(step(*a))
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        assert all(torch.equal(x, y) for run in runs for x, y in zip(run, w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_recomputed(device, dtype) -> None:
    """Under a checkpoint of the whole model, or with its saved tensors away on the host."""
    args = make(dtype, device)
    want = step(*args)

    def recomputed(leaves, *rest):
        return torch.utils.checkpoint.checkpoint(forward, leaves, *rest, use_reentrant=False)

    def offloaded(leaves, *rest):
        # (in their layout, which ``attention`` needs; the new operators' own tests change it)
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t.cuda()):
            return forward(leaves, *rest)

    for f in (recomputed, offloaded):
        assert all(torch.equal(a, b) for a, b in zip(step(*args, forward=f), want))


def test_token_by_token(device) -> None:
    """One token at a time, every row at a place of its own, over a cache of rotated keys: the
    rows of the whole sequence, within the roundings of 10 operators of unit-sized outputs."""
    weights, ids, *_ = make(torch.bfloat16, device)
    o = OPTIONS
    whole = hidden_states(weights, ids)
    start = [0, 60]
    cache = [[torch.zeros(B, KV, S, D, device=device, dtype=torch.bfloat16) for _ in range(2)] for _ in range(LAYERS)]
    rows = torch.arange(B, device=device)

    def attend(n, q, k, v, f):
        q, k = Fn.rotary_positions(q, k, f, sequence_offset=place + o["first"], interleaved=o["interleaved"],
                                   magnitude=o["magnitude"])
        for c, new in zip(cache[n], (k, v)):
            c[rows, :, place.long()] = new[:, :, 0]
        return HipKernelBackend().local_attention(q, *cache[n], sequence_offset=place)

    # rows that start later have read what lies before
    for t in range(max(start)):
        place = torch.tensor([0, t], dtype=torch.int32, device=device)
        hidden_states(weights, ids[rows, place.long()][:, None], attend=attend)
    for t in range(25):
        place = torch.tensor([s + t for s in start], dtype=torch.int32, device=device)
        one = hidden_states(weights, ids[rows, place.long()][:, None], attend=attend)
        want = whole[rows, place.long()][:, None]
        assert (one.float() - want.float()).norm() <= 2 * 10 * 2.0**-8 * want.float().norm(), t
