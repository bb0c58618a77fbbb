"""The operators of a model with capped scores together, as a decoder uses them: scaled
embedding, capped and distance-biased attention over packed documents, and the capped tied
LM head with its penalty; against 64 bits, captured and replayed, and on several streams."""

from __future__ import annotations

import math

import pytest
import torch
import torch.utils.checkpoint

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import HipKernelBackend

pytestmark = pytest.mark.gpu

B, S, HIDDEN, HEADS, KV, VOCAB = 2, 150, 128, 4, 2, 331
D = HIDDEN // HEADS
SCALE, SCORE_CAP, LOGIT_CAP, Z = 8.0, 20.0, 15.0, 1e-3


def make(dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    n = lambda *s, std: (torch.randn(*s, generator=g) * std).to(dtype).to(device)  # noqa: E731
    weights = [n(VOCAB, HIDDEN, std=0.1)]
    for _ in range(2):
        weights += [n(HIDDEN, HIDDEN, std=HIDDEN**-0.5), n(KV * D, HIDDEN, std=HIDDEN**-0.5),
                    n(KV * D, HIDDEN, std=HIDDEN**-0.5), n(HIDDEN, HIDDEN, std=0.3 * HIDDEN**-0.5)]
    ids = torch.randint(0, VOCAB, (B, S), generator=g).to(device)
    targets = torch.roll(ids, -1, 1)
    targets[:, -1] = -100
    docs = torch.cumsum(torch.rand(B, S, generator=g) < 1 / 40, 1).to(torch.int32)
    docs[1, S - 20:] = -1  # padding, which trains nothing
    targets[1, S - 20:] = -100
    up = (torch.rand(B, S, generator=g) / (B * S)).to(device)
    return weights, ids, targets, docs.to(device), up


def slopes(device):
    return torch.exp2(-2.0 * torch.arange(1, HEADS + 1, device=device, dtype=torch.float32))


def forward(weights, ids, targets, docs, bias):
    """The losses of the tokens by this library."""
    backend = HipKernelBackend()
    table, layers = weights[0], weights[1:]
    tie = Fn.TiedGrad()
    x = Fn.embedding(table, ids, tie, scale=SCALE)
    runs = Fn.document_runs(docs)
    for wq, wk, wv, wo in (layers[:4], layers[4:]):
        q, k, v = (Fn.linear(x, w).view(B, S, -1, D).transpose(1, 2) for w in (wq, wk, wv))
        o = backend.local_attention(q, k, v, score_cap=SCORE_CAP, distance_slopes=bias, documents=runs, window=90)
        x = x + Fn.linear(o.transpose(1, 2).reshape(B, S, HIDDEN), wo)
    return Fn.lm_head_cross_entropy(x, table, targets, reduction="none", validate=False, tie=tie,
                                    logit_cap=LOGIT_CAP, z_loss=Z)


def step(weights, ids, targets, docs, up, bias):
    leaves = [w.detach().requires_grad_(True) for w in weights]
    loss = forward(leaves, ids, targets, docs, bias)
    return [loss.detach(), *torch.autograd.grad(loss, leaves, up)]


def step64(weights, ids, targets, docs, up):
    """The same from the formulas, in 64 bits on the CPU."""
    f = torch.float64
    leaves = [w.detach().cpu().to(f).requires_grad_(True) for w in weights]
    ids, targets, docs, up = (t.cpu() for t in (ids, targets, docs, up))
    x = leaves[0][ids] * SCALE
    run = torch.cumsum(torch.nn.functional.pad(docs[:, 1:] != docs[:, :-1], (1, 0)), 1)
    pos = torch.arange(S)
    far = pos[:, None] - pos
    seen = (run[:, :, None] == run[:, None]) & (docs >= 0)[:, :, None] & (far >= 0) & (far < 90)
    bias = slopes("cpu").to(f)[None, :, None, None] * far.abs()
    for wq, wk, wv, wo in (leaves[1:5], leaves[5:]):
        q, k, v = ((x @ w.t()).view(B, S, -1, D).transpose(1, 2) for w in (wq, wk, wv))
        k, v = (t.repeat_interleave(HEADS // KV, 1) for t in (k, v))
        s = SCORE_CAP * torch.tanh(q @ k.transpose(2, 3) / math.sqrt(D) / SCORE_CAP) - bias
        p = torch.softmax(s.masked_fill(~seen[:, None], -1e300), 3) * seen[:, None]
        x = x + (p @ v).transpose(1, 2).reshape(B, S, HIDDEN) @ wo.t()
    y = LOGIT_CAP * torch.tanh(x @ leaves[0].t() / LOGIT_CAP)
    lse = torch.logsumexp(y, 2)
    used = targets != -100
    loss = (lse - y.gather(2, targets.clamp_min(0)[:, :, None])[:, :, 0] + Z * lse**2) * used
    return [loss.detach(), *torch.autograd.grad(loss, leaves, up.to(f))]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_against_64_bits(device, dtype) -> None:
    """From a leaf to its gradient lie at most 32 operators (16 forward, 16 back).  In bf16
    each rounds its outputs, and attention and the head their operands, by half a step at
    most: the norm of the error is below 2 * 32 half steps of the result's, where the
    errors of later operators' inputs pass on unamplified (scores and logits of a few units,
    which the caps hold).  In fp32 each sum of n <= 512 terms adds n + 8 half steps."""
    weights, *rest = make(dtype, device)
    got = step(weights, *rest, slopes(device))
    want = step64(weights, *rest)
    half = torch.finfo(dtype).eps / 2
    bound = 64 * half if dtype == torch.bfloat16 else 32 * 520 * half
    for i, (a, b) in enumerate(zip(got, want)):
        off = (a.cpu().double() - b).norm() / b.norm()
        assert off <= bound, (i, float(off), bound)
    # tokens that train nothing have no loss
    assert (got[0][rest[1] == -100] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_and_replayed(device, dtype) -> None:
    """Two graphs of the step, replayed in turn on new inputs with eager steps between, give
    the eager step's bits."""
    weights, ids, targets, docs, up = make(dtype, device)
    bias = slopes(device)
    step(weights, ids, targets, docs, up, bias)  # loads what the first call loads
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        fixed = [t.clone() for t in (ids, targets, docs, up)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(weights, *fixed, bias)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(weights, *fixed, bias)
        graphs.append((graph, fixed, out))
    for turn in range(4):
        for n, (graph, fixed, out) in enumerate(graphs):
            _, *new = make(dtype, device, seed=10 * turn + n)
            for a, b in zip(fixed, new):
                a.copy_(b)
            want = step(weights, *new, bias)
            graph.replay()
            noise = step(weights, *make(dtype, device, seed=99)[1:], bias)  # eager work behind the replay
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (turn, n)
            assert all(t.isfinite().all() for t in noise)


def test_on_two_streams_at_once(device) -> None:
    args = [make(torch.bfloat16, device, seed) for seed in range(2)]
    bias = slopes(device)
    want = [step(*a, bias) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in args]
    got = [[], []]
    for _ in range(5):
        for n, (stream, a) in enumerate(zip(streams, args)):
            with torch.cuda.stream(stream):
                got[n].append(step(*a, bias))
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        assert all(torch.equal(x, y) for run in runs for x, y in zip(run, w))


def test_generation_agrees_with_training(device) -> None:
    """One token at a time over a cache that fills up gives the rows of the whole sequence:
    both within half a step of bf16 (2^-8), and as much for the weights they round."""
    g = torch.Generator().manual_seed(5)
    b, h, kv, s, d = 3, 8, 2, 130, 64
    q, k, v = (torch.randn(b, n, s, d, generator=g).bfloat16().to(device) for n in (h, kv, kv))
    bias = torch.exp2(-torch.arange(1, h + 1, device=device, dtype=torch.float32))
    kw = dict(score_cap=30.0, distance_slopes=bias, window=70)
    whole = Fn.scored_attention(q, k, v, **kw)
    cache_k, cache_v = (torch.full((b, kv, 200, d), math.nan, device=device).bfloat16() for _ in range(2))
    start = torch.tensor([0, 40, 100], dtype=torch.int32, device=device)
    for n in range(3):
        cache_k[n, :, : int(start[n])] = k[n, :, : int(start[n])]
        cache_v[n, :, : int(start[n])] = v[n, :, : int(start[n])]
    top = float(v.abs().max())
    for t in range(30):
        for n in range(3):
            at = int(start[n]) + t
            cache_k[n, :, at], cache_v[n, :, at] = k[n, :, at], v[n, :, at]
        new = torch.stack([q[n, :, int(start[n]) + t] for n in range(3)])[:, :, None]
        one = HipKernelBackend().local_attention(new, cache_k, cache_v, sequence_offset=start + t, **kw)
        want = torch.stack([whole[n, :, int(start[n]) + t] for n in range(3)])[:, :, None]
        assert one.isfinite().all()
        assert (one.float() - want.float()).abs().max() <= 4 * 2.0**-8 * top, t


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("heads", [4, 40])  # the keys shared out over workgroups, or walked in one go
def test_checkpointed_and_offloaded(device, dtype, heads) -> None:
    """Recomputed in the backward, or with saved tensors that come back from the host in
    another layout: the same bits."""
    g = torch.Generator().manual_seed(7)
    q, k, v, do = (torch.randn(2, 130, n, 64, generator=g).to(dtype).to(device).transpose(1, 2)
                   for n in (heads, 2, 2, heads))
    docs = torch.cumsum(torch.rand(2, 130, generator=g) < 0.03, 1).to(torch.int32).to(device)

    def attend(q, k, v):
        return Fn.scored_attention(q, k, v, score_cap=20.0, documents=docs, window=50)

    def gradients(f):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = f(*leaves)
        return [o.detach(), *torch.autograd.grad(o, leaves, do)]

    want = gradients(attend)
    for got in (gradients(lambda *t: torch.utils.checkpoint.checkpoint(attend, *t, use_reentrant=False)),
                gradients(lambda *t: offloaded(attend, *t))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def offloaded(f, *args):
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu().contiguous(), lambda t: t.cuda()):
        return f(*args)


def test_head_and_embedding_checkpointed(device) -> None:
    weights, ids, targets, *_ = make(torch.bfloat16, device)

    def tokens(w):
        x = Fn.embedding(w, ids, scale=SCALE)
        return Fn.lm_head_cross_entropy(x, w, targets, reduction="none", validate=False, logit_cap=LOGIT_CAP, z_loss=Z)

    def gradient(f):
        w = weights[0].detach().requires_grad_(True)
        loss = f(w)
        return loss.detach(), *torch.autograd.grad(loss, w, torch.ones_like(loss))

    want = gradient(tokens)
    for got in (gradient(lambda w: torch.utils.checkpoint.checkpoint(tokens, w, use_reentrant=False)),
                gradient(lambda w: offloaded(tokens, w))):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
