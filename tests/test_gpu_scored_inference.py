"""scored_attention without gradients: the kernel of long prompts, whose probabilities
enter as one bf16 term, at every tile size and way of forming scores, against 64 bits."""

from __future__ import annotations

import math

import pytest
import torch

import nano_megatron_amd.functional as Fn
from tests.scored import check, reference
from tests.test_gpu_scored_attention import ids, make

pytestmark = pytest.mark.gpu


def compare(q, k, v, *, sequence_offset=0, score_cap=None, distance_slopes=None, **kw):
    with torch.no_grad():
        got = Fn.scored_attention(q, k, v, sequence_offset=sequence_offset, score_cap=score_cap,
                                  distance_slopes=distance_slopes, **kw)
        again = Fn.scored_attention(q, k, v, sequence_offset=sequence_offset, score_cap=score_cap,
                                    distance_slopes=distance_slopes, **kw)
    want = reference(q, k, v, offset=sequence_offset, cap=score_cap, slopes=distance_slopes, **kw)
    check("o", got, want["o"])
    assert torch.equal(got, again)
    return got


# more than 64 tiles of 64 queries (64 queries a workgroup), and more than 1,024 (128)
SHAPES = [
    (3, 24, 8, 65, 65, 64), (1, 20, 4, 257, 257, 64), (2, 34, 2, 63, 190, 128), (5, 14, 7, 33, 200, 80),
    (1, 18, 6, 300, 40, 32), (6, 24, 4, 200, 200, 128), (2, 40, 8, 130, 130, 96), (2, 40, 8, 130, 130, 104),
    (16, 33, 3, 129, 129, 64), (17, 32, 4, 100, 300, 128), (9, 16, 16, 513, 513, 64), (33, 16, 2, 70, 65, 88),
]


@pytest.mark.parametrize("cap,slopes", [(None, False), (20.0, False), (None, True), (50.0, True), (90.0, False)])
@pytest.mark.parametrize("shape", SHAPES)
def test_scores(device, shape, cap, slopes) -> None:
    _, hq, _, sq, sk, _ = shape
    q, k, v, _ = make(*shape, torch.bfloat16, device)
    sl = torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq).to(device) if slopes else None
    compare(q, k, v, sequence_offset=sk - sq, score_cap=cap, distance_slopes=sl)
    compare(q, k, v, causal=False, score_cap=cap, distance_slopes=sl)


@pytest.mark.parametrize("cap", [None, 30.0])
@pytest.mark.parametrize("b,h,s,mean,pad,window,prefix,d", [
    (2, 24, 300, 90, 33, 50, None, 64), (2, 24, 200, 60, 10, None, [70, 0], 64), (3, 24, 190, 1000, 1, 64, [190, 5, 64], 128),
    (1, 72, 520, 130, 64, 200, [300], 64), (9, 40, 200, 40, 20, None, None, 96), (2, 40, 900, 250, 30, 300, [40, 800], 64),
])
def test_masks(device, cap, b, h, s, mean, pad, window, prefix, d) -> None:
    q, k, v, _ = make(b, h, h // 4, s, s, d, torch.bfloat16, device)
    docs = ids(b, s, mean, device, pad=pad)
    pre = torch.tensor(prefix, dtype=torch.int32, device=device) if prefix else None
    sl = torch.exp2(-8.0 * torch.arange(1, h + 1) / h).to(device)
    got = compare(q, k, v, documents=docs, window=window, prefix=pre, score_cap=cap, distance_slopes=sl)
    assert (got.transpose(1, 2)[docs < 0] == 0).all()


@pytest.mark.parametrize("cap", [None, 30.0])
@pytest.mark.parametrize("sq", [65, 250])
def test_prompts_of_unequal_length(device, cap, sq) -> None:
    """Chunks of prompts over a cache of which every row has filled another part."""
    offs = torch.tensor([-50, -3, 0, 41, 170, 400, 90, 1], dtype=torch.int32, device=device)
    q, k, v, _ = make(8, 16, 4, sq, 400, 64, torch.bfloat16, device)
    for kw in ({}, {"window": 60}, {"documents": ids(8, 400, 70, device, pad=5)}):
        compare(q, k, v, sequence_offset=offs, score_cap=cap, **kw)


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("cap", [None, 20.0])
@pytest.mark.parametrize("b,d", [(2, 64), (2, 128), (16, 64)])
def test_hidden_rows_may_hold_anything(device, b, d, cap, value) -> None:
    h, s = 20, 260
    q, k, v, _ = make(b, h, 5, s, s, d, torch.bfloat16, device)
    docs = torch.zeros(b, s, dtype=torch.int32, device=device)
    docs[:, 40:] = 1
    docs[:, 75:] = -1
    docs[0, 75:110] = 3
    want = reference(q, k, v, documents=docs, cap=cap)["o"]
    for t in (q, k, v):
        t.transpose(1, 2)[docs < 0] = value
    with torch.inference_mode():
        got = Fn.scored_attention(q, k, v, documents=docs, score_cap=cap)
        check("o", got, want)
        # a spoilt value inside a document stays in it
        v[0, :, 50] = value
        got = Fn.scored_attention(q, k, v, documents=docs, score_cap=cap)
    other = docs[0] != 1
    check("o", got[:1, :, other], (want[0][:1, :, other], want[1][:1, :, other]))
    assert not got[0, :, 50:75].isfinite().any() and got[0, :, 40:50].isfinite().all()


def test_strides(device) -> None:
    """Views of a fused projection and of a cache that holds heads before tokens."""
    b, h, d, s = 4, 20, 64, 150
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(b, s, 3 * h * d + 8, generator=g).bfloat16().to(device)
    q, k, v = (qkv[..., n * h * d: (n + 1) * h * d].unflatten(2, (h, d)).transpose(1, 2) for n in range(3))
    compare(q, k, v, score_cap=30.0)
    cache = torch.randn(2, b, 5, 2 * s, d, generator=g).bfloat16().to(device)
    compare(q, cache[0][:, :, :s], cache[1][:, :, s // 2: s // 2 + s], window=40)


def test_captured_and_replayed(device) -> None:
    q, k, v, _ = make(2, 24, 8, 200, 200, 64, torch.bfloat16, device)
    docs = ids(2, 200, 60, device)
    f = lambda: Fn.scored_attention(q, k, v, documents=docs, score_cap=30.0)  # noqa: E731
    with torch.no_grad():
        f()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = f()
        for turn in range(3):
            q.copy_(make(2, 24, 8, 200, 200, 64, torch.bfloat16, device, seed=turn)[0])
            docs.copy_(ids(2, 200, 40, device, seed=turn + 5))
            want = f()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want)
