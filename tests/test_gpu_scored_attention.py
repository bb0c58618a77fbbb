"""scored_attention against 64 bits: caps, distance bias, documents, prefix and
window, both directions, at the sizes and masks where tiles end."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn
from tests.scored import check, reference, visible

pytestmark = pytest.mark.gpu


def make(b, hq, hkv, sq, sk, d, dtype, device, seed=0, grow=3.0):
    g = torch.Generator().manual_seed(seed)
    mk = lambda s, h: torch.randn(b, s, h, d, generator=g).to(dtype).to(device).transpose(1, 2)  # noqa: E731
    q = (torch.randn(b, sq, hq, d, generator=g) * grow).to(dtype).to(device).transpose(1, 2)
    return q, mk(sk, hkv), mk(sk, hkv), mk(sq, hq)


def ids(b, s, mean, device, seed=1, pad=0):
    g = torch.Generator().manual_seed(seed)
    t = torch.cumsum(torch.rand(b, s, generator=g) < 1.0 / mean, 1).to(torch.int32)
    if pad:
        t[:, s - pad:] = -1
        t[0, s // 3: s // 3 + pad] = -2  # padding in the middle of a row too
    return t.to(device)


def run(q, k, v, do, **kw):
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    o = Fn.scored_attention(*leaves, **kw)
    return dict(zip(("o", "dq", "dk", "dv"), (o.detach(), *torch.autograd.grad(o, leaves, do))))


def compare(q, k, v, do, *, sequence_offset=0, score_cap=None, distance_slopes=None, **kw):
    got = run(q, k, v, do, sequence_offset=sequence_offset, score_cap=score_cap, distance_slopes=distance_slopes, **kw)
    want = reference(q, k, v, do, offset=sequence_offset, cap=score_cap, slopes=distance_slopes, **kw)
    for name in got:
        check(name, got[name], want[name])
    return got


# b, hq, hkv, sq, sk, d
SHAPES = [
    (1, 1, 1, 1, 1, 64), (2, 2, 1, 2, 3, 128), (1, 4, 2, 63, 63, 64), (2, 2, 2, 64, 64, 128), (1, 6, 2, 65, 65, 80),
    (1, 2, 1, 129, 129, 64), (1, 2, 2, 200, 200, 128), (2, 4, 4, 257, 257, 64), (1, 2, 1, 7, 300, 64),
    (1, 3, 1, 300, 40, 32), (1, 8, 1, 130, 513, 128), (1, 2, 1, 100, 100, 8),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cap,slopes", [(None, False), (20.0, False), (None, True), (50.0, True), (90.0, False)])
@pytest.mark.parametrize("shape", SHAPES)
def test_scores(device, shape, cap, slopes, dtype) -> None:
    b, hq, hkv, sq, sk, d = shape
    q, k, v, do = make(*shape, dtype, device)
    sl = torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq).to(device) if slopes else None
    compare(q, k, v, do, causal=True, sequence_offset=sk - sq, score_cap=cap, distance_slopes=sl)
    compare(q, k, v, do, causal=False, score_cap=cap, distance_slopes=sl)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b,s,mean,pad,window,prefix,d", [
    (2, 70, 5, 9, None, None, 64), (1, 300, 40, 0, None, None, 128), (2, 300, 90, 33, 50, None, 64),
    (2, 200, 60, 10, None, [70, 0], 64), (1, 260, 1, 0, None, None, 64), (3, 190, 1000, 1, 64, [190, 5, 64], 128),
    (1, 130, 30, 129, None, None, 64), (2, 129, 1000, 0, 1, None, 128), (1, 520, 130, 64, 200, [300], 64),
])
def test_masks(device, dtype, causal, b, s, mean, pad, window, prefix, d) -> None:
    q, k, v, do = make(b, 4, 2, s, s, d, dtype, device)
    docs = ids(b, s, mean, device, pad=pad)
    pre = torch.tensor(prefix, dtype=torch.int32, device=device) if prefix and causal else None
    sl = torch.tensor([0.5, 0.01, 2.0, 0.0], device=device)
    got = compare(q, k, v, do, causal=causal, documents=docs, window=window, prefix=pre, score_cap=30.0,
                  distance_slopes=sl)
    seen = visible(b, s, s, causal=causal, offset=0, prefix=pre, window=window, documents=docs)
    empty = ~seen.any(2)
    assert (got["o"].transpose(1, 2)[empty] == 0).all() and (got["dq"].transpose(1, 2)[empty] == 0).all()
    again = run(q, k, v, do, causal=causal, documents=Fn.document_runs(docs), window=window, prefix=pre,
                score_cap=30.0, distance_slopes=sl)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sq", [1, 5, 33])
def test_offsets_per_row(device, dtype, sq) -> None:
    """Rows of unequal length, before, inside and past the keys."""
    offs = torch.tensor([-50, -3, 0, 41, 170, 400], dtype=torch.int32, device=device)
    q, k, v, do = make(6, 4, 2, sq, 200, 64, dtype, device)
    sl = torch.tensor([0.5, 0.01, 2.0, 0.25], device=device)
    for kw in ({}, {"window": 60}, {"distance_slopes": sl}, {"documents": ids(6, 200, 30, device, pad=5)},
               {"prefix": torch.tensor([3, 0, 9, 100, 200, 1], dtype=torch.int32, device=device), "score_cap": 9.0}):
        compare(q, k, v, do, sequence_offset=offs, **kw)
    compare(q, k, v, do, causal=False, sequence_offset=offs, distance_slopes=sl, score_cap=5.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_keys_and_no_queries(device, dtype) -> None:
    for sq, sk in ((3, 0), (0, 3), (0, 0)):
        q, k, v, do = make(2, 2, 1, sq, sk, 64, dtype, device)
        got = run(q, k, v, do, causal=False)
        assert all((t == 0).all() for t in got.values()) and got["o"].shape == q.shape
    q, k, v, do = make(0, 2, 1, 4, 4, 64, dtype, device)
    assert run(q, k, v, do)["dk"].shape == k.shape


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("sq,sk", [(200, 200), (3, 500)])
def test_hidden_rows_may_hold_anything(device, dtype, value, sq, sk) -> None:
    """A spoilt document, padding and the space behind a cache's last key leave the rest as it is."""
    q, k, v, do = make(2, 4, 2, sq, sk, 64, dtype, device)
    docs = torch.zeros(2, sk, dtype=torch.int32, device=device)
    docs[:, 40:] = 1
    docs[:, 75:] = 2
    docs[1, 100:120] = -1
    hole = torch.zeros(2, sk, dtype=torch.bool, device=device)
    hole[1, 100:120] = True
    hole[:, 150:] = True
    docs[hole] = -1
    off = 50 if sq == 3 else 0
    clean = run(q, k, v, do, documents=docs, sequence_offset=off, score_cap=20.0)
    kk, vv, qq, dd = k.clone(), v.clone(), q.clone(), do.clone()
    for t in (kk, vv):
        t.transpose(1, 2)[hole] = value
    if sq == sk:
        for t in (qq, dd):
            t.transpose(1, 2)[hole] = value
    spoilt = run(qq, kk, vv, dd, documents=docs, sequence_offset=off, score_cap=20.0)
    want = reference(q, k, v, do, documents=docs, offset=off, cap=20.0)
    for n in clean:
        check(n, spoilt[n], want[n])
    # a NaN inside a document stays in it
    kk = k.clone()
    kk[0, :, 50] = value
    vv = v.clone()
    vv[0, :, 50] = value
    spoilt = run(q, kk, vv, do, documents=docs, sequence_offset=off, score_cap=20.0)
    other = (docs[0] != 1)[off:off + sq]
    for n in ("o", "dq"):
        w = want[n]
        check(n, spoilt[n][:1, :, other], (w[0][:1, :, other], w[1][:1, :, other]))
    for n in ("dk", "dv"):
        w, other_k = want[n], docs[0] != 1
        check(n, spoilt[n][:1, :, other_k], (w[0][:1, :, other_k], w[1][:1, :, other_k]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sq", [4, 90])
def test_strides(device, dtype, sq) -> None:
    """Views of a fused projection, of a cache with other head and token orders,
    heads shared by a broadcast, misaligned starts; nothing behind a view is written."""
    b, h, d, sk = 2, 4, 64, 150
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(b, sk, 3 * h * d + 8, generator=g).to(dtype).to(device)
    base = qkv.clone()
    q, k, v = (qkv[..., n * h * d: (n + 1) * h * d].unflatten(2, (h, d)).transpose(1, 2) for n in range(3))
    q = q[:, :, sk - sq:]
    do = torch.randn(b, h, sq, d, generator=g).to(dtype).to(device)  # heads before tokens
    compare(q, k, v, do, sequence_offset=sk - sq, score_cap=30.0)
    cache = torch.randn(2, b, h, 2 * sk, d, generator=g).to(dtype).to(device)
    kc, vc = cache[0][:, :, :sk], cache[1][:, :, sk // 2: sk // 2 + sk]
    compare(q, kc, vc, do, sequence_offset=sk - sq, window=40)
    one = torch.randn(b, 1, sk, d, generator=g).to(dtype).to(device).expand(b, h, sk, d)
    compare(q, one, v, do, sequence_offset=sk - sq)
    flat = torch.randn(b * sk * h * d + 3, generator=g).to(dtype).to(device)
    odd = flat[3:].view(b, sk, h, d).transpose(1, 2)
    compare(odd[:, :, :sq], odd, v, do, sequence_offset=sk - sq)
    assert torch.equal(qkv, base)


def test_far_positions(device) -> None:
    """A distance bias far beyond the last key is as exact as next to it."""
    q, k, v, do = make(1, 2, 2, 4, 100, 64, torch.float32, device)
    sl = torch.tensor([0.5, 1.0], device=device)
    compare(q, k, v, do, causal=False, sequence_offset=3_000_000, distance_slopes=sl)
    compare(q, k, v, do, causal=False, sequence_offset=-3_000_000, distance_slopes=sl)


def test_document_runs(device) -> None:
    for b, s, mean in ((1, 1, 3), (3, 17, 2), (2, 8192, 50), (2, 8193, 4000), (1, 30000, 9000), (1, 20001, 1)):
        t = ids(b, s, mean, device, seed=s, pad=s // 5)
        got = Fn.document_runs(t).runs.cpu()
        for i, row in enumerate(t.cpu().tolist()):
            start = 0
            want = []
            for j in range(1, s + 1):
                if j == s or row[j] != row[start]:
                    want += [(start, j if row[start] >= 0 else ~j)] * (j - start)
                    start = j
            assert got[i].tolist() == [list(w) for w in want]
    wide = torch.arange(40, device=device, dtype=torch.int32).view(2, 20) // 3
    assert torch.equal(Fn.document_runs(wide[:, ::2]).runs, Fn.document_runs(wide[:, ::2].contiguous()).runs)


def test_gradient_against_differences(device) -> None:
    """dq, dk, dv in fp32 against central differences of the 64-bit forward."""
    q, k, v, do = make(1, 2, 1, 9, 9, 64, torch.float32, device, grow=1.0)
    kw = dict(score_cap=2.0, distance_slopes=torch.tensor([0.3, 0.1], device=device), window=6)
    got = run(q, k, v, do, **kw)
    f = lambda *t: float((reference(*t, cap=2.0, slopes=kw["distance_slopes"], window=6)["o"][0]  # noqa: E731
                          * do.double()).sum())
    g = torch.Generator().manual_seed(5)
    for name, at in (("dq", 0), ("dk", 1), ("dv", 2)):
        leaves = [t.double() for t in (q, k, v)]
        step = torch.randn(leaves[at].shape, generator=g, dtype=torch.float64).to(device)
        h = 1e-4
        up, down = list(leaves), list(leaves)
        up[at], down[at] = leaves[at] + h * step, leaves[at] - h * step
        slope = (f(*up) - f(*down)) / (2 * h)
        # the difference is off by h^2 times a third derivative (of order 1 to 10 here, times the
        # norm of the step), the gradient by its fp32 sums
        assert abs(float((got[name].double() * step).sum()) - slope) < 1e-5 * float(step.norm()) + 1e-5 * abs(slope)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("b,hq,hkv,sq,sk,d", [
    (1, 2, 2, 1, 33, 64), (2, 8, 1, 1, 2050, 64), (1, 4, 1, 16, 4500, 128), (3, 6, 2, 5, 1100, 80),
    (1, 40, 2, 1, 700, 64), (2, 2, 1, 17, 3000, 64), (1, 2, 1, 64, 2500, 128),
])
def test_few_queries(device, dtype, b, hq, hkv, sq, sk, d) -> None:
    """New tokens against a cache of which every row has filled another part; the
    rest holds NaN.  Both directions (the queries of a short cross attention)."""
    q, k, v, do = make(b, hq, hkv, sq, sk, d, dtype, device)
    g = torch.Generator().manual_seed(4)
    offs = torch.randint(0, sk - sq + 1, (b,), generator=g).to(torch.int32)
    offs[0] = sk - sq
    for i in range(b):
        k[i, :, int(offs[i]) + sq:] = float("nan")
        v[i, :, int(offs[i]) + sq:] = float("nan")
    offs = offs.to(device)
    sl = torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq).to(device)
    for kw in ({"score_cap": 30.0}, {"distance_slopes": sl}, {"window": sk // 3}, {"score_cap": 70.0}, {}):
        compare(q, k, v, do, sequence_offset=offs, **kw)
    docs = ids(b, sk, 200, device, pad=3)
    compare(q, k, v, do, sequence_offset=offs, documents=docs, score_cap=30.0)


def test_long_cache(device) -> None:
    """One token against a cache whose tokens lie past 2^31 bytes."""
    sk, d, wide = 70000, 64, 1 << 14
    g = torch.Generator(device=device).manual_seed(0)
    store = torch.empty(sk, wide + 64, dtype=torch.bfloat16, device=device)
    kv = store.unflatten(1, (-1, 64))[:, :2]
    kv.copy_(torch.randn(sk, 2, d, generator=g, device=device))
    k, v = (kv[:, n].view(1, 1, sk, d) for n in range(2))
    q = torch.randn(1, 2, 1, d, generator=g, device=device).bfloat16()
    for sq in (1, 40):
        qq = q.expand(1, 2, sq, d)
        o = Fn.scored_attention(qq, k, v, sequence_offset=sk - sq, score_cap=30.0)
        want = reference(qq.cpu(), k.contiguous().cpu(), v.contiguous().cpu(), offset=sk - sq, cap=30.0)
        check("o", o.cpu(), want["o"])


# more than 64 tiles of 64 queries, and more than 512 of them: the kernels that walk the keys in one go
WIDE = [
    (3, 24, 8, 65, 65, 64), (2, 34, 2, 63, 63, 128), (1, 20, 4, 257, 257, 64), (1, 18, 6, 300, 40, 32),
    (2, 17, 1, 130, 513, 128), (5, 14, 7, 33, 200, 80), (1, 66, 1, 17, 17, 8), (8, 16, 16, 257, 257, 64),
    (6, 24, 4, 200, 200, 128), (3, 48, 8, 321, 130, 64),
]


@pytest.mark.parametrize("cap,slopes", [(None, False), (20.0, False), (None, True), (50.0, True), (90.0, False)])
@pytest.mark.parametrize("shape", WIDE)
def test_scores_of_many_heads(device, shape, cap, slopes) -> None:
    _, hq, _, sq, sk, _ = shape
    q, k, v, do = make(*shape, torch.bfloat16, device)
    sl = torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq).to(device) if slopes else None
    compare(q, k, v, do, causal=True, sequence_offset=sk - sq, score_cap=cap, distance_slopes=sl)
    compare(q, k, v, do, causal=False, score_cap=cap, distance_slopes=sl)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("b,h,s,mean,pad,window,prefix,d", [
    (2, 24, 70, 5, 9, None, None, 64), (1, 24, 300, 40, 0, None, None, 128), (2, 24, 300, 90, 33, 50, None, 64),
    (2, 24, 200, 60, 10, None, [70, 0], 64), (1, 24, 260, 1, 0, None, None, 64), (3, 24, 190, 1000, 1, 64, [190, 5, 64], 128),
    (1, 24, 130, 30, 129, None, None, 64), (2, 40, 129, 1000, 0, 1, None, 128), (1, 72, 520, 130, 64, 200, [300], 64),
])
def test_masks_of_many_heads(device, causal, b, h, s, mean, pad, window, prefix, d) -> None:
    q, k, v, do = make(b, h, h // 4, s, s, d, torch.bfloat16, device)
    docs = ids(b, s, mean, device, pad=pad)
    pre = torch.tensor(prefix, dtype=torch.int32, device=device) if prefix and causal else None
    sl = torch.exp2(-8.0 * torch.arange(1, h + 1) / h).to(device)
    kw = dict(causal=causal, documents=docs, window=window, prefix=pre, score_cap=30.0, distance_slopes=sl)
    got = compare(q, k, v, do, **kw)
    again = run(q, k, v, do, **kw)
    assert all(torch.equal(got[n], again[n]) for n in got)


@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_hidden_rows_of_many_heads_may_hold_anything(device, value) -> None:
    b, h, s = 2, 20, 200
    q, k, v, do = make(b, h, 5, s, s, 64, torch.bfloat16, device)
    docs = torch.zeros(b, s, dtype=torch.int32, device=device)
    docs[:, 40:] = 1
    docs[:, 75:] = -1
    docs[0, 75:110] = 3
    hole = docs < 0
    want = reference(q, k, v, do, documents=docs, cap=20.0)
    for t in (q, k, v, do):
        t.transpose(1, 2)[hole] = value
    got = run(q, k, v, do, documents=docs, score_cap=20.0)
    for n in got:
        check(n, got[n], want[n])
    # a spoilt key inside a document stays in it
    k[0, :, 50] = value
    got = run(q, k, v, do, documents=docs, score_cap=20.0)
    other = docs[0] != 1
    for n in got:
        w = want[n]
        check(n, got[n][:1, :, other], (w[0][:1, :, other], w[1][:1, :, other]))


@pytest.mark.parametrize("sq", [20, 65])
def test_offsets_per_row_of_many_heads(device, sq) -> None:
    offs = torch.tensor([-50, -3, 0, 41, 170, 400], dtype=torch.int32, device=device)
    q, k, v, do = make(6, 16, 4, sq, 200, 64, torch.bfloat16, device)
    sl = torch.exp2(-0.5 * torch.arange(1, 17)).to(device)
    for kw in ({}, {"window": 60}, {"distance_slopes": sl}, {"documents": ids(6, 200, 30, device, pad=5)},
               {"prefix": torch.tensor([3, 0, 9, 100, 200, 1], dtype=torch.int32, device=device), "score_cap": 9.0}):
        compare(q, k, v, do, sequence_offset=offs, **kw)


@pytest.mark.parametrize("d", [40, 72, 88, 96, 104, 120])
@pytest.mark.parametrize("hq,hkv,sq,sk", [(8, 1, 700, 200), (66, 6, 90, 130), (4, 1, 3, 900)])
def test_head_dims(device, hq, hkv, sq, sk, d) -> None:
    """Also where workgroups share the queries of a key, and the keys of a query."""
    q, k, v, do = make(1, hq, hkv, sq, sk, d, torch.bfloat16, device)
    sl = torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq).to(device)
    compare(q, k, v, do, causal=False, score_cap=30.0)
    compare(q, k, v, do, sequence_offset=sk - sq, distance_slopes=sl)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("d", [1, 3, 33, 127])
def test_odd_head_dims(device, dtype, d) -> None:
    for shape in ((2, 4, 2, 70, 70, d), (1, 4, 1, 2, 200, d)):
        q, k, v, do = make(*shape, dtype, device)
        compare(q, k, v, do, sequence_offset=shape[4] - shape[3], score_cap=30.0)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_broadcast_gradient_and_inference(device, dtype) -> None:
    """The gradient of a sum is one element seen everywhere; without gradients the values are
    those of the same formula (in bf16 the output's rounding apart, whose bound both meet)."""
    q, k, v, _ = make(2, 4, 2, 90, 90, 64, dtype, device)
    leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
    Fn.scored_attention(*leaves, score_cap=20.0).sum().backward()
    want = reference(q, k, v, torch.ones_like(q), cap=20.0)
    for name, leaf in zip(("dq", "dk", "dv"), leaves):
        check(name, leaf.grad, want[name])
    with torch.inference_mode():
        check("o", Fn.scored_attention(q, k, v, score_cap=20.0), want["o"])
    # gradients of some inputs only
    only = v.detach().requires_grad_(True)
    (dv,) = torch.autograd.grad(Fn.scored_attention(q, k, only, score_cap=20.0).sum(), only)
    check("dv", dv, want["dv"])
