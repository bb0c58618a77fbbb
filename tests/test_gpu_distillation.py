"""lm_head_distillation against 64 bits, both directions: sizes, absent and repeated entries,
temperatures, targets, chunks, streams and captures."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import _lib

pytestmark = pytest.mark.gpu

U32 = 2.0**-24
WEIGHT = 0.7


def make(rows, hidden, vocab, top, dtype, device, seed=0, targets=True):
    """A third of the rows have fewer entries, a tenth none; some ids repeat."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hidden, generator=g).to(dtype).to(device)
    w = (torch.randn(vocab, hidden, generator=g) * 3 / math.sqrt(hidden)).to(dtype).to(device)
    ids = torch.randint(0, vocab, (rows, top), generator=g)
    values = (torch.randn(rows, top, generator=g) * 4 + 10).float()
    drop = torch.rand(rows, top, generator=g) < (torch.rand(rows, 1, generator=g) < 0.33) * 0.5
    drop |= torch.rand(rows, 1, generator=g) < 0.1
    values[drop] = float("nan")  # absent entries hold anything
    ids[drop] = -1
    t = None
    if targets:
        t = torch.where(torch.rand(rows, generator=g) < 0.5, ids[:, 0].clamp_min(0), torch.randint(0, vocab, (rows,), generator=g))
        t[torch.rand(rows, generator=g) < 0.2] = -100
        t = t.to(device)
    up = torch.randn(rows, generator=g).to(device)
    return x, w, values.to(device), ids.to(device), t, up


def reference(x, w, values, ids, t, up, temperature=1.0, weight=WEIGHT):
    """(loss, dx, dw) in 64 bits with a bound for each (u = 2^-24).  A logit is off by e =
    (hidden + 8) u sum |x w|, and what is relative to the row's largest by 2 max e.  A sum of the
    vocabulary's exponentials adds at most vocab / 256 + 64 in a row; an exponential is off by
    2^-22 and by 4 u of its exponent; so are the teacher's, with 80 in a row.  Then first-order
    sums of these through the formulas, 2^-22 of every part, half a step of bf16 for the gradient
    of the logits (an operand of the products that follow) and of each type for the results."""
    f = torch.float64
    half = torch.finfo(x.dtype).eps / 2
    bf16 = x.dtype == torch.bfloat16
    xd, wd = x.to(f), w.to(f)
    s = xd @ wd.t()
    e = (x.shape[1] + 8) * U32 * (xd.abs() @ wd.abs().t())
    row_e = e.amax(1, keepdim=True)
    vocab = w.shape[0]
    add = (vocab / 256 + 64) * U32
    d = s - s.amax(1, keepdim=True)

    def softmax(k):
        lse = torch.logsumexp(d * k, 1, keepdim=True)
        q = torch.exp(d * k - lse)
        lse_off = 2 * row_e * k + add + 2.0**-21 + (q * d.abs()).sum(1, keepdim=True) * k * 4 * U32 + 2 * U32 * lse.abs()
        return q, lse, lse_off, (e + row_e) * k + lse_off + 4 * U32 * (d.abs() * k + lse.abs()) + 2.0**-21

    inv = 1 / temperature
    q, lse, lse_off, q_rel = softmax(inv)
    there = (ids >= 0) & (values != -math.inf)
    some = there.any(1, keepdim=True)
    v = torch.where(there, values.to(f), -1e300)
    dv = torch.where(there, v - v.amax(1, keepdim=True), 0.0)
    p = torch.where(there, torch.exp(dv * inv), 0.0)
    total = p.sum(1, keepdim=True).clamp_min(1e-300)
    p = p / total
    p_rel = 4 * U32 * dv.abs() * inv + 4 * U32 * (p * dv.abs()).sum(1, keepdim=True) * inv + 84 * U32 + 2.0**-20
    at = ids.clamp_min(0).long()
    diff = (dv - d.gather(1, at)) * inv
    lt = torch.log(total)
    square = temperature**2
    loss = square * ((p * diff).sum(1, keepdim=True) + lse - lt) * some
    part = (p * (p_rel + 80 * U32) * diff.abs() + p * (e.gather(1, at) + row_e + 6 * U32 * (dv.abs() + d.gather(1, at).abs())) * inv)
    bound = square * some * (part.sum(1, keepdim=True) + lse_off + 84 * U32 + 2.0**-20 + 4 * U32 * (lse.abs() + lt.abs()))
    bound = bound + 8 * U32 * square * some * ((p * diff).abs().sum(1, keepdim=True) + lse.abs() + lt.abs())
    upd = up.to(f)[:, None]
    ga = torch.where(some, upd * temperature, 0.0)
    p_all = torch.zeros_like(q).scatter_add_(1, at, p)
    p_off = torch.zeros_like(q).scatter_add_(1, at, p * p_rel) + 1024 * U32 * p_all
    g = ga * (q - p_all)
    g_off = ga.abs() * (q * q_rel + p_off + 2.0**-22 * (q + p_all))
    if t is not None:
        q1, lse1, lse1_off, q1_rel = softmax(1.0)
        used = (t != -100)[:, None]
        y = t.clamp_min(0)[:, None]
        ce = lse1 - d.gather(1, y)
        loss = loss + weight * ce * used
        bound = bound + weight * used * (lse1_off + e.gather(1, y) + row_e + 8 * U32 * (lse1.abs() + d.gather(1, y).abs() + ce.abs()))
        gb = torch.where(used, upd * weight, 0.0)
        hot = torch.zeros_like(q).scatter_(1, y, 1.0)
        g = g + gb * (q1 - hot)
        g_off = g_off + gb.abs() * (q1 * q1_rel + 2.0**-22 * (q1 + hot))
    bound = bound + 8 * U32 * loss.abs()
    g_off = g_off + bf16 * half * g.abs()
    n = lambda k: (k + 8) * U32  # noqa: E731
    dx, dw = g @ wd, g.t() @ xd
    dx_bound = (g_off + n(vocab) * g.abs()) @ wd.abs() + half * dx.abs()
    dw_bound = (g_off + n(x.shape[0]) * g.abs()).t() @ xd.abs() + half * dw.abs()
    return (loss[:, 0], bound[:, 0]), (dx, dx_bound), (dw, dw_bound)


def run(x, w, values, ids, t, up, weight=WEIGHT, **kw):
    x, w = x.detach().requires_grad_(True), w.detach().requires_grad_(True)
    loss = Fn.lm_head_distillation(x, w, values, ids, t, reduction="none", target_weight=weight, **kw)
    return (loss.detach(), *torch.autograd.grad(loss, (x, w), up))


def check(got, want):
    for name, a, (value, bound) in zip(("loss", "dx", "dw"), got, want):
        off = (a.double() - value).abs()
        assert (off <= bound * 1.01 + 1e-37).all(), (name, float((off - bound).max()), float(off.max()))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,hidden,vocab,top", [
    (1, 64, 8, 1), (1, 8, 1, 3), (3, 8, 17, 2), (63, 72, 1001, 5), (64, 256, 320, 16), (65, 64, 257, 31),
    (129, 128, 1000, 32), (200, 200, 515, 33), (257, 64, 777, 64), (513, 136, 300, 65), (20, 64, 4000, 1024),
    (300, 1024, 50257, 50),
])
@pytest.mark.parametrize("temperature,targets", [(1.0, False), (1.0, True), (2.0, False), (4.0, True), (0.5, True)])
def test_distillation(device, rows, hidden, vocab, top, temperature, targets, dtype) -> None:
    args = make(rows, hidden, vocab, top, dtype, device, targets=targets)
    got = run(*args, temperature=temperature)
    check(got, reference(*args, temperature=temperature))
    again = run(*args, temperature=temperature)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    with torch.no_grad():  # without gradients: the same bits
        loss = Fn.lm_head_distillation(*args[:5], reduction="none", target_weight=WEIGHT, temperature=temperature)
    assert torch.equal(loss, got[0])


@pytest.mark.parametrize("rows,hidden,vocab,top", [
    (65, 72, 66001, 20),  # few rows, a long table
    (257, 64, 16001, 20), (200, 136, 33001, 20), (1025, 64, 33001, 20),
    (4100, 8, 33001, 20),  # a gradient larger than the last-level cache
])
@pytest.mark.parametrize("temperature", [1.0, 3.0])
def test_every_tile_size(device, rows, hidden, vocab, top, temperature) -> None:
    args = make(rows, hidden, vocab, top, torch.bfloat16, device)
    check(run(*args, temperature=temperature), reference(*args, temperature=temperature))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("temperature", [0.01, 0.1, 30.0, 100.0])
def test_extreme_temperatures(device, temperature, dtype) -> None:
    args = make(70, 64, 300, 20, dtype, device)
    check(run(*args, temperature=temperature), reference(*args, temperature=temperature))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_large_logits(device, dtype) -> None:
    """Logits of hundreds on both sides: nothing overflows, the loss is a difference."""
    x, w, values, ids, t, up = make(70, 64, 300, 20, dtype, device)
    args = (x, w * 100, values * 60 - 500, ids, t, up)
    check(run(*args), reference(*args))
    # all of one row far below zero, and all far above
    x = torch.where(torch.arange(70, device=device)[:, None] % 2 == 0, 8.0, -8.0).to(dtype).expand(70, 64).contiguous()
    for sign in (1, -1):
        args = (x, (w.float() * 0.1 + sign).to(dtype), values, ids, t, up)
        check(run(*args, temperature=0.5), reference(*args, temperature=0.5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_absent_entries(device, dtype) -> None:
    """Absent by id or by a logit of minus infinity, whatever the other holds; the type's
    lowest value is a logit like another; rows without any have no first term."""
    x, w, values, ids, t, up = make(60, 64, 300, 12, dtype, device)
    ids, values = ids.clamp_min(0), values.nan_to_num(3.0)
    lowest = torch.finfo(values.dtype).min
    mask = torch.rand(60, 12, generator=torch.Generator().manual_seed(8)).to(device) < 0.4
    mask[:5] = True
    by_id = run(x, w, torch.where(mask, float("inf"), values), torch.where(mask, -7, ids), t, up, temperature=2.0)
    by_value = run(x, w, torch.where(mask, -math.inf, values), ids, t, up, temperature=2.0)
    assert all(torch.equal(a, b) for a, b in zip(by_id, by_value))
    lost = torch.where(mask, lowest, values)
    lost[:5] = values[:5]
    low = run(x, w, lost, ids, t, up, temperature=2.0)
    # beside present ones its probability is 0: the same but in the rows that had nothing else
    assert torch.equal(low[0][5:], by_id[0][5:])
    alone = run(x, w, torch.full_like(values, lowest), ids, t, up)  # all the same: each 1 / 12
    check(alone, reference(x, w, torch.zeros_like(values), ids, t, up))
    nothing = run(x, w, values, torch.full_like(ids, -1), None, up)
    assert not any(a.any() for a in nothing)
    # nor a gradient, whatever comes down to such rows and lies in them
    x2, up2 = x.clone(), up.clone()
    x2[2], up2[2] = float("nan"), float("inf")
    ids2 = ids.clone()
    ids2[2] = -1
    t2 = t.clone()
    t2[2] = -100
    got = run(x2, w, values, ids2, t2, up2)
    assert got[0][2] == 0 and not got[1][2].any()
    assert got[0].isfinite().all() and got[1].isfinite().all()
    clean = run(x, w, values, ids2, t2, up)  # its zero gradient meets no NaN in the table's either
    assert torch.equal(got[2], clean[2])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_repeated_ids(device, dtype) -> None:
    """One token in every entry, and the target too: its probabilities add up to 1."""
    x, w, values, ids, t, up = make(40, 64, 300, 70, dtype, device)
    values = values.nan_to_num(3.0)
    same = torch.full_like(ids, 5)
    for target in (None, torch.full((40,), 5, device=device), torch.full((40,), 6, device=device)):
        check(run(x, w, values, same, target, up), reference(x, w, values, same, target, up))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_types_and_strides(device, dtype) -> None:
    """ids and targets of 4 and 8 bytes, bf16 logits, columns of wider tensors, one teacher row
    for all, more dimensions, a table at an odd start: the same bits."""
    x, w, values, ids, t, up = make(60, 64, 300, 9, dtype, device)
    values = values.bfloat16().float()
    want = run(x, w, values, ids, t, up, temperature=2.0)

    def same(*args, **kw):
        got = run(*args, temperature=2.0, **kw)
        return all(torch.equal(a.reshape(b.shape), b) for a, b in zip(got, want))

    assert same(x, w, values.bfloat16(), ids.int(), t.int(), up)
    wide_v = torch.full((60, 20), float("nan"), device=device)
    wide_i = torch.full((60, 31), 10**6, dtype=torch.int32, device=device)
    wide_v[:, 3:12], wide_i[:, 7:16] = values, ids
    assert same(x, w, wide_v[:, 3:12], wide_i[:, 7:16], t, up)
    assert same(x, w, values.t().contiguous().t(), ids.t().contiguous().t(), t, up)
    assert same(x.view(3, 20, 64), w, values.view(3, 20, 9), ids.view(3, 20, 9), t.view(3, 20), up.view(3, 20))
    odd = torch.empty(60 * 64 + 1, dtype=dtype, device=device)[1:].view(60, 64).copy_(x)
    table = torch.empty(300 * 64 + 1, dtype=dtype, device=device)[1:].view(300, 64).copy_(w)
    assert same(odd, table, values, ids, t, up)
    assert same(x.t().contiguous().t(), w.t().contiguous().t(), values, ids, t, up)
    one = run(x, w, values[:1].expand(60, 9), ids[3:4].expand(60, 9), t, up)
    dense = run(x, w, values[:1].expand(60, 9).contiguous(), ids[3:4].expand(60, 9).contiguous(), t, up)
    assert all(torch.equal(a, b) for a, b in zip(one, dense))


@pytest.mark.parametrize("rows,hidden,vocab,chunk,product", [
    (1024, 768, 32000, None, (1, 1, 32000, 768, 1024)),  # the table's gradient in two calls,
    (1100, 768, 31997, 1024, (1, 1, 32000, 768, 1024)),  # added up over chunks,
    (3000, 2048, 31999, None, (0, 1, 3000, 2048, 31999)),  # the hidden states' in two
])
def test_gradients_in_two_calls(device, rows, hidden, vocab, chunk, product) -> None:
    first = ctypes.c_int64()
    _lib.call("nmb_gemm_bf16_first_rows", *product, ctypes.byref(first))
    assert 0 < first.value < product[2]
    args = make(rows, hidden, vocab, 7, torch.bfloat16, device)
    got = run(*args, temperature=2.0, chunk=chunk)
    check(got, reference(*args, temperature=2.0))
    again = run(*args, temperature=2.0, chunk=chunk)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_chunks_and_reductions(device, dtype) -> None:
    args = make(300, 64, 500, 7, dtype, device)
    check(run(*args, temperature=2.0, chunk=128), reference(*args, temperature=2.0))
    x, w, values, ids, t, up = args
    none = Fn.lm_head_distillation(x, w, values, ids, t, reduction="none")
    total = Fn.lm_head_distillation(x, w, values, ids, t, reduction="sum")
    mean = Fn.lm_head_distillation(x, w, values, ids, t)
    counted = ((ids >= 0).any(1) | (t != -100)).sum()
    # sums of 300 fp32 terms, in any order
    assert (total - none.sum()).abs() <= 300 * U32 * none.abs().sum()
    assert (mean - none.sum() / counted).abs() <= 302 * U32 * none.abs().sum() / counted
    only = Fn.lm_head_distillation(x, w, values, ids)
    alone = Fn.lm_head_distillation(x, w, values, ids, reduction="none")
    assert (only - alone.sum() / (ids >= 0).any(1).sum()).abs() <= 302 * U32 * alone.abs().sum()
    nothing = Fn.lm_head_distillation(x, w, values, torch.full_like(ids, -1))
    assert nothing == 0
    leaves = [x[:0].detach().requires_grad_(True), w.detach().requires_grad_(True)]
    empty = Fn.lm_head_distillation(*leaves, values[:0], ids[:0], t[:0], reduction="sum")
    dx, dw = torch.autograd.grad(empty, leaves)
    assert empty == 0 and dx.shape == (0, 64) and not dw.any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_agrees_with_the_cross_entropy(device, dtype) -> None:
    """One teacher entry is a target: the first term is the cross entropy, bits aside."""
    x, w, _, _, t, up = make(90, 64, 300, 1, dtype, device)
    values = torch.full((90, 1), 4.0, device=device)
    got = run(x, w, values, torch.where(t == -100, -1, t)[:, None], None, up)
    check(got, reference(x, w, values, torch.where(t == -100, -1, t)[:, None], None, up))
    leaves = [a.detach().requires_grad_(True) for a in (x, w)]
    ce = Fn.lm_head_cross_entropy(*leaves, t, reduction="none", z_loss=1e-30)  # (its unrounded form)
    # (both within the bounds of one formula)
    want = reference(x, w, values, torch.where(t == -100, -1, t)[:, None], None, up)
    assert ((got[0] - ce.detach()).double().abs() <= 2.02 * want[0][1] + 1e-30).all()


def test_differences(device) -> None:
    """The gradient along a direction against the central difference of the formula in 64 bits,
    whose own error at steps of 1e-5 is below 1e-8 of the parts."""
    x, w, values, ids, t, up = make(20, 32, 50, 6, torch.float32, device)
    got = run(x, w, values, ids, t, up, temperature=2.0)
    want = reference(x, w, values, ids, t, up, temperature=2.0)
    g = torch.Generator().manual_seed(3)
    along = [torch.randn(a.shape, generator=g).to(device).double() for a in (x, w)]

    def value(h):
        at = [a.double() + h * v for a, v in zip((x, w), along)]
        return (reference(*at, values, ids, t, up, temperature=2.0)[0][0] * up.double()).sum()

    difference = (value(1e-5) - value(-1e-5)) / 2e-5
    slope = sum((a.double() * v).sum() for a, v in zip(got[1:], along))
    bound = sum((b[1] * v.abs()).sum() for b, v in zip(want[1:], along))
    size = sum((b[0] * v).abs().sum() for b, v in zip(want[1:], along))
    assert (slope - difference).abs() <= 1.01 * bound + 1e-8 * size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_some_gradients_and_the_tie(device, dtype) -> None:
    x, w, values, ids, t, up = make(70, 64, 300, 8, dtype, device)
    want = run(x, w, values, ids, t, up)
    for n in range(2):
        leaves = [x, w]
        leaves[n] = leaves[n].detach().requires_grad_(True)
        loss = Fn.lm_head_distillation(*leaves, values, ids, t, reduction="none", target_weight=WEIGHT)
        assert torch.equal(torch.autograd.grad(loss, leaves[n], up)[0], want[1 + n])
    # tied with the embedding, whose backward adds its own
    tokens = torch.randint(0, 300, (70,), generator=torch.Generator().manual_seed(1)).to(device)
    table = w.detach().requires_grad_(True)
    tie = Fn.TiedGrad()
    hidden = Fn.embedding(table, tokens, tie)
    loss = Fn.lm_head_distillation(hidden, table, values, ids, t, reduction="none", tie=tie, target_weight=WEIGHT)
    tied, = torch.autograd.grad(loss, table, up)
    apart = run(hidden.detach(), w, values, ids, t, up)
    rows = w.detach().requires_grad_(True)
    through, = torch.autograd.grad(Fn.embedding(rows, tokens), rows, apart[1])
    # two roundings of the sum's parts and one of the sum
    half = torch.finfo(dtype).eps / 2
    off = (tied.double() - through.double() - apart[2].double()).abs()
    assert (off <= 3.01 * half * (through.double().abs() + apart[2].double().abs())).all()


def test_refusals_on_the_device(device) -> None:
    x, w, values, ids, t, up = make(10, 64, 300, 4, torch.bfloat16, device)
    bad = ids.clone()
    bad[3, 1] = 300
    with pytest.raises(ValueError, match="teacher_ids"):
        Fn.lm_head_distillation(x, w, values, bad, t)
    far = t.clone()
    far[2] = 300
    with pytest.raises(ValueError, match="targets"):
        Fn.lm_head_distillation(x, w, values, ids, far)
    with pytest.raises(ValueError, match="targets"):
        Fn.lm_head_distillation(x, w, values, ids, far, validate=Fn.TargetCheck(far, 300))
    with pytest.raises(ValueError, match="one device"):
        Fn.lm_head_distillation(x, w, values.cpu(), ids, t)
    with pytest.raises(ValueError, match="multiple of 8"):
        Fn.lm_head_distillation(x[:, :60], w[:, :60], values, ids, t)
    # gradients past what their products address: before the loss, and only where they are wanted
    long_table = torch.zeros(1 << 22, 8, dtype=torch.bfloat16, device=device)
    few = x[:, :8].detach().contiguous().requires_grad_(True)
    with pytest.raises(ValueError, match="below 2\\^22"):
        Fn.lm_head_distillation(few, long_table, values, ids, t)
    assert Fn.lm_head_distillation(few.detach(), long_table, values, ids, t).isfinite()


def test_graphs_are_freed(device) -> None:
    x, w, values, ids, t, up = make(100, 64, 300, 4, torch.bfloat16, device)
    run(x, w, values, ids, t, up)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(3):
        table = w.detach().requires_grad_(True)
        tie = Fn.TiedGrad()
        hidden = Fn.embedding(table, torch.zeros(100, dtype=torch.int64, device=device), tie)
        loss = Fn.lm_head_distillation(hidden, table, values, ids, t, tie=tie, validate=False)
        del loss, hidden, tie, table  # never differentiated
        run(x, w, values, ids, t, up)
    assert torch.cuda.memory_allocated() == before


def test_no_second_derivative(device) -> None:
    x, w, values, ids, t, up = make(10, 64, 300, 4, torch.float32, device)
    x = x.detach().requires_grad_(True)
    loss = Fn.lm_head_distillation(x, w, values, ids, t, reduction="none")
    first, = torch.autograd.grad(loss.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_unchecked_ids_poison_their_rows(device, dtype) -> None:
    """Ids and targets far past the vocabulary, and logits that are not numbers: their rows'
    losses and gradients are NaN, no others'."""
    x, w, values, ids, t, up = make(40, 64, 300, 6, dtype, device)
    ids, values, t = ids.clamp_min(0), values.nan_to_num(3.0), t.clamp_min(0)
    want = run(x, w, values, ids, t, up, validate=False)
    bad_ids, bad_values, bad_t = ids.clone(), values.clone(), t.clone()
    bad_ids[3, 2] = 300
    bad_ids[4, 0] = 1 << 40
    bad_values[5, 1], bad_values[6, 5] = float("nan"), float("inf")
    bad_t[7], bad_t[8] = 1 << 40, -5
    got = run(x, w, bad_values, bad_ids, bad_t, up, validate=False)
    rows = torch.zeros(40, dtype=torch.bool, device=device)
    rows[3:9] = True
    assert got[0][rows].isnan().all() and torch.equal(got[0][~rows], want[0][~rows])
    assert got[1][3:7].isnan().all() and torch.equal(got[1][~rows], want[1][~rows])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_captured_and_replayed(device, dtype) -> None:
    """Two graphs of one step, replayed in turn on new values between eager steps."""
    def step(args):
        return run(*args, temperature=2.0, validate=False)

    graphs = []
    for _ in range(2):
        fixed = [a.clone() for a in make(300, 64, 700, 9, dtype, device)]
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step(fixed)
        torch.cuda.current_stream().wait_stream(stream)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step(fixed)
        graphs.append((graph, fixed, out))
    for turn in range(4):
        for n, (graph, fixed, out) in enumerate(graphs):
            new = make(300, 64, 700, 9, dtype, device, seed=10 * turn + n)
            for a, b in zip(fixed, new):
                a.copy_(b)
            want = step(new)
            graph.replay()
            step(make(300, 64, 700, 9, dtype, device, seed=99))  # eager work behind the replay
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want)), (turn, n)


@pytest.mark.parametrize("rows", [1, 1023, 8192, 8193, 70001, 2_100_001])
@pytest.mark.parametrize("targets", [False, True])
def test_means_of_many_rows(device, rows, targets) -> None:
    """Sums are formed in 64 bits and rounded once, a mean after its division: half a step of
    fp32, and 64-bit sums' own errors."""
    x, w, values, ids, t, _ = make(rows, 16, 64, 3, torch.bfloat16, device, targets=targets)
    none = Fn.lm_head_distillation(x, w, values, ids, t, reduction="none").double()
    counted = (ids >= 0).any(1)
    if targets:
        counted |= t != -100
    count = max(int(counted.sum()), 1)
    for reduction, over in (("sum", 1), ("mean", count)):
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        total = Fn.lm_head_distillation(*leaves, values, ids, t, reduction=reduction)
        assert total.shape == () and total.dtype == torch.float32
        want = none.sum() / over
        assert (total.double() - want).abs() <= U32 * want.abs() + rows * 2.0**-52 * none.abs().sum() / over
        got = torch.autograd.grad(total * 3, leaves)
        leaves = [x.clone().requires_grad_(True), w.clone().requires_grad_(True)]
        # (one division of two fp32 numbers: by a Python number it is a product with a reciprocal)
        up = torch.full((rows,), 3.0, device=device) / torch.tensor(float(over), device=device)
        loss = Fn.lm_head_distillation(*leaves, values, ids, t, reduction="none")
        assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(loss, leaves, up)))


def test_captured_means(device) -> None:
    """The mean of enough rows that a library's sum would take several workgroups, captured and
    replayed between eager steps."""
    def step(args):
        leaves = [args[0].detach().requires_grad_(True), args[1].detach().requires_grad_(True)]
        loss = Fn.lm_head_distillation(*leaves, *args[2:5], validate=False)
        return (loss, *torch.autograd.grad(loss, leaves))

    fixed = [a.clone() for a in make(70001, 16, 64, 3, torch.bfloat16, device)]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(fixed)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(fixed)
    for turn in range(4):
        new = make(70001, 16, 64, 3, torch.bfloat16, device, seed=turn + 1)
        for a, b in zip(fixed, new):
            a.copy_(b)
        want = step(new)
        graph.replay()
        step(make(70001, 16, 64, 3, torch.bfloat16, device, seed=99))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), turn


def test_losses_may_be_written_to(device) -> None:
    x, w, values, ids, t, _ = make(40, 64, 100, 5, torch.bfloat16, device)
    x.requires_grad_(True)
    for reduction in ("none", "sum", "mean"):
        loss = Fn.lm_head_distillation(x, w, values, ids, t, reduction=reduction)
        want, = torch.autograd.grad(loss.sum(), x, retain_graph=True)
        loss.mul_(2)
        got, = torch.autograd.grad(loss.sum(), x)
        assert torch.equal(got, 2 * want)


def test_two_streams(device) -> None:
    states = [make(400, 64, 2000, 20, torch.bfloat16, device, seed=n) for n in range(2)]
    want = [run(*st, validate=False) for st in states]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for n, (stream, st) in enumerate(zip(streams, states)):
            with torch.cuda.stream(stream):
                got[n].append(run(*st, validate=False))
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        assert all(torch.equal(a, b) for r in runs for a, b in zip(r, w))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_checkpointed_and_offloaded(device, dtype) -> None:
    x, w, values, ids, t, up = make(70, 64, 300, 8, dtype, device)
    want = run(x, w, values, ids, t, up)

    def head(x, w):
        return Fn.lm_head_distillation(x, w, values, ids, t, reduction="none", target_weight=WEIGHT, validate=False)

    def gradients(f):
        leaves = [a.detach().requires_grad_(True) for a in (x, w)]
        loss = f(*leaves)
        return loss.detach(), *torch.autograd.grad(loss, leaves, up)

    def offloaded(*args):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().cpu().contiguous() if t.ndim == 2 else t.cpu(),
                                                      lambda t: t.cuda().t() if t.ndim == 2 else t.cuda()):
            return head(*args)

    for got in (gradients(lambda *a: torch.utils.checkpoint.checkpoint(head, *a, use_reentrant=False)),
                gradients(offloaded)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))
