"""rotary_positions against 64 bits, both directions: layouts, parts of the head, positions,
strides, partial gradients, streams and captures."""

from __future__ import annotations

import math

import pytest
import torch

import nano_megatron_amd as nmb
import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu

U32 = 2.0**-24


def make(b, s, h, kv, d, dtype, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randn(b, s, n, d, generator=g).to(dtype).to(device).transpose(1, 2) for n in (h, kv, h, kv)]


def reference(x, frequencies, pos, interleaved=False, magnitude=1.0, sign=1.0):
    """(value, bound) in 64 bits, pairs as complex numbers.  An angle is off by 2^-51 of its
    size and 1.5e-9, sine and cosine by 2e-9 and 3 u (u = 2^-24), their product with the
    magnitude by u, the two products and the sum by u each, the result by half a step."""
    r = 2 * len(frequencies)
    j = torch.arange(r // 2, device=x.device)
    first, second = (2 * j, 2 * j + 1) if interleaved else (j, j + r // 2)
    angle = (pos.double()[..., None] * frequencies)[:, None]
    z = torch.complex(x[..., first].double(), x[..., second].double())
    turned = z * torch.polar(torch.full_like(angle, magnitude), sign * angle)
    out = x.double().clone()
    out[..., first], out[..., second] = turned.real, turned.imag
    size = (z.real.abs() + z.imag.abs()) * abs(magnitude)
    off = size * (2.0**-51 * angle.abs() + 4e-9 + 8 * U32)
    bound = torch.zeros_like(out)
    bound[..., first] = bound[..., second] = off
    bound += torch.finfo(x.dtype).eps / 2 * out.abs() * (bound > 0)
    return out, bound


def check(got, want):
    value, bound = want
    off = (got.double() - value).abs()
    assert (off <= bound * 1.01).all(), (float((off - bound).max()), float(off.max()))


def places(b, s, device, offset=0):
    return torch.arange(offset, offset + s, device=device)[None].expand(b, s)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,s,h,kv,d,r", [
    (1, 1, 1, 1, 2, 2), (2, 3, 4, 2, 64, 64), (1, 1, 32, 8, 128, 128), (32, 1, 32, 8, 128, 64), (2, 5, 3, 1, 80, 32),
    (1, 7, 5, 5, 96, 96), (2, 33, 2, 1, 65, 64), (1, 9, 3, 2, 66, 64), (1, 5, 2, 1, 128, 126), (3, 4, 2, 2, 48, 2),
    (1, 6, 2, 1, 40, 18), (1, 3, 7, 3, 256, 256), (2, 2, 1, 1, 1024, 1000), (1, 2, 2, 1, 2051, 2048), (2, 2, 3, 1, 30, 30),
    (1, 4, 2, 1, 33, 20), (1, 4, 17, 2, 70, 14), (1, 5, 3, 1, 40, 6), (2, 3, 2, 2, 16, 4), (1, 3, 2, 1, 9, 8), (2, 200, 16, 16, 64, 64), (1, 600, 32, 8, 128, 96),
    (4, 2100, 3, 2, 80, 40),
])
def test_rotary(device, b, s, h, kv, d, r, interleaved, dtype) -> None:
    q, k, gq, gk = make(b, s, h, kv, d, dtype, device)
    f = Fn.rotary_frequencies(r, device=device)
    kw = dict(sequence_offset=5, interleaved=interleaved, magnitude=1.25)
    leaves = [t.detach().requires_grad_(True) for t in (q, k)]
    out = Fn.rotary_positions(*leaves, f, **kw)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    pos = places(b, s, device, 5)
    for t, o in zip((q, k), out):
        check(o.detach(), reference(t, f, pos, interleaved, 1.25))
        assert torch.equal(o[..., r:], t[..., r:])
    for t, o in zip((gq, gk), grads):
        check(o, reference(t, f, pos, interleaved, 1.25, -1.0))
        assert torch.equal(o[..., r:], t[..., r:])
    plain = Fn.rotary_positions(q, k, f, **kw)  # without gradients, and queries alone: the same bits
    assert all(torch.equal(a, o) for a, o in zip(plain, out))
    assert torch.equal(Fn.rotary_positions(q, None, f, **kw), out[0])
    assert out[0].transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_positions(device, dtype) -> None:
    """Offsets per row, positions per token or per row and token, of both types and any
    strides; far, negative and equal ones."""
    b, s, d = 3, 40, 64
    q, k, *_ = make(b, s, 4, 2, d, dtype, device)
    f = Fn.rotary_frequencies(d, device=device)
    g = torch.Generator().manual_seed(4)
    start = torch.tensor([0, 131_071, 999_999], dtype=torch.int32, device=device)
    any_order = torch.randint(-3_000_000, 3_000_000, (b, s), generator=g).to(device)
    far = torch.randint(-(1 << 40), 1 << 40, (s,), generator=g).to(device)
    cases = [
        (dict(sequence_offset=start), start[:, None] + torch.arange(s, device=device)),
        (dict(sequence_offset=-7), places(b, s, device, -7)),
        (dict(sequence_offset=(1 << 40) - 100), places(b, s, device, (1 << 40) - 100)),
        (dict(positions=any_order), any_order),
        (dict(positions=any_order.to(torch.int32)), any_order),
        (dict(positions=any_order.t().contiguous().t()), any_order),
        (dict(positions=any_order[:1].expand(b, s)), any_order[:1].expand(b, s)),
        (dict(positions=any_order[0]), any_order[:1].expand(b, s)),
        (dict(positions=torch.stack((any_order, any_order), 2).to(torch.int32)[..., 0]), any_order),
        (dict(positions=far), far[None].expand(b, s)),
        (dict(positions=torch.full((s,), 11, device=device)), torch.full((b, s), 11, device=device)),
    ]
    for kw, pos in cases:
        for t, o in zip((q, k), Fn.rotary_positions(q, k, f, **kw)):
            check(o, reference(t, f, pos))


@pytest.mark.parametrize("scaling", [None, "linear", "base", "parts"])
def test_scaled(device, scaling) -> None:
    q, k, *_ = make(2, 300, 4, 2, 128, torch.float32, device)
    f = Fn.rotary_frequencies(64, 5e5, scaling=scaling, factor=8.0, original_length=2048, device=device)
    pos = places(2, 300, device, 100_000)
    for t, o in zip((q, k), Fn.rotary_positions(q, k, f, sequence_offset=100_000)):
        check(o, reference(t, f, pos))


def test_every_eighth_of_a_turn(device) -> None:
    """Sine and cosine at and around every multiple of an eighth of a turn: pairs (1, 0)."""
    eighths = torch.arange(-16, 17, dtype=torch.float64) * (math.pi / 4)
    off = torch.tensor([0.0, 1e-12, -1e-12, 1e-9, -1e-9, 1e-4, -1e-4, 0.3], dtype=torch.float64)
    f = (eighths[:, None] + off).reshape(-1).to(device)
    x = torch.zeros(1, 1, 2, 2 * len(f), device=device)
    x[..., 0::2] = 1
    out = Fn.rotary_positions(x, None, f, interleaved=True, positions=torch.ones(2, dtype=torch.int64, device=device))
    assert (out[..., 0::2].double() - torch.cos(f)).abs().max() <= 4e-9 + 4 * U32
    assert (out[..., 1::2].double() - torch.sin(f)).abs().max() <= 4e-9 + 4 * U32


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
def test_strides(device, interleaved, dtype) -> None:
    """Slices of one projection, heads-first memory, odd strides and starts, one head for
    all, a head_dim that is not contiguous; gradients likewise."""
    b, s, h, kv, d, r = 2, 19, 6, 2, 72, 50
    q, k, gq, gk = make(b, s, h, kv, d, dtype, device)
    f = Fn.rotary_frequencies(r, device=device)

    def run(q, k, gq, gk):
        leaves = [t.detach().requires_grad_(True) for t in (q, k)]
        out = Fn.rotary_positions(*leaves, f, interleaved=interleaved)
        return [t.detach() for t in (*out, *torch.autograd.grad(out, leaves, (gq, gk)))]

    want = run(q, k, gq, gk)
    nan = float("nan")

    def odd(t):  # rows of d + 3 elements that start at the second
        wide = torch.full((*t.shape[:3], d + 3), nan, dtype=dtype, device=device)
        wide[..., 1:d + 1] = t
        return wide[..., 1:d + 1]

    both = torch.cat((q, k, k), 1).transpose(1, 2).contiguous().transpose(1, 2)
    grads = torch.cat((gq, gk), 1).transpose(1, 2).contiguous().transpose(1, 2)
    layouts = [
        (*both.split((h, kv, kv), 1)[:2], gq, gk),
        (q.contiguous(), k.contiguous(), gq.contiguous(), gk.contiguous()),
        (odd(q), odd(k), odd(gq), odd(gk)),
        (q.transpose(2, 3).contiguous().transpose(2, 3), k, gq, gk.transpose(2, 3).contiguous().transpose(2, 3)),
        (q, k, *grads.split((h, kv), 1)),
    ]
    for layout in layouts:
        assert all(torch.equal(a, w) for a, w in zip(run(*layout), want))
    one = [t[:, :1].expand(-1, n, -1, -1) for t, n in ((q, h), (k, kv), (gq, h), (gk, kv))]
    assert all(torch.equal(a, w) for a, w in zip(run(*one), run(*(t.contiguous() for t in one))))


def test_some_gradients(device) -> None:
    q, k, gq, gk = make(2, 30, 4, 2, 64, torch.float32, device)
    f = Fn.rotary_frequencies(64, device=device)
    pos = places(2, 30, device)
    for which, (x, gx) in enumerate(((q, gq), (k, gk))):
        leaf = x.detach().requires_grad_(True)
        out = Fn.rotary_positions(*((leaf, k) if which == 0 else (q, leaf)), f)
        grad, = torch.autograd.grad(out[which], leaf, gx)
        check(grad, reference(gx, f, pos, sign=-1.0))
    leaves = [t.detach().requires_grad_(True) for t in (q, k)]
    out = Fn.rotary_positions(*leaves, f)
    only_k = torch.autograd.grad(out[1], leaves, gk, allow_unused=True)
    assert only_k[0] is None or not only_k[0].any()
    check(only_k[1], reference(gk, f, pos, sign=-1.0))
    out = Fn.rotary_positions(*leaves, f)
    ones = torch.autograd.grad(out[0].sum() + out[1].sum(), leaves)  # broadcast gradients
    for t, o in zip((q, k), ones):
        check(o, reference(torch.ones_like(t), f, pos, sign=-1.0))
    x = q.detach().requires_grad_(True)  # one tensor as both
    out = Fn.rotary_positions(x, x, f)
    twice, = torch.autograd.grad(out, x, (gq, gq))
    assert torch.equal(twice, 2 * torch.autograd.grad(Fn.rotary_positions(x, None, f), x, gq)[0])


def test_differences(device) -> None:
    """The gradient along a direction against the difference of the map in 64 bits (it is
    linear: no error but rounding)."""
    q, _, gq, _ = make(2, 50, 3, 1, 40, torch.float32, device)
    f = Fn.rotary_frequencies(36, device=device)
    pos = places(2, 50, device)
    along = torch.randn(q.shape, generator=torch.Generator().manual_seed(2)).to(device).double()

    def value(x):
        return (reference(x, f, pos)[0] * gq.double()).sum()

    leaf = q.detach().requires_grad_(True)
    grad, = torch.autograd.grad(Fn.rotary_positions(leaf, None, f), leaf, gq)
    difference = (value(q.double() + along) - value(q.double() - along)) / 2
    bound = (reference(gq, f, pos, sign=-1.0)[1] * along.abs()).sum()
    assert ((grad.double() * along).sum() - difference).abs() <= bound


def test_copied_elements_keep_their_bits(device) -> None:
    """NaN of any payload, infinities and the type's lowest value behind the rotated part."""
    bits = torch.arange(-(1 << 15), 1 << 15, dtype=torch.int32).to(torch.int16).view(1, 1, 512, 128).to(device)
    x = bits.view(torch.bfloat16).clone()
    x[..., :64] = 1.0
    out = Fn.rotary_positions(x, None, Fn.rotary_frequencies(64, device=device))
    assert torch.equal(out[..., 64:].view(torch.int16), x[..., 64:].view(torch.int16))
    assert out[..., :64].isfinite().all()


def test_frequencies_that_are_not_numbers(device) -> None:
    """They make their own pair NaN and no other."""
    q, *_ = make(1, 5, 2, 1, 64, torch.float32, device)
    f = Fn.rotary_frequencies(64, device=device)
    want = Fn.rotary_positions(q, None, f, sequence_offset=1)
    for bad in (float("nan"), float("inf")):
        g = f.clone()
        g[7] = bad
        got = Fn.rotary_positions(q, None, g, sequence_offset=1)
        pair = torch.zeros(64, dtype=torch.bool, device=device)
        pair[7] = pair[39] = True
        assert got[..., pair].isnan().all() and torch.equal(got[..., ~pair], want[..., ~pair])


def test_empty(device) -> None:
    f = Fn.rotary_frequencies(64, device=device)
    for shape in ((0, 4, 3, 64), (2, 4, 0, 64), (2, 0, 3, 64)):
        q = torch.zeros(shape, device=device, requires_grad=True)
        out = Fn.rotary_positions(q, q, f)
        assert out[0].shape == shape
        assert torch.autograd.grad(out, q, out)[0].shape == shape


def test_past_32_bit_offsets(device) -> None:
    """70,000 tokens of 32,768 elements (2.3e9), read from one token's memory."""
    x = torch.randn(1, 256, 1, 128, generator=torch.Generator().manual_seed(1)).bfloat16().to(device)
    f = Fn.rotary_frequencies(128, device=device)
    y = Fn.rotary_positions(x.expand(1, 256, 70_000, 128), None, f)
    for at in (0, 65_535, 65_536, 69_999):
        assert torch.equal(y[:, :, at:at + 1], Fn.rotary_positions(x, None, f, sequence_offset=at)), at


def test_agrees_with_the_table_form(device) -> None:
    """The half layout over the whole head is apply_rotary_pos_emb, whose fp32 angle of
    position p is off by p 2^-24 and whose three roundings and rounded tables add 2^-8 each."""
    q, k, *_ = make(2, 64, 4, 2, 64, torch.bfloat16, device)
    pos = torch.arange(64, device=device)
    cos, sin = nmb.RotaryEmbedding(64)(pos, dtype=torch.bfloat16)
    old = nmb.apply_rotary_pos_emb(q, k, cos, sin)
    new = nmb.RotaryPositions(64)(q, k)
    for a, b, x in zip(old, new, (q, k)):
        assert ((a.float() - b.float()).abs() <= 6 * 2.0**-8 * 2 * x.float().abs().amax()).all()


def test_module(device) -> None:
    rotary = nmb.RotaryPositions(80, rotary_dim=32, interleaved=True, scaling="parts", factor=4.0, original_length=1024,
                                 magnitude=1.1).to(device).to(torch.bfloat16)
    q, k, *_ = make(2, 10, 4, 2, 80, torch.bfloat16, device)
    f = Fn.rotary_frequencies(32, scaling="parts", factor=4.0, original_length=1024, device=device)
    start = torch.tensor([3, 70_000], dtype=torch.int32, device=device)
    want = Fn.rotary_positions(q, k, f, sequence_offset=start, interleaved=True, magnitude=1.1)
    got = rotary(q, k, sequence_offset=start)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and not list(rotary.state_dict())


def test_module_captured_at_its_first_call(device) -> None:
    """Its frequencies came with the module, in 64 bits whatever it was turned into."""
    rotary = nmb.RotaryPositions(64).to(torch.bfloat16).to(device)
    q, k, *_ = make(1, 10, 2, 1, 64, torch.bfloat16, device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = rotary(q, k)
    graph.replay()
    want = Fn.rotary_positions(q, k, Fn.rotary_frequencies(64, device=device))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_captured_and_replayed(device) -> None:
    b, s = 3, 70
    fixed = make(b, s, 8, 2, 64, torch.bfloat16, device)
    pos = torch.randint(0, 1000, (b, s), device=device)
    f = Fn.rotary_frequencies(64, device=device)

    def step(q, k, gq, gk, pos):
        leaves = [t.detach().requires_grad_(True) for t in (q, k)]
        out = Fn.rotary_positions(*leaves, f, positions=pos)
        return [t.detach() for t in (*out, *torch.autograd.grad(out, leaves, (gq, gk)))]

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step(*fixed, pos)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(*fixed, pos)
    for seed in range(1, 5):
        new = make(b, s, 8, 2, 64, torch.bfloat16, device, seed)
        moved = torch.randint(0, 1_000_000, (b, s), generator=torch.Generator().manual_seed(seed)).to(device)
        for a, t in zip((*fixed, pos), (*new, moved)):
            a.copy_(t)
        graph.replay()
        got = [t.clone() for t in out]
        want = step(*new, moved)
        torch.cuda.synchronize()
        assert all(torch.equal(a, w) for a, w in zip(got, want)), seed


def test_checkpointed_and_offloaded(device) -> None:
    q, k, gq, gk = make(2, 30, 4, 2, 64, torch.bfloat16, device)
    pos = torch.randint(0, 1000, (2, 30), device=device)
    f = Fn.rotary_frequencies(64, device=device)

    def turn(q, k):
        return Fn.rotary_positions(q, k, f, positions=pos)

    def gradients(g):
        leaves = [t.detach().requires_grad_(True) for t in (q, k)]
        out = g(*leaves)
        return [*out, *torch.autograd.grad(out, leaves, (gq, gk))]

    def offloaded(*args):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().cpu().contiguous() if t.ndim == 2 else t.cpu(),
                                                      lambda t: t.cuda().t() if t.ndim == 2 else t.cuda()):
            return turn(*args)

    want = gradients(turn)
    for got in (gradients(lambda *t: torch.utils.checkpoint.checkpoint(turn, *t, use_reentrant=False)),
                gradients(offloaded)):
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_device_refusals(device) -> None:
    q, k, *_ = make(2, 10, 4, 2, 64, torch.bfloat16, device)
    f = Fn.rotary_frequencies(64)
    with pytest.raises(ValueError, match="frequencies must be on"):
        Fn.rotary_positions(q, k, f)
    f = f.to(device)
    with pytest.raises(ValueError, match="one device"):
        Fn.rotary_positions(q, k.cpu(), f)
    with pytest.raises(ValueError, match="positions"):
        Fn.rotary_positions(q, k, f, positions=torch.arange(10))
    with pytest.raises(ValueError, match="positions"):
        Fn.rotary_positions(q, k, f, positions=torch.arange(11, device=device))
    with pytest.raises(ValueError, match="positions"):
        Fn.rotary_positions(q, k, f, positions=torch.arange(10.0, device=device))
    with pytest.raises(ValueError, match="exclude"):
        Fn.rotary_positions(q, k, f, positions=torch.arange(10, device=device), sequence_offset=3)
    with pytest.raises(ValueError, match="sequence_offset"):
        Fn.rotary_positions(q, k, f, sequence_offset=torch.zeros(3, dtype=torch.int32, device=device))
    with pytest.raises(ValueError, match="2\\^40"):
        Fn.rotary_positions(q, k, f, sequence_offset=1 << 41)
