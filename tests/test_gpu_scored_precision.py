"""What the training forward of scored_attention keeps beyond its rounded output: the
probabilities' second bf16 term and the part of the output that its rounding cut off, for
the backward's row sums."""

from __future__ import annotations

import math

import pytest
import torch

import nano_megatron_amd.functional as Fn
from tests.scored import reference
from tests.test_gpu_scored_attention import make, run

pytestmark = pytest.mark.gpu

# the few-query kernel (one workgroup a row tile, and keys shared out), 64 and 128 queries a
# workgroup, 64, 96 and 128 columns
SHAPES = [
    (2, 2, 2, 63, 63, 64), (1, 4, 2, 64, 64, 128), (2, 8, 2, 5, 2500, 64), (1, 8, 1, 3, 3000, 128),
    (3, 24, 8, 65, 65, 64), (2, 34, 2, 63, 190, 128), (5, 14, 7, 33, 200, 80),
    (16, 33, 3, 129, 129, 64), (17, 32, 4, 100, 300, 128), (33, 16, 2, 70, 65, 88),
]
MODES = [(None, False), (20.0, False), (None, True), (50.0, True), (90.0, False)]


def scores(hq, slopes, device):
    return torch.exp2(-8.0 * torch.arange(1, hq + 1) / hq).to(device) if slopes else None


@pytest.mark.parametrize("cap,slopes", MODES)
@pytest.mark.parametrize("shape", SHAPES)
def test_output_and_what_its_rounding_cut_off(device, shape, cap, slopes) -> None:
    """o + o_low is the output up to the products' fp32 errors (those of ``reference``'s bound
    without its roundings to bf16) and u^2 = 2^-16 of P and of o, what is left of each behind
    two terms; o is the rounding of that."""
    b, hq, hkv, sq, sk, d = shape
    q, k, v, _ = make(*shape, torch.bfloat16, device)
    sl = scores(hq, slopes, device)
    meta = (1.0 / math.sqrt(d), cap or 0.0, 1, 0, sk - sq)
    o, aux, _ = Fn._scored_fwd(q, k, v, (meta, sl, None, None, None), True)
    low = aux[Fn._lse_bytes(b, hq, sq):].view(torch.bfloat16).view(b, sq, hq, d).transpose(1, 2)
    want, bound = reference(q, k, v, offset=sk - sq, cap=cap, slopes=sl)["o"]
    # the same attention of |v|: sum P |v|
    spread = reference(q, k, v.abs(), offset=sk - sq, cap=cap, slopes=sl)["o"][0]
    u = 2.0**-8
    rest = (bound - 1.01 * u * spread - 2.01 * u * want.abs()).clamp_min(0)  # of the fp32 errors alone
    tight = rest + 1.01 * u * u * (spread + want.abs()) + 2.0**-23 * spread
    off = (o.double() + low.double() - want).abs()
    assert (off <= tight).all(), float((off / tight).max())
    # half a step of o at most, the remainder rounded in turn
    assert (low.double().abs() <= 1.01 * u * o.double().abs() + 1e-37).all()
    lost = (o.double() - want).norm() / want.norm()
    assert float(off.norm() / want.norm()) < 0.1 * float(lost)


@pytest.mark.parametrize("cap,slopes", MODES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gradients_by_their_norm(device, shape, cap, slopes) -> None:
    """dq and dk round twice: dS as an operand, and the result, by 2^-8 / sqrt 3 of a value
    at its mantissa's start and half that at its end, 1.66e-3 in the mean square of many
    values; both together sqrt 2 times that, 2.35e-3.  15% more are allowed for: few values,
    P's own rounding never enters, and the fp32 errors are below 1e-4.  With delta from the
    rounded output alone the error would be `without`, which the test's inputs take past the
    tolerance where that is asserted."""
    b, hq, hkv, sq, sk, d = shape
    q, k, v, do = make(*shape, torch.bfloat16, device)
    sl = scores(hq, slopes, device)
    got = run(q, k, v, do, sequence_offset=sk - sq, score_cap=cap, distance_slopes=sl)
    want = reference(q, k, v, do, offset=sk - sq, cap=cap, slopes=sl)
    one = math.sqrt(2) * 1.66e-3
    for name in ("dq", "dk"):
        value = want[name][0]
        off = float((got[name].double() - value).norm() / value.norm())
        assert off < 1.15 * one, (name, off)
    assert float((got["dv"].double() - want["dv"][0]).norm() / want["dv"][0].norm()) < 1.15 * one
    # dq with delta from the rounded output, everything else exact: dS is off by P (delta' -
    # delta), which is dq of a gradient that reaches P through delta alone
    f = torch.float64
    o64 = want["o"][0]
    shift = (do.to(f) * (o64.bfloat16().to(f) - o64)).sum(3, keepdim=True)
    group = hq // hkv
    kf, qf = k.to(f).repeat_interleave(group, 1), q.to(f)
    s = qf @ kf.transpose(2, 3) / math.sqrt(d)
    bent = torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        s, bent = cap * t, 1 - t * t
    far = torch.arange(sq, device=device)[:, None] + sk - sq - torch.arange(sk, device=device)
    if sl is not None:
        s = s - sl.to(f).view(1, -1, 1, 1) * far.abs()
    p = torch.softmax(s.masked_fill(far < 0, -math.inf), 3)
    without = float(((p * shift * bent) @ kf / math.sqrt(d)).norm() / want["dq"][0].norm())
    if shape in SHAPES[:2] or shape == SHAPES[4]:
        assert math.hypot(one, without) > 1.15 * one, without
