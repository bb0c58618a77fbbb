"""A distance bias that grows with the distance: negative slopes."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn
from tests.scored import check, reference
from tests.test_gpu_scored_attention import ids, make, run
from tests.test_gpu_scored_nan import fastest

pytestmark = pytest.mark.gpu


def compare(q, k, v, do, *, sequence_offset=0, score_cap, distance_slopes, **kw):
    """The bounds of ``reference`` take a score's bias as off by 2^-23 of it, with its sign,
    which for slopes below 0 takes from the bound instead of adding to it: by up to f = 2
    2^-23 |slope| keys of a head (no distance counts for more).  A probability is off by the
    factor exp(2 f) more, hence o by 2 f max|v|, dO.o and dP - delta <= 2 D max|dO| max|v| by
    2 f of D max|dO| max|v| and of themselves, and the sums over keys (whose probabilities
    add up to 1) and over queries (each at most 1) by as much of their factors.
    With biases of hundreds many probabilities also lie below 2^-126, where the kernels'
    exponentials are 0: each term of a sum may miss 2^-126 of its factors."""
    got = run(q, k, v, do, sequence_offset=sequence_offset, score_cap=score_cap, distance_slopes=distance_slopes, **kw)
    want = reference(q, k, v, do, offset=sequence_offset, cap=score_cap, slopes=distance_slopes, **kw)
    top = {n: float(t.abs().max()) for n, t in (("q", q), ("k", k), ("v", v), ("do", do))}
    (_, hq, sq, d), (_, hkv, sk, _) = q.shape, k.shape
    f = (2 * 2.0**-23 * sk * distance_slopes.double().abs() * (distance_slopes < 0)).view(1, hq, 1, 1)
    f_kv = f.view(hkv, -1).amax(1).view(1, hkv, 1, 1)
    ds, queries = d * top["do"] * top["v"] / d**0.5, sq * hq // hkv
    more = {"o": 2 * f * top["v"], "dq": (6 * f + 2.0**-125 * sk) * ds * top["k"],
            "dk": (6 * f_kv + 2.0**-125) * queries * ds * top["q"], "dv": (2 * f_kv + 2.0**-126) * queries * top["do"]}
    for name, value in got.items():
        check(name, value, (want[name][0], want[name][1] + more[name]))
        assert value.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("cap", [None, 30.0, 55.0, 90.0])
@pytest.mark.parametrize("shape", [(2, 8, 2, 700, 700, 64), (1, 4, 2, 300, 300, 128), (2, 20, 4, 260, 260, 80),
                                   (2, 8, 2, 3, 1500, 64)])
def test_negative_slopes(device, shape, cap, dtype) -> None:
    """Of both signs at once; documents and a window, and queries before and behind the keys."""
    b, hq, _, sq, sk, _ = shape
    q, k, v, do = make(*shape, dtype, device)
    sl = torch.linspace(-3.0, 0.5, hq, device=device)
    compare(q, k, v, do, sequence_offset=sk - sq, score_cap=cap, distance_slopes=sl)
    compare(q, k, v, do, causal=False, score_cap=cap, distance_slopes=sl)
    compare(q, k, v, do, causal=False, sequence_offset=sk + 50, score_cap=cap, distance_slopes=sl, window=200)
    compare(q, k, v, do, sequence_offset=sk - sq, score_cap=cap, distance_slopes=sl, documents=ids(b, sk, 200, device, pad=9))


@pytest.mark.parametrize("sq", [3, 1024])
def test_negative_slopes_take_no_longer(device, sq) -> None:
    """(The weights of the furthest keys left fp32's range, and every row was run again by
    itself: 7.2 ms instead of 0.04 with 1,024 queries.)"""
    q, k, v, _ = make(2, 16, 4, sq, 1024, 64, torch.bfloat16, device)
    sl = torch.exp2(-8.0 * torch.arange(1, 17, device=device) / 16)
    f = lambda s: Fn.scored_attention(q, k, v, sequence_offset=1024 - sq, score_cap=30.0, distance_slopes=s)  # noqa: E731
    f(sl), f(-sl)
    assert fastest(lambda: f(-sl), 10) < 4 * fastest(lambda: f(sl), 10)
