"""rotary_frequencies, and what rotary_positions refuses, before any device work."""

from __future__ import annotations

import math

import pytest
import torch

from nano_megatron_amd import RotaryPositions, _lib
from nano_megatron_amd import functional as Fn

FAKE = 256  # a non-null address that is never dereferenced
ONE = _lib.i64x3((64, 64, 64))


def test_frequencies() -> None:
    f = Fn.rotary_frequencies(8, 10_000.0)
    assert f.dtype == torch.float64
    # a power's error is a few steps of 64 bits
    assert torch.allclose(f, torch.tensor([1, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)
    assert torch.equal(Fn.rotary_frequencies(8, scaling="linear", factor=4.0), f / 4)
    base = Fn.rotary_frequencies(8, scaling="base", factor=4.0)
    assert base[0] == 1 and math.isclose(base[-1], f[-1] / 4, rel_tol=1e-13)
    assert torch.equal(Fn.rotary_frequencies(2, scaling="base", factor=4.0), torch.ones(1, dtype=torch.float64))


def test_frequencies_by_parts() -> None:
    """Pairs of 159, 15.9, 1.59 and 0.159 turns in 1,000 tokens, with 1 and 32 as the ends."""
    f = Fn.rotary_frequencies(8, 10_000.0)
    got = Fn.rotary_frequencies(8, scaling="parts", factor=8.0, original_length=1000)
    assert got[0] == f[0] and math.isclose(got[3], f[3] / 8, rel_tol=1e-15)
    for j in (1, 2):
        stays = (1000 * float(f[j]) / (2 * math.pi) - 1) / 31
        assert 0 < stays < 1
        assert math.isclose(got[j], float(f[j]) * (stays + (1 - stays) / 8), rel_tol=1e-14)
    narrow = Fn.rotary_frequencies(8, scaling="parts", factor=8.0, original_length=1000, slow_turns=0.0, fast_turns=0.1)
    assert torch.equal(narrow, f)  # every pair turns more often than that


@pytest.mark.parametrize("kw,message", [
    (dict(rotary_dim=0), "even"), (dict(rotary_dim=7), "even"), (dict(rotary_dim=-2), "even"),
    (dict(theta=0.0), "theta"), (dict(theta=math.inf), "theta"), (dict(factor=0.0), "factor"),
    (dict(factor=math.nan), "factor"), (dict(scaling="other"), "scaling"), (dict(scaling="parts"), "original_length"),
    (dict(scaling="parts", original_length=0), "original_length"),
    (dict(scaling="parts", original_length=8, slow_turns=2.0, fast_turns=2.0), "slow_turns"),
])
def test_frequency_refusals(kw, message) -> None:
    with pytest.raises(ValueError, match=message):
        Fn.rotary_frequencies(**{"rotary_dim": 8, **kw})


F4 = torch.ones(4, dtype=torch.float64)


@pytest.mark.parametrize("kw,message", [
    (dict(q=torch.ones(2, 3, 8)), "shape"), (dict(k=torch.ones(2, 3, 8)), "shape"),
    (dict(k=torch.ones(2, 1, 4, 8)), "agree"), (dict(k=torch.ones(1, 1, 5, 8)), "agree"),
    (dict(k=torch.ones(2, 1, 5, 10)), "agree"), (dict(k=torch.ones(2, 1, 5, 8).bfloat16()), "one dtype"),
    (dict(frequencies=F4.float()), "float64"), (dict(frequencies=F4[None]), "float64"),
    (dict(frequencies=F4[:0]), "float64"), (dict(frequencies=torch.ones(5, dtype=torch.float64)), "float64"),
    (dict(frequencies=F4.clone().requires_grad_(True)), "no gradient"),
    (dict(magnitude=math.nan), "magnitude"), (dict(magnitude=1e31), "magnitude"),
    (dict(q=torch.ones(2, 3, 5, 8).half(), k=None), "float16"),
    (dict(), "GPU only"), (dict(k=None), "GPU only"),
])
def test_refusals(kw, message) -> None:
    args = {"q": torch.ones(2, 3, 5, 8), "k": torch.ones(2, 1, 5, 8), "frequencies": F4, **kw}
    with pytest.raises(ValueError, match=message):
        Fn.rotary_positions(**args)


def test_module_checks() -> None:
    with pytest.raises(ValueError, match="exceed"):
        RotaryPositions(64, rotary_dim=66)
    with pytest.raises(ValueError, match="heads of 64"):
        RotaryPositions(64)(torch.ones(1, 1, 1, 32))
    assert len(RotaryPositions(64, rotary_dim=16).frequencies(torch.device("cpu"))) == 8


@pytest.mark.parametrize("change,message", [
    (dict(rot=0), "rotary_dim"), (dict(rot=3), "rotary_dim"), (dict(rot=66), "rotary_dim"), (dict(batch=-1), "shape"),
    (dict(seq=1 << 31), "shape"), (dict(hq=-1), "shape"), (dict(q=None), "null"), (dict(qs=None), "null"),
    (dict(qo=None), "null"), (dict(k=None), "null"), (dict(kos=None), "null"), (dict(freq=None), "null"),
    (dict(size=2), "4 or 8"), (dict(offsets=FAKE), "exclude"), (dict(dtype=5), "dtype"),
    (dict(batch=1 << 16, seq=1 << 16), "too many"),
])
def test_entry(change, message) -> None:
    a = {**dict(q=FAKE, qs=ONE, qo=FAKE, qos=ONE, hq=2, k=FAKE, ks=ONE, ko=FAKE, kos=ONE, hk=1, freq=FAKE, rot=64,
                pos=FAKE, size=4, pb=0, ps=1, offsets=None, offset=0, batch=2, seq=3, dim=64, inter=0, inv=0, mag=1.0,
                dtype=_lib.NMB_BF16), **change}
    with pytest.raises(ValueError, match=message):
        _lib.call("nmb_rotary", *a.values(), None)
