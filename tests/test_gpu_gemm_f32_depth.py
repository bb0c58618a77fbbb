"""The fp32 GEMM over numbers of K tiles: none whole, one, two, the least that a loop takes and
more, with and without a remainder, split and not, against fp64."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(128, 64), (512, 4096), (192, 68)])
@pytest.mark.parametrize("k", [4, 28, 32, 36, 64, 68, 96, 100, 128, 156, 160, 192, 224, 260])
@pytest.mark.parametrize("at,bt", [(False, True), (False, False), (True, False), (True, True)])
def test_numbers_of_k_tiles(m, n, k, at, bt) -> None:
    """Leading dimensions of whole 16 bytes; 512 x 4096 is not split.  Bound: a recursive sum of k
    products is off by 2^-24 k sum |a b| at most, and each is rounded no more than once."""
    g = torch.Generator(device="cuda").manual_seed(m + 3 * n + 5 * k)
    a = torch.randn((k, m) if at else (m, k), generator=g, device="cuda")
    b = torch.randn((n, k) if bt else (k, n), generator=g, device="cuda")
    a, b = a.t() if at else a, b.t() if bt else b
    out = Fn.mm(a, b)
    bound = 2.0 ** -24 * (k + 2) * (a.double().abs() @ b.double().abs())
    assert ((out.double() - a.double() @ b.double()).abs() <= bound).all()
