"""The autograd nodes in C++ are those of this header, bindings and library, or are not used."""

from __future__ import annotations

import pathlib
import re

import pytest

from nano_megatron_amd import _lib
from nano_megatron_amd import functional as Fn


def test_one_version() -> None:
    header = (pathlib.Path(__file__).resolve().parents[1] / "include" / "nmb.h").read_text()
    version = int(re.search(r"#define NMB_ABI_VERSION (\d+)", header).group(1))
    assert version == _lib.ABI_VERSION == _lib.load().nmb_abi_version() == Fn._nodes().abi_version


@pytest.mark.parametrize("built", [1, 3, None])
def test_nodes_of_another_version_are_refused(monkeypatch, built) -> None:
    nodes = Fn._nodes()
    if built is None:
        monkeypatch.delattr(nodes, "abi_version")
    else:
        monkeypatch.setattr(nodes, "abi_version", built)
    with pytest.raises(RuntimeError, match="nano_megatron_amd.build"):
        Fn._nodes.__wrapped__()
