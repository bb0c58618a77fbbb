"""scored_attention where inputs are not numbers: which results are lost, and that finding
out does not take long."""

from __future__ import annotations

import math

import pytest
import torch

import nano_megatron_amd.functional as Fn
from tests.scored import visible
from tests.test_gpu_scored_attention import check, ids, make, reference, run

pytestmark = pytest.mark.gpu


def fastest(f, n=3):
    times = []
    for _ in range(n):
        start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        f()
        end.record()
        torch.cuda.synchronize()
        times.append(start.elapsed_time(end))
    return min(times)


# the tiled kernels, the few-query kernel, and shared walks over the queries
SHAPES = [(2, 16, 4, 300, 300, 64), (2, 4, 2, 130, 130, 128), (1, 8, 2, 700, 700, 80), (2, 4, 2, 5, 900, 64)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["q", "k", "v", "do"])
@pytest.mark.parametrize("shape", SHAPES)
def test_what_is_lost(device, shape, what, dtype) -> None:
    """One NaN row of an input: the results that a formula over visible pairs gives are NaN
    in all elements, the others are as without it."""
    b, hq, hkv, sq, sk, d = shape
    q, k, v, do = make(*shape, dtype, device)
    docs = ids(b, sk, 90, device, seed=7)
    kw = dict(documents=docs, sequence_offset=sk - sq, window=60)
    want = reference(q, k, v, do, documents=docs, offset=sk - sq, window=60, cap=20.0)
    at, head = (sq // 2 if what in ("q", "do") else sk - 20), 1
    dict(q=q, k=k, v=v, do=do)[what][0, head, at] = math.nan
    got = run(q, k, v, do, score_cap=20.0, **kw)
    seen = visible(b, sq, sk, causal=True, offset=sk - sq, prefix=None, window=60, documents=docs)[0]
    group = hq // hkv
    heads = torch.zeros(hq, dtype=torch.bool, device=device)
    heads[head if what in ("q", "do") else slice(head * group, (head + 1) * group)] = True
    rows = torch.zeros(sq, dtype=torch.bool, device=device)  # queries whose scores, or row sums, are lost
    if what in ("q", "do"):
        rows[at] = True
    else:
        rows = seen[:, at]
    rows = rows & seen.any(1)
    lost_q = heads[:, None] & rows
    keys = (seen & rows[:, None]).any(0)
    kv_heads = heads.view(hkv, group).any(1)
    lost_k = kv_heads[:, None] & keys
    empty = torch.zeros_like(lost_k)
    lost = {"o": torch.zeros_like(lost_q) if what == "do" else lost_q, "dq": lost_q, "dk": lost_k,
            # dO reaches dV of the keys it sees; a NaN in V reaches its own key's gradient not at all
            "dv": empty if what == "v" else lost_k}
    for name, value in got.items():
        mask = lost[name]
        assert value[0][mask].isnan().all(), name
        clean = ~torch.cat([mask[None], torch.zeros_like(mask)[None].expand(b - 1, *mask.shape)])
        check(name, value[clean], (want[name][0][clean], want[name][1][clean]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("what", ["all of do", "all of q", "one row of q", "one row of do", "one key"])
def test_a_lost_step_ends_soon(device, dtype, what) -> None:
    """A step whose loss is no longer a number, or that one token spoils: within 40 times the
    time of an ordinary one (the rows that it takes one by one end at once; walked through to
    their ends they took 180 times at these sizes, and more at longer ones)."""
    shape = (2, 16, 4, 1024, 1024, 64) if dtype == torch.bfloat16 else (1, 8, 2, 1024, 1024, 64)
    q, k, v, do = make(*shape, dtype, device)
    f = lambda: run(q, k, v, do, score_cap=20.0)  # noqa: E731
    f()
    clean = fastest(f)
    if what == "all of do":
        do.fill_(math.nan)
    elif what == "all of q":
        q.fill_(math.nan)
    elif what == "one key":
        k[:, :, 900] = math.nan
    else:
        (q if what == "one row of q" else do)[:, :, 900] = math.nan
    assert fastest(f) < 40 * clean
