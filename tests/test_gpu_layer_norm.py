"""layer_norm against 64 bits, both directions: sizes, strides, residuals, partial
gradients, streams and captures."""

from __future__ import annotations

import pytest
import torch

import nano_megatron_amd.functional as Fn
from nano_megatron_amd import HipKernelBackend, LayerNorm

pytestmark = pytest.mark.gpu

EPS = 1e-5
U32 = 2.0**-24


def make(rows, cols, dtype, device, seed=0, residual=True, bias=True, offset=3.0):
    g = torch.Generator().manual_seed(seed)

    def t(*shape, std=1.0, mean=0.0):
        return (torch.randn(*shape, generator=g) * std + mean).to(dtype).to(device)

    return {"x": t(rows, cols, mean=offset), "w": t(cols, std=0.3, mean=1.0), "b": t(cols) if bias else None,
            "res": t(rows, cols, std=2.0) if residual else None, "gy": t(rows, cols),
            "gh": t(rows, cols) if residual else None}


def run(st, eps=EPS):
    leaves = {n: st[n].detach().requires_grad_(True) for n in ("x", "res", "w", "b") if st[n] is not None}
    out = Fn.layer_norm(leaves["x"], leaves["w"], leaves.get("b"), eps, residual=leaves.get("res"))
    out = out if isinstance(out, tuple) else (out,)
    grads = torch.autograd.grad(out, list(leaves.values()), [st[n] for n in ("gy", "gh")[:len(out)]])
    got = dict(zip(("y", "h"), (t.detach() for t in out)))
    got.update(zip(("d" + n for n in leaves), grads))
    return got


def reference(st, eps=EPS):
    """Values in 64 bits, each with its bound.  A sum of n fp32 terms, added at most 32 in a
    row and then pairwise, is off by 45 u of the sum of their sizes (u = 2^-24).  The mean is
    off by e = 45 u mean|h|; n = (h - mu) s by s (e + 2 u (|h| + |mu|)) and, through s, by
    |n| r, where the variance's sum is off by 2 * 45 u plus (e + u |mu|)^2 of it, s by half
    that and 6 u; the products of the gradient by 2 u each; sums over rows, added rows / 256
    and then 40 in a row, by so many u of their sizes.  Results by half a step of their type."""
    f = torch.float64
    dtype = st["x"].dtype
    half = torch.finfo(dtype).eps / 2
    rows, cols = st["x"].shape
    h = st["x"].to(f)
    out = {}
    if st["res"] is not None:
        full = h + st["res"].to(f)
        out["h"] = (full, half * full.abs() + U32 * full.abs())
        h = (st["x"].float() + st["res"].float()).to(dtype).to(f)
    w = st["w"].to(f)
    b = torch.zeros_like(w) if st["b"] is None else st["b"].to(f)
    mu = h.mean(1, keepdim=True)
    var = ((h - mu) ** 2).mean(1, keepdim=True)
    s = 1 / torch.sqrt(var + eps)
    n = (h - mu) * s
    e = 46 * U32 * h.abs().mean(1, keepdim=True)
    r = 60 * U32 + (e * s) ** 2 + 2 * e * s * n.abs().mean(1, keepdim=True)
    n_off = s * (e + 2 * U32 * (h.abs() + mu.abs())) + n.abs() * r
    y = n * w + b
    out["y"] = (y, n_off * w.abs() + 3 * U32 * ((n * w).abs() + b.abs()) + half * y.abs())
    gy = st["gy"].to(f)
    g = gy * w
    m1, m2 = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
    m1_off = 46 * U32 * g.abs().mean(1, keepdim=True)
    m2_off = 46 * U32 * (g * n).abs().mean(1, keepdim=True) + (g.abs() * n_off).mean(1, keepdim=True)
    core = g - m1 - n * m2
    dx = s * core
    dx_off = s * (4 * U32 * (g.abs() + m1.abs() + (n * m2).abs()) + m1_off + n.abs() * m2_off + n_off * m2.abs()) \
        + dx.abs() * r
    if st["gh"] is not None:
        dx = dx + st["gh"].to(f)
        dx_off = dx_off + 2 * U32 * (dx.abs() + st["gh"].to(f).abs())
    out["dx"] = (dx, dx_off + half * dx.abs())
    if st["res"] is not None:
        out["dres"] = out["dx"]
    depth = (rows / 256 + 42) * U32
    dw = (gy * n).sum(0)
    out["dw"] = (dw, depth * (gy * n).abs().sum(0) + (gy.abs() * n_off).sum(0) + half * dw.abs())
    if st["b"] is not None:
        db = gy.sum(0)
        out["db"] = (db, depth * gy.abs().sum(0) + half * db.abs())
    return out


def check(got, want):
    assert set(got) == set(want)
    for name, (value, bound) in want.items():
        off = (got[name].double() - value).abs()
        # second order: bounds are of first order in the roundings
        assert (off <= bound * 1.01 + 1e-37).all(), (name, float((off - bound).max()), float(off.max()))


SHAPES = [
    (1, 1), (3, 1), (5, 2), (7, 3), (9, 4), (2, 5), (7, 7), (1, 8), (4, 9), (33, 31), (130, 40), (2, 64), (9, 65),
    (5, 128), (17, 130), (17, 256), (3, 257), (6, 385), (6, 513), (5, 768), (4, 777), (130, 1024), (3, 1001),
    (2, 1537), (5, 2048), (3, 2049), (2, 4097), (2, 6145), (2, 8192), (1, 8193), (3, 16383), (2, 16384), (700, 768),
    (4099, 40), (2100, 1000),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("residual,bias", [(True, True), (False, False)])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_layer_norm(device, rows, cols, residual, bias, dtype) -> None:
    st = make(rows, cols, dtype, device, residual=residual, bias=bias)
    got = run(st)
    check(got, reference(st))
    again = run(st)
    assert all(torch.equal(got[n], again[n]) for n in got)
    with torch.no_grad():  # without gradients: the same bits
        out = Fn.layer_norm(st["x"], st["w"], st["b"], EPS, residual=st["res"])
    out = out if residual else (out,)
    assert all(torch.equal(a, got[n]) for a, n in zip(out, ("y", "h")))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_rows_far_from_zero(device, dtype) -> None:
    """The mean, a thousand times the spread, is off before the squares are summed."""
    st = make(50, 768, dtype, device, residual=False, offset=1000.0 if dtype == torch.float32 else 40.0)
    check(run(st), reference(st))


def test_constant_rows_give_the_bias(device) -> None:
    w, b = torch.full((96,), 2.0, device=device), torch.arange(96.0, device=device)
    assert torch.equal(Fn.layer_norm(torch.full((3, 96), 5.0, device=device), w, b), b.expand(3, 96))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_differences(device, dtype) -> None:
    """The gradient along a direction against the central difference of the formula in 64
    bits, whose own error (third derivatives at steps of 1e-4) is below 1e-6 of its size."""
    st = make(6, 200, dtype, device)
    got, want = run(st), reference(st)
    f = torch.float64
    gen = torch.Generator().manual_seed(3)
    along = {n: torch.randn(st[n].shape, generator=gen).to(device, f) for n in ("x", "w", "b")}

    def value(t):
        # the residual's rounding has no derivative: the sum as it is stored, moved
        h = (st["x"].float() + st["res"].float()).to(dtype).to(f) + t * along["x"]
        n = (h - h.mean(1, keepdim=True)) / torch.sqrt(h.var(1, correction=0, keepdim=True) + EPS)
        y = n * (st["w"].to(f) + t * along["w"]) + st["b"].to(f) + t * along["b"]
        return (y * st["gy"].to(f)).sum() + (h * st["gh"].to(f)).sum()

    difference = (value(1e-4) - value(-1e-4)) / 2e-4
    slope = sum((got["d" + n].double() * along[n]).sum() for n in along)
    bound = sum((want["d" + n][1] * along[n].abs()).sum() for n in along)
    size = sum((want["d" + n][0] * along[n]).abs().sum() for n in along)
    assert (slope - difference).abs() <= 1.01 * bound + 1e-6 * size


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_strides(device, dtype) -> None:
    """Columns of a wider tensor (rows of odd strides and starts), tensors of more
    dimensions, every second column, one row for all, transposed gradients."""
    base = make(30, 77, dtype, device)
    want = run(base)
    for name in ("x", "res", "gy", "gh"):
        wide = torch.full((30, 133), float("nan"), dtype=dtype, device=device)
        wide[:, 5:82] = base[name]
        got = run({**base, name: wide[:, 5:82]})
        assert all(torch.equal(got[n], want[n]) for n in want), name
        apart = torch.full((30, 154), float("nan"), dtype=dtype, device=device)
        apart[:, ::2] = base[name]
        got = run({**base, name: apart[:, ::2]})
        assert all(torch.equal(got[n], want[n]) for n in want), name
        got = run({**base, name: base[name].t().contiguous().t()})
        assert all(torch.equal(got[n], want[n]) for n in want), name
    many = {n: t.view(2, 3, 5, 77) if t is not None and t.ndim == 2 else t for n, t in base.items()}
    got = run({**many, "gy": many["gy"].transpose(0, 2).contiguous().transpose(0, 2)})
    for n, t in want.items():
        assert got[n].shape == (many["x"].shape if t.ndim == 2 else t.shape)
        assert torch.equal(got[n].reshape(t.shape), t)
    one = {**base, **{n: base[n][:1].expand(30, 77) for n in ("x", "gy")}}
    got, dense = run(one), run({n: None if t is None else t.contiguous() for n, t in one.items()})
    assert all(torch.equal(got[n], dense[n]) for n in dense)
    vector = Fn.layer_norm(base["x"][3], base["w"], base["b"])
    assert torch.equal(vector, Fn.layer_norm(base["x"], base["w"], base["b"])[3])
    every_second = torch.stack((base["w"], base["b"]), 1)
    assert torch.equal(Fn.layer_norm(base["x"], every_second[:, 0], every_second[:, 1]),
                       Fn.layer_norm(base["x"], base["w"], base["b"]))


def test_strided_weights_get_gradients(device) -> None:
    st = make(30, 77, torch.float32, device)
    want = run(st)
    both = torch.stack((st["w"], st["b"]), 1).requires_grad_(True)
    y, h = Fn.layer_norm(st["x"], both[:, 0], both[:, 1], EPS, residual=st["res"])
    grad, = torch.autograd.grad(y, both, st["gy"])
    assert torch.equal(grad[:, 0], want["dw"]) and torch.equal(grad[:, 1], want["db"])


def test_graphs_are_freed(device) -> None:
    """Outputs that are saved themselves (the sum) keep no graph alive, used or not."""
    st = make(300, 768, torch.bfloat16, device)
    run(st)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(3):
        x = st["x"].detach().requires_grad_(True)
        y, h = Fn.layer_norm(x, st["w"], st["b"], EPS, residual=st["res"])
        del y, h, x
        run(st)
    assert torch.cuda.memory_allocated() == before


def test_some_gradients(device) -> None:
    """Only what is asked for, through one output, both or neither."""
    st = make(40, 200, torch.float32, device)
    want = run(st)
    for names in (("x",), ("w",), ("b",), ("res",), ("x", "b"), ("w", "res")):
        leaves = {n: st[n].detach().requires_grad_(n in names) for n in ("x", "w", "b", "res")}
        y, h = Fn.layer_norm(leaves["x"], leaves["w"], leaves["b"], EPS, residual=leaves["res"])
        got = torch.autograd.grad((y, h) if h.requires_grad and h.grad_fn else y, [leaves[n] for n in names],
                                  (st["gy"], st["gh"]) if h.requires_grad and h.grad_fn else st["gy"])
        assert all(torch.equal(g, want["d" + n]) for g, n in zip(got, names)), names
    leaves = [st[n].detach().requires_grad_(True) for n in ("x", "w", "b", "res")]
    y, h = Fn.layer_norm(*leaves[:3], EPS, residual=leaves[3])
    through_sum = torch.autograd.grad(h, leaves, st["gh"], retain_graph=True, allow_unused=True)
    assert torch.equal(through_sum[0], st["gh"]) and torch.equal(through_sum[3], st["gh"])
    assert all(t is None or not t.any() for t in through_sum[1:3])
    only_y = torch.autograd.grad(y, leaves, st["gy"])
    check({"dx": only_y[0]}, {"dx": reference({**st, "gh": torch.zeros_like(st["gy"])})["dx"]})
    y, h = Fn.layer_norm(*leaves[:3], EPS, residual=leaves[3])
    ones = torch.autograd.grad(y.sum() + h.sum(), leaves)  # broadcast gradients
    want = run({**st, "gy": torch.ones_like(st["gy"]), "gh": torch.ones_like(st["gh"])})
    assert all(torch.equal(a, want["d" + n]) for a, n in zip(ones, ("x", "w", "b", "res")))
    # the same tensor as input and residual gets both gradients
    x = st["x"].detach().requires_grad_(True)
    y, h = Fn.layer_norm(x, st["w"], st["b"], EPS, residual=x)
    twice, = torch.autograd.grad((y, h), x, (st["gy"], st["gh"]))
    assert torch.equal(twice, 2 * run({**st, "res": st["x"]})["dx"])


def test_no_rows(device) -> None:
    st = make(0, 96, torch.bfloat16, device)
    got = run(st)
    assert got["y"].shape == got["dx"].shape == (0, 96)
    assert not got["dw"].any() and not got["db"].any()


@pytest.mark.parametrize("cols", [40, 768, 3000, 9000])
def test_a_row_of_nan_stays_in_its_row(device, cols) -> None:
    st = make(40, cols, torch.bfloat16, device)
    want = run(st)
    for bad in (float("nan"), float("inf")):
        x = st["x"].clone()
        x[7, cols // 2] = bad
        got = run({**st, "x": x})
        keep = torch.arange(40, device=device) != 7
        for n in ("y", "h", "dx"):
            assert torch.equal(got[n][keep], want[n][keep])
        assert got["y"][7].isnan().any() and got["dw"].isnan().any()
        assert torch.equal(got["db"], want["db"])


def test_past_32_bit_offsets(device) -> None:
    """140,000 rows of 16,384 (2.3e9 elements), read from one row and written dense."""
    row = torch.randn(16384, generator=torch.Generator().manual_seed(1)).bfloat16().to(device)
    w, b = torch.full_like(row, 1.5), torch.full_like(row, 0.25)
    y = Fn.layer_norm(row.expand(140_000, 16384), w, b)
    want = Fn.layer_norm(row, w, b)
    for at in (0, 65_535, 131_071, 131_072, 139_999):
        assert torch.equal(y[at], want), at


def test_module_and_backend(device) -> None:
    st = make(20, 96, torch.bfloat16, device)
    for norm in (LayerNorm(96, device=device, dtype=torch.bfloat16),
                 HipKernelBackend().layer_norm(96, 1e-6, bias=False, device=device, dtype=torch.bfloat16)):
        with torch.no_grad():
            norm.weight.copy_(st["w"])
        y, h = norm(st["x"], st["res"])
        want = Fn.layer_norm(st["x"], norm.weight, norm.bias, norm.eps, residual=st["res"])
        assert torch.equal(y, want[0]) and torch.equal(h, want[1])
        assert torch.equal(norm(h), y)  # the sum as it is stored
        assert sorted(norm.state_dict()) == (["bias", "weight"] if norm.bias is not None else ["weight"])


@pytest.mark.parametrize("rows,cols", [(300, 768), (40, 5000)])
def test_captured_and_replayed(device, rows, cols) -> None:
    """Forward and backward in one graph, replayed on new values between eager work."""
    fixed = make(rows, cols, torch.bfloat16, device)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(fixed)
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(fixed)
    for seed in range(1, 5):
        new = make(rows, cols, torch.bfloat16, device, seed=seed)
        for n, t in fixed.items():
            t.copy_(new[n])
        graph.replay()
        got = {n: t.clone() for n, t in out.items()}
        want = run(new)
        torch.cuda.synchronize()
        assert all(torch.equal(got[n], want[n]) for n in want), seed


def test_two_streams(device) -> None:
    states = [make(500, 768, torch.bfloat16, device, seed=n) for n in range(2)]
    want = [run(st) for st in states]
    streams = [torch.cuda.Stream() for _ in states]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for n, (stream, st) in enumerate(zip(streams, states)):
            with torch.cuda.stream(stream):
                got[n].append(run(st))
    torch.cuda.synchronize()
    for runs, w in zip(got, want):
        assert all(torch.equal(r[n], w[n]) for r in runs for n in w)


def test_checkpointed_and_offloaded(device) -> None:
    st = make(50, 200, torch.bfloat16, device)
    want = run(st)

    def gradients(f):
        leaves = [st[n].detach().requires_grad_(True) for n in ("x", "res", "w", "b")]
        out = f(*leaves)
        grads = torch.autograd.grad(out, leaves, (st["gy"], st["gh"]))
        return dict(zip(("y", "h", "dx", "dres", "dw", "db"), (*out, *grads)))

    def norm(x, res, w, b):
        return Fn.layer_norm(x, w, b, EPS, residual=res)

    def offloaded(*args):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.t().cpu().contiguous() if t.ndim == 2 else t.cpu(),
                                                      lambda t: t.cuda().t() if t.ndim == 2 else t.cuda()):
            return norm(*args)

    for got in (gradients(lambda *t: torch.utils.checkpoint.checkpoint(norm, *t, use_reentrant=False)),
                gradients(offloaded)):
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_no_second_derivative(device) -> None:
    st = make(4, 64, torch.float32, device)
    x = st["x"].detach().requires_grad_(True)
    first, = torch.autograd.grad(Fn.layer_norm(x, st["w"], st["b"]).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        first.sum().backward()


def test_one_device(device) -> None:
    st = make(4, 64, torch.float32, device)
    for name in ("w", "b", "res"):
        bad = {**st, name: st[name].cpu()}
        with pytest.raises(ValueError, match="one device"):
            Fn.layer_norm(bad["x"], bad["w"], bad["b"], residual=bad["res"])
