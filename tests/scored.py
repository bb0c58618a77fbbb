"""Scored attention in 64 bits, with bounds on how far kernels may be from it."""

from __future__ import annotations

import math

import torch


def visible(b, sq, sk, *, causal, offset, prefix, window, documents):
    """[B, Sq, Sk] truth values, pair by pair."""
    dev = documents.device if documents is not None else "cpu"
    off = offset.long().to(dev).view(b, 1) if torch.is_tensor(offset) else torch.full((b, 1), offset, device=dev)
    pos = (off + torch.arange(sq, device=dev))[:, :, None]
    key = torch.arange(sk, device=dev)[None, None]
    seen = torch.ones(b, sq, sk, dtype=torch.bool, device=dev)
    if causal:
        seen &= (key <= pos) if prefix is None else (key <= pos) | (key < prefix.long().to(dev).view(b, 1, 1))
    if window:
        seen &= (pos - key).abs() < window
    if documents is not None:
        ids = documents.long()
        change = torch.zeros_like(ids)
        change[:, 1:] = (ids[:, 1:] != ids[:, :-1]).long()
        run = torch.cumsum(change, 1)
        inside = (pos >= 0) & (pos < sk)
        at = pos[:, :, 0].clamp(0, max(sk - 1, 0))
        seen &= inside & (run.gather(1, at)[:, :, None] == run[:, None]) & (ids.gather(1, at) >= 0)[:, :, None]
    return seen


def reference(q, k, v, do=None, *, causal=True, offset=0, scale=None, cap=None, slopes=None, documents=None,
              prefix=None, window=None):
    """{name: (value, bound)} for o and, with do, dq, dk, dv, in 64 bits on the
    inputs' device.  The bound of each element is for kernels that round the
    probabilities and the score gradients to the inputs' type before the next
    product (u: half a step of it), and everything else in 32 bits:

    * a score is off by e = (D + 8) 2^-24 sum |q k| scale, in its cap (whose
      argument and value are at most cap) by 2^-20 cap more, in its bias by
      2^-23 of the bias, hence a probability by the factor exp(2 e_row), e_row
      the largest of its row, and by (keys + 16) 2^-24 from the sums;
    * o and dv by u of every term of their sums, and by u of the result; o by as much
      again where the sum that divides it is that of the rounded probabilities: with
      p_j (1 + d_j), |d_j| <= u, and D = sum p_j d_j, |D| <= u,
      sum p_j (1 + d_j) v_j / (1 + D) - o = (sum p_j d_j v_j - D o) / (1 + D);
    * delta = sum dO o by sum |dO| bound(o), and dS by that times P;
    * dq, dk by the same sums over dS.
    """
    f = torch.float64
    b, hq, sq, d = q.shape
    hkv, sk = k.shape[1], k.shape[2]
    bf16 = q.dtype == torch.bfloat16
    u = torch.finfo(q.dtype).eps / 2
    scale = scale if scale else 1.0 / math.sqrt(d)
    qf, kf, vf = q.to(f), k.to(f).repeat_interleave(hq // hkv, 1), v.to(f).repeat_interleave(hq // hkv, 1)
    seen = visible(b, sq, sk, causal=causal, offset=offset, prefix=prefix, window=window,
                   documents=documents)[:, None].to(q.device)
    # hidden keys may hold anything
    some_q, some_k = seen.any(3, keepdim=True).to(q.device), seen.any(2).to(q.device)[..., None]
    qf, kf, vf = (torch.where(t, x, 0.0) for t, x in ((some_q, qf), (some_k, kf), (some_k, vf)))
    s = qf @ kf.transpose(2, 3) * scale
    e = (d + 8) * 2.0**-24 * (qf.abs() @ kf.abs().transpose(2, 3)) * scale
    bent = torch.ones_like(s)
    if cap:
        t = torch.tanh(s / cap)
        s, bent = t * cap, 1 - t * t
        e = e * bent + 2.0**-20 * cap
    if slopes is not None:
        off = offset.view(b, 1, 1).to(q.device) if torch.is_tensor(offset) else offset
        pos = (torch.arange(sq, device=q.device)[None, :, None] + off).clamp(0, max(sk - 1, 0))
        bias = slopes.to(f).view(1, -1, 1, 1) * (pos - torch.arange(sk, device=q.device)).abs()[:, None].to(f)
        s = s - bias
        e = e + 2.0**-23 * bias
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(3, keepdim=True) if sk else s.new_zeros(b, hq, sq, 1)
    p = torch.exp(s - top.masked_fill(top == -math.inf, 0.0))
    total = p.sum(3, keepdim=True)
    p = p / total.masked_fill(total == 0, 1.0)
    o = p @ vf
    row = (2 * (e * seen).amax(3, keepdim=True) if sk else total) + (sk + 16) * 2.0**-24
    o_bound = (u * bf16 + row) * 1.01 * (p @ vf.abs()) + (1.01 * u * bf16 + u) * o.abs()
    out = {"o": (o, o_bound)}
    if do is None:
        return out
    df = torch.where(some_q, do.to(f), 0.0)
    dp = df @ vf.transpose(2, 3)
    delta = (p * dp).sum(3, keepdim=True)
    ds = p * (dp - delta) * bent
    spread = (d + 8) * 2.0**-24 * (df.abs() @ vf.abs().transpose(2, 3))  # of dP
    off_delta = (df.abs() * o_bound).sum(3, keepdim=True) + (d + 8) * 2.0**-24 * (df.abs() * o.abs()).sum(3, keepdim=True)
    # the cap's derivative is off by 2^-20 and by twice the error of tanh, e / cap
    off_bent = 2.0**-20 + (2 * e / cap if cap else 0.0)
    ds_bound = (u * bf16 + 1.01 * row) * ds.abs() + 1.01 * p * bent * (spread + off_delta) \
        + 1.01 * p * (dp - delta).abs() * (off_bent if cap else 0.0)
    # the fp32 sums over keys (queries) of the products
    n = 2.0**-24 * (sq * (hq // hkv) + sk + 16)
    fold = lambda t: t.view(b, hkv, hq // hkv, sk, d).sum(2)  # noqa: E731
    dq, dk, dv = ds @ kf * scale, fold(ds.transpose(2, 3) @ qf) * scale, fold(p.transpose(2, 3) @ df)
    out["dq"] = (dq, (ds_bound + n * ds.abs()) @ kf.abs() * scale + u * dq.abs())
    out["dk"] = (dk, fold((ds_bound + n * ds.abs()).transpose(2, 3) @ qf.abs()) * scale + u * dk.abs())
    out["dv"] = (dv, fold(((u * bf16 + row * 1.01 + n) * p).transpose(2, 3) @ df.abs()) + u * dv.abs())
    return out


def check(name, got, want):
    value, bound = want
    assert got.shape == value.shape, (name, got.shape, value.shape)
    # a bound of zero means the exact value (rows that see nothing); the products of the bound
    # are rounded in 64 bits themselves
    over = (got.double() - value).abs() - bound * 1.01 - 1e-37
    bad = ~(over <= 0)
    assert not bad.any(), (f"{name}: {int(bad.sum())} of {bad.numel()} outside the bound, worst off by "
                           f"{float((got.double() - value).abs()[bad].max()):.3g}, first at {bad.nonzero()[0].tolist()}")
