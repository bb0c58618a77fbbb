"""Operators of models with capped scores, trained on packed documents: what is measured of them.

A decoder whose attention scores and output logits are capped by a tanh, whose
embeddings are scaled, and whose batches hold several documents a row needs

* attention whose scores are capped, get a bias that falls with the distance,
  and are masked by documents, a prefix or a window, forward and backward, and
  for a few new tokens against a long cache of keys (``scored_attention``);
* the loss of the tied LM head with capped logits and a penalty on the
  log-normaliser, forward and backward (``lm_head_cross_entropy``);
* the embedding lookup with scaling and its table gradient (``embedding``).

``run`` computes them in plain torch operations in 32 bits, or, where ``own``
is set, by this library's calls.  ``exact`` gives the same from the
definitions in 64 bits.
"""

from __future__ import annotations

import math

import torch

own = False
DEV = "cuda"
IGNORE = -100
TYPES = {"bf16": torch.bfloat16, "fp32": torch.float32}


# ------------------------------------------------------------------ the cases
def _attn(**kw) -> dict:
    case = dict(kind="attn", dtype="bf16", train=True, causal=True, cap=0.0, slopes=False, docs=0, pad=0.0,
                prefix=0, window=0, ragged=False)
    case.update(kw)
    return case


def listed() -> list[dict]:
    return [
        # one new token of one sequence of 700: the latency of a single-user reply
        _attn(name="token_single", train=False, batch=1, heads=16, kv=16, queries=1, keys=700, dim=64, cap=50.0,
              ragged=True),
        # one new token each of 32 sequences of up to 8,192 tokens, grouped heads of 128
        _attn(name="token_batch", train=False, batch=32, heads=32, kv=8, queries=1, keys=8192, dim=128, cap=50.0,
              ragged=True),
        # five drafted tokens each of six sequences, checked at once against caches with a
        # distance bias and a window
        _attn(name="tokens_window", train=False, batch=6, heads=32, kv=8, queries=5, keys=5001, dim=64,
              slopes=True, window=2048, ragged=True),
        # one layer's attention of the 311M model: 16 x 512 tokens, capped, documents of ~200
        _attn(name="documents_short", batch=16, heads=16, kv=16, queries=512, keys=512, dim=64, cap=50.0, docs=200,
              pad=0.05),
        # the grouped-query configuration with a distance bias in place of rotary embeddings
        _attn(name="distance_gqa", batch=4, heads=32, kv=8, queries=2048, keys=2048, dim=64, slopes=True),
        # long rows of packed documents, grouped heads of 128, capped
        _attn(name="documents_long", batch=1, heads=16, kv=4, queries=8192, keys=8192, dim=128, cap=50.0,
              docs=3000),
        # an encoder-decoder style prefix on a ragged micro-batch at the default widths, fp32
        _attn(name="prefix_fp32", dtype="fp32", batch=3, heads=4, kv=2, queries=333, keys=333, dim=64, cap=20.0,
              slopes=True, prefix=100),
        # the LM head of the default width and vocabulary, 8,192 tokens
        dict(name="head_default", kind="head", dtype="bf16", rows=8192, hidden=768, vocab=50304, cap=30.0, z=1e-4),
        # a short ragged batch against a vocabulary that is no multiple of 8
        dict(name="head_ragged", kind="head", dtype="bf16", rows=709, hidden=1024, vocab=50257, cap=30.0, z=0.0),
        # the smoke configuration's head in fp32
        dict(name="head_fp32", kind="head", dtype="fp32", rows=512, hidden=256, vocab=8192, cap=15.0, z=1e-4),
        # token embedding of 4 x 2048 tokens, frequencies as in text
        dict(name="embed_default", kind="embed", dtype="bf16", tokens=8192, hidden=768, vocab=50304),
        # the smoke configuration's embedding in fp32
        dict(name="embed_fp32", kind="embed", dtype="fp32", tokens=512, hidden=256, vocab=8192),
    ]


def _log_int(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw_scores(rng) -> dict:
    """A way of scoring: a cap, a distance bias, both or neither, and a mask."""
    return dict(cap=rng.choice([0.0, 20.0, 50.0, 50.0, 80.0]), slopes=rng.random() < 0.4,
                window=rng.choice([0, 0, _log_int(rng, 16, 2048)]))


def draw(rng) -> dict:
    kind = rng.choice(["token", "token", "train", "train", "train", "fp32", "head", "head", "embed"])
    if kind == "token":
        kv = rng.choice([1, 2, 4, 8, 16])
        batch, keys = _log_int(rng, 1, 32), _log_int(rng, 1, 8192)
        return _attn(train=False, batch=batch, heads=kv * rng.choice([1, 2, 4, 8]) if kv < 16 else kv, kv=kv,
                     queries=min(keys, rng.choice([1, 1, 1, 2, 5, 16, 40])), keys=keys, dim=rng.choice([64, 128, 80]),
                     ragged=rng.random() < 0.7, **_draw_scores(rng))
    if kind in ("train", "fp32"):
        kv = rng.choice([2, 4, 8])
        bf16 = kind == "train"
        seq = _log_int(rng, 17, 4096 if bf16 else 700)
        batch = max(1, min(16, _log_int(rng, 500, 8192) // seq)) if bf16 else rng.randint(1, 4)
        causal = rng.random() < 0.8
        docs = rng.choice([0, _log_int(rng, 8, 2000)])
        return _attn(dtype="bf16" if bf16 else "fp32", batch=batch, heads=kv * rng.choice([1, 2, 4]), kv=kv,
                     queries=seq, keys=seq, dim=rng.choice([64, 64, 128, 80]), causal=causal, docs=docs,
                     pad=rng.choice([0.0, 0.1]) if docs else 0.0,
                     prefix=_log_int(rng, 1, seq) if causal and rng.random() < 0.3 else 0, **_draw_scores(rng))
    if kind == "head":
        fp32 = rng.random() < 0.25
        return dict(kind="head", dtype="fp32" if fp32 else "bf16", rows=_log_int(rng, 1, 600 if fp32 else 8192),
                    hidden=rng.choice([256, 768] if fp32 else [768, 1024]),
                    vocab=rng.choice([8192, 1001] if fp32 else [8192, 32000, 50257, 50304]),
                    cap=rng.choice([15.0, 30.0, 30.0, 100.0]), z=rng.choice([0.0, 1e-4, 1e-3]))
    return dict(kind="embed", dtype=rng.choice(["bf16", "bf16", "fp32"]), tokens=_log_int(rng, 1, 8192),
                hidden=rng.choice([256, 768, 1024]), vocab=rng.choice([8192, 32000, 50257]))


# --------------------------------------------------------------------- inputs
def _gen(seed: int, stream: int) -> torch.Generator:
    return torch.Generator(device=DEV).manual_seed(1_000_003 * seed + stream)


def _normal(shape, gen, dtype, std: float = 1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * std).to(dtype)


def _zipf(n: int, vocab: int, gen) -> torch.Tensor:
    """Token ids whose frequency falls with their rank, as in text, the ranks spread over the table."""
    rank = torch.exp(torch.rand(n, generator=gen, device=DEV, dtype=torch.float64) * math.log(vocab)) - 1
    return (rank.long().clamp(0, vocab - 1) * 7919) % vocab


def _prepare_attn(case, seed: int) -> dict:
    gen, dtype = _gen(seed, 1), TYPES[case["dtype"]]
    b, h, kv, sq, sk, d = (case[n] for n in ("batch", "heads", "kv", "queries", "keys", "dim"))
    # scores of a few units, tens at most: where a cap of 20 to 50 bends them.  The layout
    # of projections: [batch, tokens, heads, head dim], seen as [batch, heads, tokens, head dim]
    q = _normal((b, sq, h, d), gen, dtype, 4.0).transpose(1, 2)
    k = _normal((b, sk, kv, d), gen, dtype).transpose(1, 2)
    v = _normal((b, sk, kv, d), gen, dtype).transpose(1, 2)
    st = {"case": case, "q": q, "k": k, "v": v, "slopes": None, "documents": None, "prefix": None, "offset": sk - sq}
    if case["slopes"]:
        st["slopes"] = torch.exp2(-8.0 * torch.arange(1, h + 1, device=DEV, dtype=torch.float32) / h)
    if case["docs"]:
        starts = torch.rand(b, sk, generator=gen, device=DEV) < 1.0 / case["docs"]
        ids = torch.cumsum(starts, 1).to(torch.int32)
        # the end of every row is padding: tokens of no document
        ids[:, sk - int(case["pad"] * sk):] = -1
        st["documents"] = ids
    if case["prefix"]:
        st["prefix"] = torch.randint(0, case["prefix"] + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
    if case["ragged"]:
        # every sequence of the batch has its own length; behind it the cache is not filled yet
        st["offset"] = torch.randint((sk - sq) // 2, sk - sq + 1, (b,), generator=gen, device=DEV, dtype=torch.int32)
    if case["train"]:
        st["grad"] = _normal((b, sq, h, d), gen, dtype).transpose(1, 2)
        for name in ("q", "k", "v"):
            st[name].requires_grad_(True)
    return st


def prepare(case, seed: int) -> dict:
    gen, dtype = _gen(seed, 2), TYPES[case.get("dtype", "bf16")]
    if case["kind"] == "attn":
        return _prepare_attn(case, seed)
    if case["kind"] == "head":
        rows, hidden, vocab = case["rows"], case["hidden"], case["vocab"]
        # rms-normalised hidden states against a table of the usual initial spread, a few of
        # its rows grown as frequent tokens' do: logits of up to tens
        x = _normal((rows, hidden), gen, dtype)
        w = torch.randn(vocab, hidden, generator=gen, device=DEV) * 0.05
        w = (w * (1 + 4 * (torch.rand(vocab, 1, generator=gen, device=DEV) < 0.01))).to(dtype)
        t = _zipf(rows, vocab, gen)
        t[torch.rand(rows, generator=gen, device=DEV) < 0.05] = IGNORE  # prompts and padding
        weights = torch.rand(rows, generator=gen, device=DEV) / rows  # the loss weight of every token
        return {"case": case, "x": x.requires_grad_(True), "w": w.requires_grad_(True), "t": t, "weights": weights}
    w = _normal((case["vocab"], case["hidden"]), gen, dtype, 0.02)
    ids = _zipf(case["tokens"], case["vocab"], gen)
    return {"case": case, "w": w.requires_grad_(True), "ids": ids, "scale": math.sqrt(case["hidden"]),
            "grad": _normal((case["tokens"], case["hidden"]), gen, dtype)}


# ---------------------------------------------------------------- plain forms
def _plain_visible(st) -> torch.Tensor:
    """[batch, 1, queries, keys]: which keys a query sees."""
    case = st["case"]
    b, sq, sk = case["batch"], case["queries"], case["keys"]
    off = st["offset"].long()[:, None] if torch.is_tensor(st["offset"]) else st["offset"]
    pos = (torch.arange(sq, device=DEV)[None] + off).expand(b, sq)[:, :, None]
    key = torch.arange(sk, device=DEV)[None, None]
    seen = torch.ones(b, sq, sk, dtype=torch.bool, device=DEV)
    if case["causal"]:
        seen = key <= pos
        if st["prefix"] is not None:
            seen = seen | (key < st["prefix"].long()[:, None, None])
    if case["window"]:
        seen = seen & ((pos - key).abs() < case["window"])
    if st["documents"] is not None:
        ids = st["documents"].long()
        run = torch.cumsum(torch.nn.functional.pad(ids[:, 1:] != ids[:, :-1], (1, 0)), 1)
        run = torch.where(ids < 0, -1, run)
        mine = torch.gather(run, 1, pos[:, :, 0])[:, :, None]
        seen = seen & (mine == run[:, None]) & (mine >= 0)
    return seen.expand(b, sq, sk)[:, None]


def _plain_attn(st):
    case = st["case"]
    b, h, kv, sq, sk, d = (case[n] for n in ("batch", "heads", "kv", "queries", "keys", "dim"))
    dtype, scale = TYPES[case["dtype"]], 1.0 / math.sqrt(d)
    q, k, v = (st[n].detach().float() for n in ("q", "k", "v"))
    k, v = (t.repeat_interleave(h // kv, 1) for t in (k, v))
    s = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    bend = None
    if case["cap"]:
        bend = torch.tanh(s / case["cap"])
        s = bend * case["cap"]
    if st["slopes"] is not None:
        off = st["offset"][:, None, None].float() if torch.is_tensor(st["offset"]) else float(st["offset"])
        pos = torch.arange(sq, device=DEV, dtype=torch.float32)[None, :, None] + off
        far = (pos - torch.arange(sk, device=DEV, dtype=torch.float32)[None, None]).abs()
        s = s - st["slopes"][None, :, None, None] * far[:, None]
    s = torch.where(_plain_visible(st), s, -math.inf)
    top = s.amax(3, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(3, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = torch.matmul(p, v)
    if not case["train"]:
        return out.to(dtype)
    do = st["grad"].float()
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dp = torch.matmul(do, v.transpose(2, 3).contiguous())
    ds = p * (dp - (p * dp).sum(3, keepdim=True)) * scale
    if bend is not None:
        ds = ds * (1 - bend * bend)
    dq = torch.matmul(ds, k)
    dk = torch.matmul(ds.transpose(2, 3).contiguous(), q)
    dk, dv = (t.view(b, kv, h // kv, sk, d).sum(2) for t in (dk, dv))
    return tuple(t.to(dtype) for t in (out, dq, dk, dv))


def _plain_head(st):
    case, dtype = st["case"], TYPES[st["case"]["dtype"]]
    x, w, t = st["x"].detach().float(), st["w"].detach().float(), st["t"]
    bend = torch.tanh(torch.matmul(x, w.t()) / case["cap"])
    z = bend * case["cap"]
    top = z.amax(1, keepdim=True)
    e = torch.exp(z - top)
    total = e.sum(1, keepdim=True)
    lse = (top + torch.log(total))[:, 0]
    used = t != IGNORE
    at = torch.where(used, t, 0)[:, None]
    loss = torch.where(used, lse - torch.gather(z, 1, at)[:, 0] + case["z"] * lse * lse, 0.0)
    g = e / total * (1 + 2 * case["z"] * lse[:, None])
    g.scatter_add_(1, at, torch.full_like(g[:, :1], -1.0))
    g = g * (1 - bend * bend) * torch.where(used, st["weights"], 0.0)[:, None]
    return loss, torch.matmul(g, w).to(dtype), torch.matmul(g.t().contiguous(), x).to(dtype)


def _plain_embed(st):
    case, dtype = st["case"], TYPES[st["case"]["dtype"]]
    out = (st["w"].detach()[st["ids"]].float() * st["scale"]).to(dtype)
    # sums of many rows of one token, whose order torch's addition leaves open: 64 bits
    dw = torch.zeros(case["vocab"], case["hidden"], dtype=torch.float64, device=DEV)
    dw.index_add_(0, st["ids"], st["grad"].double())
    return out, (dw * st["scale"]).to(dtype)


# ------------------------------------------------------------ the library's own
def _own(st):
    from nano_megatron_amd import functional as Fn

    case = st["case"]
    if case["kind"] == "attn":
        out = Fn.scored_attention(st["q"], st["k"], st["v"], causal=case["causal"], sequence_offset=st["offset"],
                                  score_cap=case["cap"] or None, distance_slopes=st["slopes"],
                                  documents=st["documents"], prefix=st["prefix"], window=case["window"] or None)
        if not case["train"]:
            return out
        return (out.detach(), *torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["grad"]))
    if case["kind"] == "head":
        # the data loader has checked the targets
        loss = Fn.lm_head_cross_entropy(st["x"], st["w"], st["t"], ignore_index=IGNORE, reduction="none",
                                        validate=False, logit_cap=case["cap"], z_loss=case["z"])
        return (loss.detach(), *torch.autograd.grad(loss, (st["x"], st["w"]), st["weights"]))
    out = Fn.embedding(st["w"], st["ids"], scale=st["scale"])
    return (out.detach(), *torch.autograd.grad(out, (st["w"],), st["grad"]))


def run(st):
    if own:
        return _own(st)
    return {"attn": _plain_attn, "head": _plain_head, "embed": _plain_embed}[st["case"]["kind"]](st)


# ------------------------------------------------------------------ 64 bits
def _exact_attn(case, st):
    """Head by head by autograd in 64 bits; visibility by comparing every pair of tokens."""
    b, h, kv, sq, sk, d = (case[n] for n in ("batch", "heads", "kv", "queries", "keys", "dim"))
    leaves = [st[n].detach().double().requires_grad_(case["train"]) for n in ("q", "k", "v")]
    grads = [torch.zeros_like(t) for t in leaves]
    out = torch.empty_like(leaves[0], requires_grad=False)
    for i in range(b):
        off = int(st["offset"][i]) if torch.is_tensor(st["offset"]) else st["offset"]
        far = (torch.arange(off, off + sq, device=DEV)[:, None] - torch.arange(sk, device=DEV)[None])
        hidden = torch.zeros(sq, sk, dtype=torch.bool, device=DEV)
        if case["causal"]:
            hidden |= far < 0
            if st["prefix"] is not None:
                hidden[:, :int(st["prefix"][i])] = False
        if case["window"]:
            hidden |= far.abs() >= case["window"]
        if st["documents"] is not None:
            ids = st["documents"][i].tolist()
            first = list(range(sk))  # where the document of each token starts
            for j in range(1, sk):
                if ids[j] == ids[j - 1]:
                    first[j] = first[j - 1]
            first = torch.tensor([f if ids[j] >= 0 else -1 - j for j, f in enumerate(first)], device=DEV)
            hidden |= first[off:off + sq, None] != first[None]
            hidden |= (first[off:off + sq] < 0)[:, None]
        for j in range(h):
            q, k, v = leaves[0][i, j], leaves[1][i, j * kv // h], leaves[2][i, j * kv // h]
            s = (q @ k.t()) / math.sqrt(d)
            if case["cap"]:
                s = case["cap"] * torch.tanh(s / case["cap"])
            if st["slopes"] is not None:
                s = s - st["slopes"][j].double() * far.abs()
            s = s.masked_fill(hidden, -1e300)
            e = torch.exp(s - s.detach().amax(1, keepdim=True)).masked_fill(hidden, 0.0)
            o = (e / e.sum(1, keepdim=True).clamp_min(1e-300)) @ v
            out[i, j] = o.detach()
            if case["train"]:
                for g, t in zip(grads, torch.autograd.grad(o, leaves, st["grad"][i, j].double())):
                    g += t
    return (out, *grads) if case["train"] else out


def exact(case, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "attn":
        b, h, sq, sk = (case[n] for n in ("batch", "heads", "queries", "keys"))
        if case["train"] and b * h * (case["dim"] + 8) * sq * sk > 4e11:  # over about 20 seconds
            return None
        return _exact_attn(case, st)
    if case["kind"] == "head":
        x, w = (st[n].detach().double().requires_grad_(True) for n in ("x", "w"))
        z = case["cap"] * torch.tanh(x @ w.t() / case["cap"])
        lse = torch.logsumexp(z, 1)
        used = st["t"] != IGNORE
        picked = z[torch.arange(case["rows"], device=DEV), st["t"].clamp_min(0)]
        loss = (lse - picked + case["z"] * lse ** 2) * used
        return (loss.detach(), *torch.autograd.grad(loss, (x, w), st["weights"].double()))
    w = st["w"].detach().double()
    order = torch.argsort(st["ids"], stable=True)
    ids, rows = torch.unique_consecutive(st["ids"][order], return_counts=True)
    sums = torch.cumsum(st["grad"].double()[order], 0)[torch.cumsum(rows, 0) - 1]
    dw = torch.zeros_like(w)
    dw[ids] = torch.diff(sums, dim=0, prepend=torch.zeros_like(sums[:1])) * st["scale"]
    return w[st["ids"]] * st["scale"], dw


# -------------------------------------------------------------------- the work
def work(case) -> dict:
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "attn":
        b, h, kv, sq, sk, d = (case[n] for n in ("batch", "heads", "kv", "queries", "keys", "dim"))
        # keys that a query sees, and keys that any query sees, of the average row
        reach = 0.75 * sk if case["ragged"] else sk
        seen = reach if sq < sk or not case["causal"] else (reach + 1) / 2
        if case["docs"]:
            seen = min(seen, case["docs"] * (1 if case["causal"] else 2)) * (1 - case["pad"])
        if case["prefix"]:
            seen = min(reach, seen + case["prefix"] ** 2 / 4 / sk)
        if case["window"]:
            seen = min(seen, case["window"] * (1 if case["causal"] else 2))
        keys = min(reach, seen + sq) if sq < sk else sk
        rows_q, rows_k = b * sq * h * d, b * keys * kv * d
        # products: two forward; backward the scores again, dP, dV, dQ and dK
        return {"bytes": size * (rows_q * (4 if case["train"] else 2) + rows_k * (4 if case["train"] else 2)),
                "flops": 2.0 * b * h * sq * seen * d * (7 if case["train"] else 2)}
    if case["kind"] == "head":
        r, h, v = case["rows"], case["hidden"], case["vocab"]
        # logits, and the two gradients from them
        return {"bytes": size * 2 * (r * h + v * h) + 16 * r, "flops": 6.0 * r * h * v}
    n, h, v = case["tokens"], case["hidden"], case["vocab"]
    return {"bytes": size * (3 * n * h + v * h) + 8 * n, "flops": 2.0 * n * h}
