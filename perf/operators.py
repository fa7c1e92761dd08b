"""Operators of a training step on packed documents, as measurable cases: attention over packed sequences of different
lengths with grouped heads, the loss over a large vocabulary computed in pieces of it, and the global gradient norm with
clipping.  Each in its plain form (elementary torch operations in 32 bits) and through the framework's entry points.

Kinds of a case:

* ``attention``: causal attention of packed sequences, with a window where one is given, and its gradients.
* ``loss``: per-token cross entropy of a (soft-capped) linear head, and the gradients of its inputs and weights.
* ``clip``: the norm of all gradients together, and the gradients scaled to a largest norm (into other buffers, so that
  every pass finds the same gradients).
"""
from __future__ import annotations

import math
import random

import torch

own = False
DEVICE = "cuda"


def _texts(lengths):
    return ",".join(str(n) for n in lengths)


def _documents(rng, total, lo, hi):
    """Lengths of documents, spread over the logarithm, that fill `total` tokens."""
    got = []
    while sum(got) < total:
        got.append(min(total - sum(got), int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))
    return got


def _attention(name, lengths, heads, kv_heads, dim, window=0, pad=0, grad=True):
    c = dict(kind="attention", lengths=_texts(lengths), heads=heads, kv_heads=kv_heads, dim=dim, window=window, pad=pad, grad=grad)
    return dict(c, name=name) if name else c


def _loss(name, tokens, dim, vocab, softcap, ignored=0.0, grad=True):
    c = dict(kind="loss", tokens=tokens, dim=dim, vocab=vocab, softcap=softcap, ignored=ignored, grad=grad)
    return dict(c, name=name) if name else c


def _clip(name, dim, layers, vocab, dtype, out, ratio):
    """ratio: how far the gradients exceed the largest norm; 0 asks for the norm alone."""
    c = dict(kind="clip", dim=dim, layers=layers, vocab=vocab, dtype=dtype, out=out, ratio=ratio)
    return dict(c, name=name) if name else c


def listed():
    rng = random.Random(11)
    return [
        # --- the `small` preset's row of 512 tokens that holds four documents: launches and host time count
        _attention("attention small 4 documents in 512", [1, 130, 77, 304], 2, 2, 128),
        # --- rows of the 119.5 M model (4 heads, context 2048) packed with documents of 32 to 2048 tokens
        _attention("attention 4 heads documents in 16384", _documents(rng, 16384, 32, 2048), 4, 4, 128),
        # --- long documents under a sliding window of 256, the short window of every preset; grouped heads
        _attention("attention 8/4 heads window 256 32768", _documents(rng, 32768, 512, 8192), 8, 4, 128, window=256),
        # --- a whole prompt of 32768 tokens scored at once, 16 heads on two key heads
        _attention("attention 16/2 heads prompt 32768", [32768], 16, 2, 128, grad=False),
        # --- odd: three query heads a key head, heads of 64, odd lengths, rows behind the last sequence
        _attention("attention 9/3 heads of 64 odd", _documents(rng, 7001, 3, 1999), 9, 3, 64, pad=191),
        # --- the `small` preset's loss: 512 tokens, 1024 ids
        _loss("loss small 512 x 1024 ids", 512, 256, 1024, 15.0),
        # --- a vocabulary that is no multiple of anything, a tenth of the tokens not counted, no soft cap
        _loss("loss odd 4099 x 50021 ids", 4099, 384, 50021, 0.0, ignored=0.1),
        # --- a training micro-step with a large vocabulary, and the scoring pass of an evaluation
        _loss("loss 16384 x 65536 ids", 16384, 1024, 65536, 15.0),
        _loss("loss scoring 16384 x 131072 ids", 16384, 1024, 131072, 15.0, grad=False),
        # --- gradients of the `small` preset; of the 119.5 M model, clipped into bf16 buckets for the exchange; of a wide one
        _clip("clip small fp32", 256, 4, 1024, "float32", "float32", 3.0),
        _clip("clip 119M fp32 to bf16", 512, 30, 8191, "float32", "bfloat16", 2.5),
        _clip("norm wide bf16", 2048, 16, 8192, "bfloat16", "", 0.0),
    ]


# ------------------------------------------------------------------------------------------------
def _log(rng, lo, hi):
    return int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))


def draw(rng):
    """Rows of 64 to 32768 tokens in documents of any length, 1 to 16 heads in groups of 1 to 8; 64 to 32768 tokens against
    64 to 131072 ids; gradients of 1 to 30 layers of width 128 to 2048."""
    top = {}
    for c in listed():
        w = work(c)
        k = c["kind"]
        top[k] = (max(top.get(k, (0, 0))[0], w["bytes"]), max(top.get(k, (0, 0))[1], w["flops"]))
    while True:
        kind = rng.choice(["attention", "attention", "loss", "loss", "clip"])
        if kind == "attention":
            total = _log(rng, 64, 32768)
            group, kv = rng.choice([1, 1, 2, 3, 4, 5, 8]), rng.choice([1, 2, 3, 4, 6])
            lo = _log(rng, 1, max(1, total // 8))
            lengths = _documents(rng, total, lo, rng.randint(lo, total))
            if rng.random() < 0.2:
                lengths.insert(rng.randrange(len(lengths) + 1), 0)       # a slot of the row that holds no document
            if len(lengths) * max(lengths) ** 2 * group > 6e9:      # the padded plain form has to fit
                continue
            c = _attention(None, lengths, group * kv, kv, rng.choice([64, 128, 128]), rng.choice([0, 0, 0, 256, rng.randint(1, total)]),
                           rng.choice([0, 0, rng.randint(1, 300)]), rng.random() < 0.7)
            if group * kv > 16:
                continue
        elif kind == "loss":
            c = _loss(None, _log(rng, 64, 32768), 8 * _log(rng, 8, 256), _log(rng, 64, 131072), rng.choice([0.0, 15.0, 15.0, 30.0]),
                      rng.choice([0.0, 0.0, 0.3]), rng.random() < 0.7)
            if c["tokens"] * c["vocab"] > 2.2e9:
                continue
        else:
            dtype = rng.choice(["float32", "float32", "bfloat16", "float16", "mixed"])
            c = _clip(None, 8 * _log(rng, 16, 256), rng.randint(1, 30), _log(rng, 256, 16384), dtype,
                      rng.choice(["float32", "bfloat16", "same"]), rng.choice([0.0, 0.5, 2.0, 10.0]))
        w = work(c)
        if w["bytes"] <= top[kind][0] and w["flops"] <= top[kind][1]:
            return c


# ------------------------------------------------------------------------------------------------
def _lengths(case):
    return [int(n) for n in case["lengths"].split(",")]


def _shapes(case):
    """Gradients of a model: embeddings and head, per-layer scalars, per layer the projections, the MLP and a small gate."""
    D, V, L = case["dim"], case["vocab"], case["layers"]
    shapes = [(V, D), (V, D), (L,), (L,)]
    for l in range(L):
        shapes += [(3 * D, D), (D, D), (4 * D, D), (D, 4 * D)] + ([(D // 128 + 1, 32)] if l % 2 else [])
    return shapes


def _flat_views(shapes, dtypes, fill):
    """One buffer per type and the tensors as views into it, back to back."""
    sizes = {}
    for s, t in zip(shapes, dtypes):
        sizes[t] = sizes.get(t, 0) + math.prod(s)
    bufs = {t: fill(n, t) for t, n in sizes.items()}
    at, views = dict.fromkeys(sizes, 0), []
    for s, t in zip(shapes, dtypes):
        n = math.prod(s)
        views.append(bufs[t][at[t]:at[t] + n].view(s))
        at[t] += n
    return bufs, views


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device=DEVICE, dtype=torch.float32) * std).to(dtype)

    kind = case["kind"]
    if kind == "attention":
        lengths, H, KV, d = _lengths(case), case["heads"], case["kv_heads"], case["dim"]
        rows = sum(lengths) + case["pad"]
        # column blocks of the packed projection output; queries and keys of unit RMS, as after their norm
        qkv = normal(rows, H + 2 * KV, d)
        q, k, v = (t.detach().requires_grad_(case["grad"]) for t in (qkv[:, :H], qkv[:, H:H + KV], qkv[:, H + KV:]))
        ends = [0]
        for n in lengths:
            ends.append(ends[-1] + n)
        cu = torch.tensor(ends, dtype=torch.int32, device=DEVICE)
        st = dict(kind=kind, q=q, k=k, v=v, cu=cu, lengths=lengths, window=case["window"] or None, d_out=normal(rows, H, d, std=0.1),
                  grad=case["grad"])
        if own:
            # the tile lists of this packing, which every layer of a model uses in both directions
            from autoresearch_b200.ops.packed import PackedSequences
            st["seqs"] = PackedSequences(cu, rows, H, KV)
        return st
    if kind == "loss":
        N, D, V = case["tokens"], case["dim"], case["vocab"]
        x = normal(N, D)
        w = normal(V, D, std=2.5 / math.sqrt(D))
        # Zipf-like ids: log-uniform over the vocabulary
        u = torch.rand(N, generator=g, device=DEVICE)
        targets = (torch.exp(u * math.log(V)) - 1).long().clamp(0, V - 1)
        drop = torch.rand(N, generator=g, device=DEVICE) < case["ignored"]
        targets = torch.where(drop, torch.full_like(targets, -100), targets)
        weight = (0.5 + torch.rand(N, generator=g, device=DEVICE)) / N
        x.requires_grad_(case["grad"])
        w.requires_grad_(case["grad"])
        return dict(kind=kind, x=x, w=w, targets=targets, softcap=case["softcap"], weight=weight, grad=case["grad"])
    shapes = _shapes(case)
    half = torch.bfloat16 if case["dtype"] == "mixed" else getattr(torch, case["dtype"])
    dtypes = [torch.float32 if case["dtype"] == "mixed" and i % 3 == 0 else half for i in range(len(shapes))]
    bufs, grads = _flat_views(shapes, dtypes, lambda n, t: torch.empty(n, dtype=t, device=DEVICE))
    for i, t in enumerate(grads):
        t.normal_(0.0, 1e-3 * (1 + i % 5), generator=g)
    outs, out_bufs = None, {}
    if case["ratio"] and case["out"]:
        to = dtypes if case["out"] == "same" else [getattr(torch, case["out"])] * len(shapes)
        out_bufs, outs = _flat_views(shapes, to, lambda n, t: torch.zeros(n, dtype=t, device=DEVICE))
    # the expected norm, from the distribution that the gradients were drawn from
    norm = math.sqrt(sum(math.prod(s) * (1e-3 * (1 + i % 5)) ** 2 for i, s in enumerate(shapes)))
    return dict(kind=kind, grads=grads, outs=outs, out_bufs=out_bufs, max_norm=norm / case["ratio"] if case["ratio"] else None)


# ------------------------------------------------------------------------------------------------
def _plain_attention(st):
    """Sequences padded to the longest; the query heads of one key head at a time, since all scores are kept."""
    q, k, v, cu = st["q"].detach(), st["k"].detach(), st["v"].detach(), st["cu"]
    rows, H, d = q.shape
    KV, L = k.shape[1], max(st["lengths"])
    G = H // KV
    scale = 1.0 / math.sqrt(d)
    ar = torch.arange(L, device=q.device)
    valid = ar < (cu[1:] - cu[:-1])[:, None]
    idx = torch.where(valid, cu[:-1, None] + ar, 0).long()
    real = idx[valid]
    ahead = ar[:, None] - ar[None, :]
    hidden = (ahead < 0) | (ahead > (st["window"] if st["window"] is not None else L))
    out = torch.zeros_like(q)
    if st["grad"]:
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    for h in range(KV):
        qs = q[:, h * G:(h + 1) * G].float()[idx].transpose(1, 2).contiguous()      # [n, G, L, d]
        ks, vs = k[:, h].float()[idx][:, None], v[:, h].float()[idx][:, None]       # [n, 1, L, d]
        p = torch.matmul(qs, ks.transpose(-1, -2)).mul_(scale).masked_fill_(hidden, float("-inf"))
        p.sub_(p.amax(-1, keepdim=True)).exp_()
        p.div_(p.sum(-1, keepdim=True))
        o = torch.matmul(p, vs)
        out[real, h * G:(h + 1) * G] = o.transpose(1, 2)[valid].to(out.dtype)
        if st["grad"]:
            do = st["d_out"][:, h * G:(h + 1) * G].float()[idx].masked_fill(~valid[:, :, None, None], 0.0).transpose(1, 2).contiguous()
            dv[real, h] = torch.matmul(p.transpose(-1, -2), do).sum(1)[valid].to(dv.dtype)
            ds = torch.matmul(do, vs.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p)
            dq[real, h * G:(h + 1) * G] = (torch.matmul(ds, ks) * scale).transpose(1, 2)[valid].to(dq.dtype)
            dk[real, h] = (torch.matmul(ds.transpose(-1, -2), qs).sum(1) * scale)[valid].to(dk.dtype)
    return dict(out=out, dq=dq, dk=dk, dv=dv) if st["grad"] else dict(out=out)


def _plain_loss(st):
    x, w, t, cap = st["x"].detach().float(), st["w"].detach().float(), st["targets"], st["softcap"]
    s = x @ w.t()
    if cap:
        s = s.div_(cap).tanh_().mul_(cap)
    m = s.amax(-1, keepdim=True)
    lse = (s - m).exp_().sum(-1, keepdim=True).log_() + m
    counts = (t >= 0) & (t < w.shape[0])
    at = torch.where(counts, t, 0)[:, None]
    losses = torch.where(counts, (lse - s.gather(1, at))[:, 0], 0.0)
    if not st["grad"]:
        return dict(losses=losses)
    slope = (s / cap).square_().neg_().add_(1.0) if cap else None
    d = s.sub_(lse).exp_()
    d.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    d.mul_(torch.where(counts, st["weight"], 0.0)[:, None])
    if cap:
        d.mul_(slope)
    return dict(losses=losses, dx=(d @ w).to(st["x"].dtype), dw=(d.t() @ x).to(st["w"].dtype))


def _plain_clip(st):
    norm = torch.stack([t.float().square().sum(dtype=torch.float64) for t in st["grads"]]).sum().sqrt()
    if st["max_norm"] is None:
        return dict(norm=norm.float())
    scale = (st["max_norm"] / norm).clamp(max=1.0).float()
    for t, o in zip(st["grads"], st["outs"]):
        o.copy_(t.float() * scale)
    return dict(norm=norm.float(), clipped=st["out_bufs"])


def _own(st):
    if st["kind"] == "attention":
        from autoresearch_b200.ops.packed import packed_attention
        out = packed_attention(st["q"], st["k"], st["v"], st["seqs"], window=st["window"])
        if not st["grad"]:
            return dict(out=out)
        dq, dk, dv = torch.autograd.grad(out, (st["q"], st["k"], st["v"]), st["d_out"])
        return dict(out=out.detach(), dq=dq, dk=dk, dv=dv)
    if st["kind"] == "loss":
        from autoresearch_b200.ops.linear_ce import linear_cross_entropy
        losses = linear_cross_entropy(st["x"], st["w"], st["targets"], softcap=st["softcap"])
        if not st["grad"]:
            return dict(losses=losses)
        dx, dw = torch.autograd.grad(losses, (st["x"], st["w"]), st["weight"])
        return dict(losses=losses.detach(), dx=dx, dw=dw)
    from autoresearch_b200.optim.clip import clip_grad_norm, grad_norm
    if st["max_norm"] is None:
        return dict(norm=grad_norm(st["grads"]))
    return dict(norm=clip_grad_norm(st["grads"], st["max_norm"], out=st["outs"]), clipped=st["out_bufs"])


def run(state):
    if own:
        return _own(state)
    return {"attention": _plain_attention, "loss": _plain_loss, "clip": _plain_clip}[state["kind"]](state)


# ------------------------------------------------------------------------------------------------
def work(case):
    kind = case["kind"]
    if kind == "attention":
        H, KV, d = case["heads"], case["kv_heads"], case["dim"]
        lengths = _lengths(case)
        w = case["window"] or sum(lengths)
        pairs = sum(n * (n + 1) // 2 if n <= w + 1 else (w + 1) * (w + 2) // 2 + (n - w - 1) * (w + 1) for n in lengths)
        n = sum(lengths)
        one, kv = 2 * n * H * d, 2 * n * KV * d
        # forward: q, k, v, out and two products; backward: d_out as well, dq, dk, dv and five products
        if not case["grad"]:
            return {"bytes": 2 * one + 2 * kv, "flops": 4.0 * pairs * H * d}
        return {"bytes": 4 * one + 4 * kv, "flops": 14.0 * pairs * H * d}
    if kind == "loss":
        N, D, V = case["tokens"], case["dim"], case["vocab"]
        by = 2 * (N + V) * D + 12 * N
        return {"bytes": 2 * by if case["grad"] else by, "flops": (6.0 if case["grad"] else 2.0) * N * D * V}
    size = {"float32": 4.0, "bfloat16": 2.0, "float16": 2.0, "mixed": 8 / 3}
    n = sum(math.prod(s) for s in _shapes(case))
    read = size[case["dtype"]] * n
    if not case["ratio"]:
        return {"bytes": read, "flops": 2.0 * n}
    # the scale is known once every gradient has been read: they are read again to be scaled
    return {"bytes": 2 * read + (read if case["out"] == "same" else size[case["out"]] * n), "flops": 3.0 * n}


# ------------------------------------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"attention": _exact_attention, "loss": _exact_loss, "clip": _exact_clip}[case["kind"]](st)


def _exact_attention(st):
    """Sequence by sequence and head by head, from the definition."""
    q, k, v = (st[n].detach().double() for n in "qkv")
    rows, H, d = q.shape
    G = H // k.shape[1]
    do = st["d_out"].double()
    out, dq, dk, dv = (torch.zeros_like(t) for t in (q, q, k, v))
    at = 0
    for n in st["lengths"]:
        i = torch.arange(n, device=q.device)
        seen = i[None, :] <= i[:, None]
        if st["window"] is not None:
            seen &= i[None, :] >= i[:, None] - st["window"]
        sl = slice(at, at + n)
        for h in range(H):
            kv = h // G
            s = (q[sl, h] @ k[sl, kv].T) / math.sqrt(d)
            p = torch.softmax(torch.where(seen, s, -math.inf), dim=1)
            out[sl, h] = p @ v[sl, kv]
            if st["grad"]:
                dp = do[sl, h] @ v[sl, kv].T
                ds = p * (dp - (p * dp).sum(1, keepdim=True)) / math.sqrt(d)
                dq[sl, h] = ds @ k[sl, kv]
                dk[sl, kv] += ds.T @ q[sl, h]
                dv[sl, kv] += p.T @ do[sl, h]
        at += n
    return dict(out=out, dq=dq, dk=dk, dv=dv) if st["grad"] else dict(out=out)


def _exact_loss(st):
    """Some rows at a time, since a row of 64-bit logits is as long as the vocabulary."""
    x, w, t = st["x"].detach().double(), st["w"].detach().double(), st["targets"]
    cap, V = st["softcap"], w.shape[0]
    losses = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
    dx, dw = torch.zeros_like(x), torch.zeros_like(w)
    step = max(1, (1 << 28) // V)
    for a in range(0, x.shape[0], step):
        xs, ts = x[a:a + step], t[a:a + step]
        z = xs @ w.T
        s = cap * torch.tanh(z / cap) if cap else z
        hot = ts[:, None] == torch.arange(V, device=x.device)[None, :]
        counted = hot.any(1)
        losses[a:a + step] = torch.where(counted, torch.logsumexp(s, 1) - (s * hot).sum(1), 0.0)
        if st["grad"]:
            d = (torch.softmax(s, 1) - hot.double()) * (st["weight"][a:a + step].double() * counted)[:, None]
            if cap:
                d = d * (1 - torch.tanh(z / cap) ** 2)
            dx[a:a + step] = d @ w
            dw += d.T @ xs
    return dict(losses=losses, dx=dx, dw=dw) if st["grad"] else dict(losses=losses)


def _exact_clip(st):
    norm = math.sqrt(math.fsum(float((t.double() ** 2).sum()) for t in st["grads"]))
    if st["max_norm"] is None:
        return dict(norm=norm)
    c = min(1.0, st["max_norm"] / norm)
    bufs = {}
    for t, o in zip(st["grads"], st["outs"]):
        bufs.setdefault(o.dtype, []).append((t.double() * c).reshape(-1))
    return dict(norm=norm, clipped={t: torch.cat(b) for t, b in bufs.items()})
