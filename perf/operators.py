"""Performance cases of the language-model operators: token embedding with its
gradient by sorted tokens, multi-head attention that keeps no probabilities
(forward, backward, one query over a cache), and a Linear with softmax
cross-entropy that keeps no logits.

Everything is fp32 (the framework's only floating type).  Tensors follow the
framework's ColMajor layout: a [rows, cols] matrix is a torch tensor of shape
(cols, rows), so `t.T` is the logical matrix.  A sequence [B, S, F] is a
[B*S, F] matrix whose rows are in the reference order (row b + B*s) or by
sample (row s + S*b); token ids are ColMajor [B, S] in both.

`own` chooses what run() does: the framework's operators, or their plain form
in elementary torch operations.
"""
import math

import torch

own = False

REF, BY_SAMPLE = 0, 1


# ------------------------------------------------------------------ helpers
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 6151 + 29)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _empty(*shape):
    return torch.empty(shape, device="cuda")


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi], odd ones among them."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _tokens(g, n, vocab, zipf, padded):
    """n token ids: uniform, or with the frequencies of text (the k-th most
    frequent id about 1/k as often as the first); `padded` of 16 are -1."""
    u = torch.rand(n, generator=g, device="cuda", dtype=torch.float64)
    ids = torch.floor(torch.exp(u * math.log(vocab + 1)) - 1) if zipf else torch.floor(u * vocab)
    ids = ids.clamp(0, vocab - 1).to(torch.int32)
    if zipf:  # frequent ids lie anywhere in the table
        perm = torch.randperm(vocab, generator=g, device="cuda").to(torch.int32)
        ids = perm[ids.long()]
    if padded:
        ids[torch.randint(0, 16, (n,), generator=g, device="cuda") < padded] = -1
    return ids


def _rows_of_ids(c, ids):
    """The ids in the order of the sequence's rows."""
    return ids if c["rows"] == REF else ids.view(c["steps"], c["batch"]).t().reshape(-1)


# --------------------------------------------------------- token embedding
def _emb_prepare(c, g):
    B, S, V, D = c["batch"], c["steps"], c["vocab"], c["dim"]
    s = {"ids": _tokens(g, B * S, V, c["zipf"], c["padded"]), "Wt": _randn(g, V, D) / math.sqrt(D),
         "out": _empty(D, B * S)}
    if c["train"]:
        s.update(dY=_randn(g, D, B * S) / (B * S), gWt=_empty(V, D))
    return s


def _emb_forward(c, ids, Wt, scale):
    p = _rows_of_ids(c, ids).long()
    held = (p >= 0) & (p < c["vocab"])
    return (Wt[p.clamp(0, c["vocab"] - 1)] * (scale * held)[:, None]).t().contiguous()


def _emb_backward(c, ids, dY, scale, into):
    p = _rows_of_ids(c, ids).long()
    held = (p >= 0) & (p < c["vocab"])
    return into.index_add_(0, p.clamp(0, c["vocab"] - 1), (dY * (scale * held)).t())


def _emb_run(c, s):
    B, S, V, D = c["batch"], c["steps"], c["vocab"], c["dim"]
    scale = math.sqrt(D)
    if own:
        from cppnet_amd import ops
        ops.token_embedding_forward(s["ids"], s["Wt"], s["out"], B, S, V, D, scale=scale, rows=c["rows"])
        if not c["train"]:
            return [s["out"]]
        ops.token_embedding_backward(s["ids"], s["dY"], s["gWt"], B, S, V, D, scale=scale, rows=c["rows"])
        return [s["out"], s["gWt"]]
    out = _emb_forward(c, s["ids"], s["Wt"], scale)
    if not c["train"]:
        return [out]
    return [out, _emb_backward(c, s["ids"], s["dY"], scale, torch.zeros_like(s["Wt"]))]


def _emb_exact(c, s):
    W = s["Wt"].double().requires_grad_(True)
    p = _rows_of_ids(c, s["ids"]).long()
    padded = torch.cat([W, W.new_zeros(1, c["dim"])])  # ids outside the table read a row of zeros
    p = torch.where((p >= 0) & (p < c["vocab"]), p, torch.full_like(p, c["vocab"]))
    out = padded[p].t() * math.sqrt(c["dim"])
    if not c["train"]:
        return [out.detach()]
    return [out.detach(), torch.autograd.grad(out, W, s["dY"].double())[0]]


def _emb_work(c):
    N, V, D = c["batch"] * c["steps"], c["vocab"], c["dim"]
    used = min(N, V)  # rows of the table that are read at most
    if not c["train"]:
        return {"bytes": 4 * (N + used * D + N * D), "flops": N * D}
    return {"bytes": 4 * (2 * N + used * D + 2 * N * D + V * D), "flops": 3 * N * D}


# --------------------------------------------------------------- attention
def _lengths(c):
    """Keys of each sample: all of them, or lengths of a ragged batch."""
    B, Sk = c["batch"], c["keys"]
    if not c["ragged"]:
        return [Sk] * B
    return [max(1, Sk - (b * 7919 + 13) % (Sk // 2 + 1)) for b in range(B)]


def _starts(c):
    """The position of each sample's first query among the keys."""
    if c["decode"]:
        return [n - c["queries"] for n in _lengths(c)]
    return [c["keys"] - c["queries"]] * c["batch"]


def _att_prepare(c, g):
    B, Sq, Sk, H, KH, dh = (c[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    s = {"q": _randn(g, H * dh, B * Sq), "k": _randn(g, KH * dh, B * Sk), "v": _randn(g, KH * dh, B * Sk),
         "out": _empty(H * dh, B * Sq), "lse": _empty(H, B * Sq)}
    s["k_len"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
    s["q_start"] = torch.tensor(_starts(c), dtype=torch.int32, device="cuda") if c["decode"] else None
    if c["train"]:
        s.update(dout=_randn(g, H * dh, B * Sq), dq=_empty(H * dh, B * Sq), dk=_empty(KH * dh, B * Sk),
                 dv=_empty(KH * dh, B * Sk))
    return s


def _heads(c, t, heads, steps):
    """(heads*dh, B*steps) storage -> [B, heads, steps, dh]."""
    B, dh = c["batch"], c["head_dim"]
    if c["rows"] == REF:
        return t.view(heads, dh, steps, B).permute(3, 0, 2, 1)
    return t.view(heads, dh, B, steps).permute(2, 0, 3, 1)


def _stored(c, t):
    """[B, heads, steps, dh] -> (heads*dh, B*steps) storage."""
    B, heads, steps, dh = t.shape
    order = (1, 3, 2, 0) if c["rows"] == REF else (1, 3, 0, 2)
    return t.permute(order).reshape(heads * dh, B * steps)


def _allowed(c, s, device):
    """[B, 1, Sq, Sk]: whether a query reads a key."""
    B, Sq, Sk = c["batch"], c["queries"], c["keys"]
    j = torch.arange(Sk, device=device)
    n = s["k_len"].long() if c["ragged"] else torch.full((B,), Sk, device=device)
    ok = (j[None, None, :] < n[:, None, None]).expand(B, Sq, Sk)
    if c["causal"]:
        first = s["q_start"].long() if c["decode"] else torch.full((B,), Sk - Sq, device=device)
        i = torch.arange(Sq, device=device)[None, :] + first[:, None]
        ok = ok & (j[None, None, :] <= i[:, :, None])
    return ok[:, None]


def _att_forward(c, q, k, v, ok):
    """Attention of [B, heads, Sq, dh] over keys repeated to as many heads:
    outputs, log-sum-exp, and the probabilities."""
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(c["head_dim"]))
    s = s.masked_fill(~ok, -math.inf)
    m = s.amax(3, keepdim=True)
    p = torch.exp(s - torch.where(torch.isfinite(m), m, torch.zeros_like(m)))
    l = p.sum(3, keepdim=True)
    p = p / torch.where(l > 0, l, torch.ones_like(l))
    return torch.matmul(p, v), (m + torch.log(l)).squeeze(3), p


def _att_backward(c, q, k, v, out, p, do):
    """Gradients of q and of the repeated keys and values."""
    dp = torch.matmul(do, v.transpose(2, 3))
    ds = p * (dp - (do * out).sum(3, keepdim=True)) * (1.0 / math.sqrt(c["head_dim"]))
    return torch.matmul(ds, k), torch.matmul(ds.transpose(2, 3), q), torch.matmul(p.transpose(2, 3), do)


def _shared(c, t):
    """Sum over the query heads of each key head."""
    B, H, S, dh = t.shape
    return t.view(B, c["kv_heads"], H // c["kv_heads"], S, dh).sum(2)


def _att_run(c, s):
    B, Sq, Sk, H, KH, dh = (c[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    if own:
        from cppnet_amd import ops
        how = {"causal": c["causal"], "k_len": s["k_len"], "q_start": s["q_start"], "rows": c["rows"]}
        ops.attention_forward(s["q"], s["k"], s["v"], s["out"], s["lse"], B, Sq, Sk, H, KH, dh, **how)
        if not c["train"]:
            return [s["out"], s["lse"]]
        ops.attention_backward(s["q"], s["k"], s["v"], s["out"], s["lse"], s["dout"], s["dq"], s["dk"], s["dv"],
                               B, Sq, Sk, H, KH, dh, **how)
        return [s["out"], s["lse"], s["dq"], s["dk"], s["dv"]]
    q = _heads(c, s["q"], H, Sq)
    k = _heads(c, s["k"], KH, Sk).repeat_interleave(H // KH, 1)
    v = _heads(c, s["v"], KH, Sk).repeat_interleave(H // KH, 1)
    o, lse, p = _att_forward(c, q, k, v, _allowed(c, s, q.device))
    res = [_stored(c, o), _stored(c, lse[..., None])]
    if c["train"]:
        dq, dk, dv = _att_backward(c, q, k, v, o, p, _heads(c, s["dout"], H, Sq))
        res += [_stored(c, dq), _stored(c, _shared(c, dk)), _stored(c, _shared(c, dv))]
    return res


def _att_one(q, k, v, scale, n, first, causal):
    """One head of one sample, [Sq, dh] over [Sk, dh]: outputs and log-sum-exp."""
    z = (q @ k[:n].T) * scale
    if causal:
        i = torch.arange(q.shape[0], device=q.device) + first
        z = torch.where(torch.arange(n, device=q.device)[None, :] > i[:, None], -math.inf, z)
    lse = torch.logsumexp(z, 1)
    w = torch.exp(z - torch.where(lse > -math.inf, lse, 0.0)[:, None])
    return w @ v[:n], lse


def _att_exact(c, s):
    B, Sq, Sk, H, KH, dh = (c[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    wide = [_heads(c, s[n].double(), h, m).contiguous()
            for n, h, m in (("q", H, Sq), ("k", KH, Sk), ("v", KH, Sk))]
    do = _heads(c, s["dout"].double(), H, Sq) if c["train"] else None
    out, lse = torch.zeros_like(wide[0]), wide[0].new_zeros(B, H, Sq, 1)
    grads = [torch.zeros_like(t) for t in wide]
    for b, (n, first) in enumerate(zip(_lengths(c), _starts(c))):
        for h in range(H):
            at = [(b, h), (b, h // (H // KH)), (b, h // (H // KH))]
            one = [t[i].clone().requires_grad_(c["train"]) for t, i in zip(wide, at)]
            o, e = _att_one(*one, 1.0 / math.sqrt(dh), n, first, c["causal"])
            out[b, h], lse[b, h, :, 0] = o.detach(), e.detach()
            if c["train"]:
                for g, i, d in zip(grads, at, torch.autograd.grad(o, one, do[b, h])):
                    g[i] += d
    return [_stored(c, t) for t in [out, lse] + (grads if c["train"] else [])]


def _att_work(c):
    B, Sq, Sk, H, KH, dh = (c[k] for k in ("batch", "queries", "keys", "heads", "kv_heads", "head_dim"))
    pairs = held = 0
    for n, first in zip(_lengths(c), _starts(c)):
        held += n
        if not c["causal"]:
            pairs += Sq * n
        else:  # query i reads keys 0 .. first + i, cut to [0, n]
            pairs += sum(min(n, max(0, first + i + 1)) for i in range(Sq))
    q, kv, l = B * Sq * H * dh, held * KH * dh, B * Sq * H
    if not c["train"]:
        return {"bytes": 4 * (2 * q + 2 * kv + l), "flops": 4 * dh * H * pairs}
    # forward, then the backward's five products; q, k, v, out and their gradients once each
    return {"bytes": 4 * (4 * q + 4 * kv + l), "flops": 14 * dh * H * pairs}


# ------------------------------------- Linear with softmax cross-entropy
def _ce_prepare(c, g):
    N, D, V = c["batch"], c["dim"], c["vocab"]
    s = {"X": _randn(g, D, N), "W": _randn(g, V, D) / math.sqrt(D), "b": 0.1 * _randn(g, V) if c["bias"] else None,
         "t": _tokens(g, N, V, True, c["padded"]), "loss": _empty(1), "lse": _empty(N)}
    if c["train"]:
        s.update(dX=_empty(D, N), dW=_empty(V, D), db=_empty(V) if c["bias"] else None)
    return s


def _ce_plain(X, W, b, t, train):
    """Loss (mean over the rows with a target), log-sum-exp, and the gradients
    of X (D, N), W (V, D) and b."""
    z = X.t() @ W.t()
    if b is not None:
        z = z + b
    m = z.amax(1, keepdim=True)
    e = torch.exp(z - m)
    l = e.sum(1, keepdim=True)
    lse = (m + torch.log(l)).squeeze(1)
    held = t >= 0
    count = held.sum().clamp(min=1)
    at = t.long().clamp(min=0)
    loss = torch.where(held, lse - z.gather(1, at[:, None]).squeeze(1), torch.zeros_like(lse)).sum() / count
    if not train:
        return [loss.reshape(1), lse]
    onehot = (at[:, None] == torch.arange(W.shape[0], device=W.device)[None, :]).float()
    G = (e / l - onehot) * (held / count)[:, None]
    res = [loss.reshape(1), lse, (G @ W).t().contiguous(), G.t() @ X.t()]
    return res if b is None else res + [G.sum(0)]


def _ce_run(c, s):
    N, D, V = c["batch"], c["dim"], c["vocab"]
    if own:
        from cppnet_amd import ops
        if not c["train"]:
            ops.linear_ce_forward(s["X"], s["W"], s["b"], s["t"], s["loss"], s["lse"], N, D, V)
            return [s["loss"], s["lse"]]
        ops.linear_ce_head(s["X"], s["W"], s["b"], s["t"], s["loss"], s["lse"], s["dX"], s["dW"], s["db"], N, D, V)
        return [s[k] for k in ("loss", "lse", "dX", "dW", "db") if s[k] is not None]
    return _ce_plain(s["X"], s["W"], s["b"], s["t"], c["train"])


def _ce_exact(c, s):
    leaves = [t.double().requires_grad_(c["train"]) for t in (s["X"], s["W"], s["b"]) if t is not None]
    z = torch.matmul(leaves[1], leaves[0])  # [V, N]
    if c["bias"]:
        z = z + leaves[2][:, None]
    lse = torch.logsumexp(z, 0)
    rows = (s["t"] >= 0).nonzero().squeeze(1)
    loss = (lse[rows] - z[s["t"][rows].long(), rows]).sum() / max(1, rows.numel())
    res = [loss.detach().reshape(1), lse.detach()]
    return res + list(torch.autograd.grad(loss, leaves)) if c["train"] else res


def _ce_work(c):
    N, D, V = c["batch"], c["dim"], c["vocab"]
    b = V if c["bias"] else 0
    if not c["train"]:
        return {"bytes": 4 * (N * D + V * D + b + 2 * N), "flops": 2 * N * D * V}
    return {"bytes": 4 * (2 * (N * D + V * D + b) + 2 * N), "flops": 6 * N * D * V}


# ------------------------------------------- a language model's training step
# Embedding -> q, k, v projections -> causal attention -> output projection
# with the skip sum -> cross-entropy against the next token, the output weights
# being the embedding's table; backward to every parameter.
def _lm_prepare(c, g):
    B, S, V, D = c["batch"], c["steps"], c["vocab"], c["dim"]
    N = B * S
    return {"ids": _tokens(g, N, V, True, 0), "t": _tokens(g, N, V, True, 1), "Wt": _randn(g, V, D) / math.sqrt(D),
            "Wqkv": _randn(g, 3 * D, D) / math.sqrt(D), "Wo": _randn(g, D, D) / math.sqrt(D),
            "x": _empty(D, N), "qkv": _empty(3 * D, N), "a": _empty(D, N), "lse": _empty(c["heads"], N),
            "h": _empty(D, N), "loss": _empty(1), "hlse": _empty(N), "dh": _empty(D, N), "da": _empty(D, N),
            "dqkv": _empty(3 * D, N), "dx": _empty(D, N), "gWt": _empty(V, D), "gWqkv": _empty(3 * D, D),
            "gWo": _empty(D, D)}


def _lm_att(c):
    return {"batch": c["batch"], "queries": c["steps"], "keys": c["steps"], "heads": c["heads"],
            "kv_heads": c["heads"], "head_dim": c["dim"] // c["heads"], "causal": True, "ragged": False,
            "decode": False, "rows": c["rows"], "train": True}


def _lm_run(c, s):
    B, S, V, D, H = (c[k] for k in ("batch", "steps", "vocab", "dim", "heads"))
    N, dh, scale = B * S, D // H, math.sqrt(D)
    if own:
        from cppnet_amd import ops
        rows = c["rows"]
        ops.token_embedding_forward(s["ids"], s["Wt"], s["x"], B, S, V, D, scale=scale, rows=rows)
        ops.linear_forward(s["x"], s["Wqkv"], None, s["qkv"], N, D, 3 * D)
        q, k, v = s["qkv"][:D], s["qkv"][D:2 * D], s["qkv"][2 * D:]
        ops.attention_forward(q, k, v, s["a"], s["lse"], B, S, S, H, H, dh, causal=True, rows=rows)
        ops.linear_forward_act(s["a"], s["Wo"], None, s["h"], s["x"], N, D, D, "residual")
        ops.linear_ce_head(s["h"], s["Wt"], None, s["t"], s["loss"], s["hlse"], s["dh"], s["gWt"], None, N, D, V)
        ops.linear_backward(s["a"], s["Wo"], s["dh"], s["gWo"], None, s["da"], N, D, D, accumulate=False)
        dq, dk, dv = s["dqkv"][:D], s["dqkv"][D:2 * D], s["dqkv"][2 * D:]
        ops.attention_backward(q, k, v, s["a"], s["lse"], s["da"], dq, dk, dv, B, S, S, H, H, dh, causal=True, rows=rows)
        ops.linear_backward_act(s["x"], s["Wqkv"], s["dqkv"], s["gWqkv"], None, s["dx"], s["dh"], N, D, 3 * D, "residual")
        ops.token_embedding_backward(s["ids"], s["dx"], s["gWt"], B, S, V, D, scale=scale, accumulate=True, rows=rows)
        return [s["loss"], s["gWt"], s["gWqkv"], s["gWo"]]
    a = _lm_att(c)
    x = _emb_forward(c, s["ids"], s["Wt"], scale)
    qkv = s["Wqkv"] @ x
    q, k, v = (_heads(a, t, H, S) for t in (qkv[:D], qkv[D:2 * D], qkv[2 * D:]))
    o, _, p = _att_forward(a, q, k, v, _allowed(a, s, x.device))
    ctx = _stored(a, o)
    h = s["Wo"] @ ctx + x
    loss, _, dh_, gW = _ce_plain(h, s["Wt"], None, s["t"], True)
    dctx = _heads(a, s["Wo"].t() @ dh_, H, S)
    dqkv = torch.cat([_stored(a, t) for t in _att_backward(a, q, k, v, o, p, dctx)])
    dx = s["Wqkv"].t() @ dqkv + dh_
    return [loss, _emb_backward(c, s["ids"], dx, scale, gW), dqkv @ x.t(), dh_ @ ctx.t()]


def _lm_exact(c, s):
    B, S, V, D, H = (c[k] for k in ("batch", "steps", "vocab", "dim", "heads"))
    dh = D // H
    W, Wqkv, Wo = (s[n].double().requires_grad_(True) for n in ("Wt", "Wqkv", "Wo"))
    x = W[_rows_of_ids(c, s["ids"]).long()] * math.sqrt(D)  # [N, D]
    q, k, v = (x @ Wqkv.T).split(D, 1)
    order = (lambda t: t.view(S, B, H, dh).permute(1, 2, 0, 3)) if c["rows"] == REF else \
        (lambda t: t.view(B, S, H, dh).permute(0, 2, 1, 3))
    q, k, v = (order(t) for t in (q, k, v))
    later = torch.ones(S, S, dtype=torch.bool, device=x.device).triu(1)
    w = torch.softmax((q @ k.transpose(2, 3) / math.sqrt(dh)).masked_fill(later, -math.inf), 3)
    o = w @ v
    o = (o.permute(2, 0, 1, 3) if c["rows"] == REF else o.permute(0, 2, 1, 3)).reshape(B * S, D)
    z = torch.log_softmax((o @ Wo.T + x) @ W.T, 1)
    rows = (s["t"] >= 0).nonzero().squeeze(1)
    loss = -z[rows, s["t"][rows].long()].sum() / max(1, rows.numel())
    return [loss.detach().reshape(1)] + list(torch.autograd.grad(loss, (W, Wqkv, Wo)))


def _lm_work(c):
    B, S, V, D, H = (c[k] for k in ("batch", "steps", "vocab", "dim", "heads"))
    N = B * S
    pairs = B * S * (S + 1) // 2
    return {"bytes": 4 * (2 * V * D + 8 * D * D + 2 * N),
            "flops": 6 * N * D * V + 24 * N * D * D + 14 * D * pairs}


KINDS = {
    "embedding": (_emb_prepare, _emb_run, _emb_exact, _emb_work),
    "attention": (_att_prepare, _att_run, _att_exact, _att_work),
    "linear_ce": (_ce_prepare, _ce_run, _ce_exact, _ce_work),
    "lm_step": (_lm_prepare, _lm_run, _lm_exact, _lm_work),
}


def _emb(name, batch, steps, vocab, dim, zipf=True, padded=0, rows=BY_SAMPLE, train=True):
    return {"name": name, "kind": "embedding", "batch": batch, "steps": steps, "vocab": vocab, "dim": dim,
            "zipf": zipf, "padded": padded, "rows": rows, "train": train}


def _att(name, batch, queries, keys, heads, kv_heads, head_dim, causal=True, ragged=False, decode=False,
         rows=BY_SAMPLE, train=True):
    return {"name": name, "kind": "attention", "batch": batch, "queries": queries, "keys": keys, "heads": heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "causal": causal, "ragged": ragged, "decode": decode,
            "rows": rows, "train": train}


def _ce(name, batch, dim, vocab, bias=False, padded=0, train=True):
    return {"name": name, "kind": "linear_ce", "batch": batch, "dim": dim, "vocab": vocab, "bias": bias,
            "padded": padded, "train": train}


def listed():
    return [
        # the tokens of one decoding step of 8 sequences
        _emb("embedding_token", 8, 1, 32000, 512, train=False),
        # the framework's transformer configuration: 32 x 256 uniform ids of 8192, width 512
        _emb("embedding_config", 32, 256, 8192, 512, zipf=False),
        # text over a large vocabulary, an eighth of it padding, rows in the reference order
        _emb("embedding_text", 7, 2047, 50001, 1000, padded=2, rows=REF),
        # one new token of each of 16 sequences over caches of up to 4096, 4 query heads a key head
        _att("attention_decode", 16, 1, 4096, 16, 4, 128, ragged=True, decode=True, train=False),
        # a small model's batch, where launches count
        _att("attention_small", 4, 63, 63, 4, 4, 32),
        # the framework's transformer configuration: 32 x 256, width 512 in 8 heads
        _att("attention_config", 32, 256, 256, 8, 8, 64),
        # an encoder's ragged batch, odd sizes, rows in the reference order
        _att("attention_ragged", 5, 1001, 1001, 6, 3, 80, causal=False, ragged=True, rows=REF),
        # long sequences, wide heads, 4 query heads a key head
        _att("attention_long", 2, 4096, 4096, 16, 4, 128),
        # a small batch over the configuration's vocabulary, with a bias
        _ce("linear_ce_small", 64, 512, 8192, bias=True),
        # evaluation of an odd number of rows over an odd vocabulary
        _ce("linear_ce_eval", 1021, 513, 32003, bias=True, train=False),
        # training over a large vocabulary, a sixteenth of the targets padding
        _ce("linear_ce_train", 8192, 1024, 32000, padded=1),
        # all of them together with the framework's Linear, tied weights
        {"name": "lm_step", "kind": "lm_step", "batch": 8, "steps": 512, "vocab": 16384, "dim": 512, "heads": 8,
         "rows": BY_SAMPLE},
    ]


def draw(rng):
    kind = rng.choice(["embedding", "attention", "attention", "linear_ce", "lm_step"])
    rows = rng.choice([REF, BY_SAMPLE, BY_SAMPLE])
    if kind == "embedding":
        train = rng.random() < 0.8
        steps = _log(rng, 1, 4096)
        c = _emb("", _log(rng, 1, max(1, min(64, 16384 // steps))), steps, _log(rng, 50, 50000), _log(rng, 16, 1024),
                 rng.random() < 0.6, rng.choice([0, 0, 2]), rows, train)
    elif kind == "attention":
        kv = rng.choice([1, 2, 4, 5])
        heads = kv * rng.choice([1, 1, 2, 4])
        dh = rng.choice([32, 64, 128, rng.randint(8, 128)])
        if rng.random() < 0.3:
            c = _att("", _log(rng, 1, 32), rng.choice([1, 1, 1, 2, 5]), _log(rng, 64, 8192), heads, kv, dh, True, True,
                     True, rows, False)
        else:
            keys = _log(rng, 16, 4096)
            queries = keys if rng.random() < 0.75 else rng.randint(1, keys)
            c = _att("", _log(rng, 1, max(1, min(32, 8192 // keys))), queries, keys, heads, kv, dh, rng.random() < 0.7,
                     rng.random() < 0.3, False, rows, rng.random() < 0.75)
    elif kind == "linear_ce":
        c = _ce("", _log(rng, 1, 8192), _log(rng, 32, 1024), _log(rng, 100, 32000), rng.random() < 0.3,
                rng.choice([0, 1]), rng.random() < 0.7)
    else:
        heads = rng.choice([2, 4, 8])
        c = {"kind": kind, "batch": rng.randint(1, 8), "steps": _log(rng, 16, 512), "vocab": _log(rng, 500, 16384),
             "dim": heads * rng.randint(16, 64), "heads": heads, "rows": rows}
    c.pop("name", None)
    return c


def prepare(case, seed):
    state = KINDS[case["kind"]][0](case, _gen(seed))
    state["case"] = case
    return state


def run(state):
    c = state["case"]
    return KINDS[c["kind"]][1](c, state)


def exact(case, seed):
    return KINDS[case["kind"]][2](case, KINDS[case["kind"]][0](case, _gen(seed)))


def work(case):
    return KINDS[case["kind"]][3](case)
