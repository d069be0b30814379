"""GPU tests of the language-model operators (token embedding, attention
without kept probabilities, Linear with cross-entropy) against their 64-bit
forms in lm_ops_ref.py, whose bounds are derived there."""
import numpy as np
import pytest
import torch

import lm_ops_ref as ref
from cppnet_amd import _capi, ops

pytestmark = pytest.mark.gpu

REF, SAMPLE = ops.ROWS_REF, ops.ROWS_BY_SAMPLE
GUARD = 37  # floats around every operand: an odd offset, so that float4s are unaligned


class Buffers:
    """Device operands inside guarded allocations."""

    def __init__(self):
        self.all = []

    def new(self, a, dtype=np.float32, offset=GUARD):
        a = np.ascontiguousarray(a, dtype).ravel()
        whole = np.full(a.size + 2 * GUARD, 77, dtype)
        whole[offset:offset + a.size] = a
        t = torch.from_numpy(whole).cuda()
        self.all.append((t, offset, a.size))
        return t[offset:offset + a.size]

    def empty(self, n, offset=GUARD):
        return self.new(np.full(n, np.nan, np.float32), offset=offset)

    def intact(self):
        torch.cuda.synchronize()
        for t, offset, n in self.all:
            w = t.cpu().numpy()
            assert (w[:offset] == 77).all() and (w[offset + n:] == 77).all(), "values around an operand were written"


def host(t):
    torch.cuda.synchronize()
    return t.cpu().numpy()


# [B, S, F] <-> the framework's storage
def stored(x, rows):
    return x.transpose(2, 1, 0) if rows == REF else x.transpose(2, 0, 1)


def logical(flat, B, S, F, rows):
    return flat.reshape(F, S, B).transpose(2, 1, 0) if rows == REF else flat.reshape(F, B, S).transpose(1, 2, 0)


# ---------------------------------------------------------------- embedding
EMB = [  # B, S, V, D, ids, rows
    (1, 1, 1, 1, "uniform", REF), (8, 1, 1000, 64, "uniform", SAMPLE), (3, 5, 7, 33, "padded", REF),
    (3, 5, 7, 33, "padded", SAMPLE), (4, 64, 50, 512, "uniform", SAMPLE), (2, 257, 300, 130, "zipf", REF),
    (5, 401, 3, 66, "uniform", SAMPLE), (7, 300, 5000, 257, "same", SAMPLE), (2, 1024, 999, 40, "padded", SAMPLE),
    (1, 77, 40, 1000, "none", REF), (33, 31, 1025, 3, "zipf", SAMPLE),
    (3, 4100, 600, 36, "zipf", REF),  # more ids than one piece of the comparing sort
    (9, 4096, 70000, 36, "zipf", SAMPLE), (5, 8000, 200, 20, "padded", REF), (4, 10007, 65535, 6, "uniform", SAMPLE),
    (1, 33000, 2, 5, "same", REF),    # the radix sort, one to three passes
]


def make_ids(rng, kind, n, V):
    if kind == "same":
        return np.full(n, V - 1, np.int32)
    if kind == "none":
        return np.where(rng.random(n) < 0.5, -1, V).astype(np.int32)
    ids = rng.integers(0, V, n) if kind != "zipf" else np.floor(np.exp(rng.random(n) * np.log(V + 1)) - 1)
    ids = np.clip(ids, 0, V - 1).astype(np.int32)
    if kind == "padded":
        ids[rng.random(n) < 0.3] = -1
        ids[rng.random(n) < 0.1] = V
        ids[rng.random(n) < 0.05] = np.iinfo(np.int32).min
    return ids


@pytest.mark.parametrize("B,S,V,D,kind,rows", EMB)
def test_token_embedding(gpu, B, S, V, D, kind, rows):
    print(f"[token embedding] {B}x{S} V={V} D={D} {kind} rows={rows}", flush=True)
    rng = np.random.default_rng(B * 1000 + S * 10 + D)
    ids = make_ids(rng, kind, B * S, V)
    W, dY, base = rng.standard_normal((V, D)), rng.standard_normal((B * S, D)), rng.standard_normal((V, D))
    W, dY, base = (x.astype(np.float32) for x in (W, dY, base))
    scale = np.float32(np.sqrt(D) * 1.1)
    # dY's rows follow `rows`; ids are ColMajor [B, S]
    order = ids if rows == REF else ids.reshape(S, B).T.ravel()
    buf = Buffers()
    tid, tW, tY = buf.new(ids, np.int32), buf.new(W), buf.new(dY.T)
    out, oob = buf.empty(B * S * D), buf.new([3], np.int32)
    ops.token_embedding_forward(tid, tW, out, B, S, V, D, float(scale), oob, rows)
    want = np.where(((order >= 0) & (order < V))[:, None], W[np.clip(order, 0, V - 1)] * scale, np.float32(0))
    np.testing.assert_array_equal(host(out).reshape(D, B * S).T, want)
    assert host(oob)[0] == 3 + ((ids < 0) | (ids >= V)).sum()
    for acc in (False, True):
        gW = buf.new(base) if acc else buf.empty(V * D)
        ops.token_embedding_backward(tid, tY, gW, B, S, V, D, float(scale), acc, rows)
        want, lim = ref.embedding_grad(order, dY.astype(np.float64), V, float(scale), base if acc else None)
        got = host(gW).reshape(V, D)
        print("  worst share of the bound", ref.check("gW", got, want, lim))
        unused = np.setdiff1d(np.arange(V), order)
        np.testing.assert_array_equal(got[unused], base[unused] if acc else np.zeros((unused.size, D), np.float32))
        again = buf.new(base) if acc else buf.empty(V * D)
        ops.token_embedding_backward(tid, tY, again, B, S, V, D, float(scale), acc, rows)
        np.testing.assert_array_equal(host(again).reshape(V, D), got)
    buf.intact()


# ---------------------------------------------------------------- attention
ATT = [  # B, Sq, Sk, H, KH, dh, causal, k_len, q_start, rows
    (1, 1, 1, 1, 1, 1, False, None, None, SAMPLE),
    (1, 1, 1, 1, 1, 8, True, None, None, REF),
    (2, 5, 5, 2, 1, 32, True, None, None, SAMPLE),
    (2, 33, 33, 2, 2, 33, True, None, None, REF),
    (3, 64, 64, 4, 2, 64, False, [64, 0, 31], None, SAMPLE),
    (2, 130, 130, 2, 1, 64, True, [130, 77], None, SAMPLE),
    (2, 31, 97, 6, 2, 80, True, None, None, SAMPLE),
    (2, 97, 31, 2, 2, 40, True, None, None, SAMPLE),     # the first 66 queries read nothing
    (2, 20, 50, 2, 1, 128, True, [7, 50], [-5, 33], REF),
    (4, 1, 300, 8, 2, 64, True, [1, 300, 0, 123], [0, 299, -1, 122], SAMPLE),
    (3, 2, 200, 4, 4, 128, True, [2, 200, 129], [0, 198, 127], REF),
    (1, 1, 1025, 16, 1, 96, False, None, None, SAMPLE),
    (1, 257, 257, 1, 1, 128, True, None, None, SAMPLE),
    (2, 200, 300, 3, 1, 17, False, [300, 299], None, REF),
    (1, 40, 600, 4, 2, 100, False, [-3], None, SAMPLE),
    (2, 513, 513, 2, 1, 64, True, [900, 400], None, SAMPLE),
    (3, 96, 160, 4, 2, 128, True, [160, 0, 3], None, REF),
    (1, 300, 300, 2, 1, 96, True, None, None, SAMPLE),
    (2, 129, 65, 4, 4, 32, False, [65, 64], None, SAMPLE),
    (3, 200, 700, 8, 2, 64, True, [700, 650, 100], [500, -40, 2000], SAMPLE),
    (2, 385, 130, 3, 3, 128, True, None, [0, -200], REF),
    (1, 65, 1100, 5, 5, 81, False, None, None, SAMPLE),
]


def att_run(buf, x, kw, dims, dout=None, scale=None):
    q, k, v = x
    B, Sq, Sk, H, KH, dh = dims
    rows = kw["rows"]
    how = dict(causal=kw["causal"], rows=rows, scale=scale,
               k_len=None if kw["k_len"] is None else buf.new(kw["k_len"], np.int32),
               q_start=None if kw["q_start"] is None else buf.new(kw["q_start"], np.int32))
    t = [buf.new(stored(a, rows)) for a in (q, k, v)]
    out, lse = buf.empty(B * Sq * H * dh), buf.empty(B * Sq * H)
    ops.attention_forward(*t, out, lse, *dims, **how)
    res = {"out": logical(host(out), B, Sq, H * dh, rows), "lse": logical(host(lse), B, Sq, H, rows)}
    if dout is not None:
        g = [buf.empty(a.numel()) for a in t]
        ops.attention_backward(*t, out, lse, buf.new(stored(dout, rows)), *g, *dims, **how)
        for name, a, S, h in zip(("dq", "dk", "dv"), g, (Sq, Sk, Sk), (H, KH, KH)):
            res[name] = logical(host(a), B, S, h * dh, rows)
    return res


def per_head(x, h):
    B, S, F = x.shape
    return x.reshape(B, S, h, F // h).transpose(0, 2, 1, 3)


@pytest.mark.parametrize("B,Sq,Sk,H,KH,dh,causal,k_len,q_start,rows", ATT)
def test_attention(gpu, B, Sq, Sk, H, KH, dh, causal, k_len, q_start, rows):
    print(f"[attention] B={B} {Sq}x{Sk} heads {H}/{KH} dh={dh} causal={causal} {k_len} {q_start} rows={rows}", flush=True)
    rng = np.random.default_rng(Sq * 7 + Sk * 3 + dh + H)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v, do = f(B, Sq, H * dh), f(B, Sk, KH * dh), f(B, Sk, KH * dh), f(B, Sq, H * dh)
    n = np.full(B, Sk) if k_len is None else np.clip(k_len, 0, Sk)
    for b in range(B):  # what lies past a sample's keys is nobody's
        k[b, n[b]:], v[b, n[b]:] = np.nan, np.inf
    buf = Buffers()
    kw = dict(causal=causal, k_len=k_len, q_start=q_start, rows=rows)
    dims = (B, Sq, Sk, H, KH, dh)
    got = att_run(buf, (q, k, v), kw, dims, do)
    d = lambda x, h: per_head(x.astype(np.float64), h)  # noqa: E731
    ok = ref.allowed(B, Sq, Sk, causal, k_len, q_start)
    for b in range(B):
        k[b, n[b]:], v[b, n[b]:] = 0, 0
    want = ref.attention(d(q, H), d(k, KH), d(v, KH), ok, dh ** -0.5, d(do, H))
    for name, (w, lim) in want.items():
        x = got[name].transpose(0, 2, 1) if name == "lse" else per_head(got[name], KH if name in ("dk", "dv") else H)
        print("  ", name, ref.check(name, x, w, lim))
    buf.intact()


def test_attention_lse_is_optional_and_scale_may_be_any(gpu):
    rng = np.random.default_rng(5)
    B, Sq, Sk, H, KH, dh = 2, 40, 70, 2, 1, 48
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v = f(B, Sq, H * dh), f(B, Sk, KH * dh), f(B, Sk, KH * dh)
    for scale in (-0.3, 0.0, 2.0):
        buf = Buffers()
        got = att_run(buf, (q, k, v), dict(causal=True, k_len=None, q_start=None, rows=SAMPLE), (B, Sq, Sk, H, KH, dh),
                      f(B, Sq, H * dh), scale)
        d = lambda x, h: per_head(x.astype(np.float64), h)  # noqa: E731
        want = ref.attention(d(q, H), d(k, KH), d(v, KH), ref.allowed(B, Sq, Sk, True, None, None), scale)
        for name in ("out", "lse"):
            x = got[name].transpose(0, 2, 1) if name == "lse" else per_head(got[name], H)
            ref.check(name, x, *want[name])
    buf = Buffers()
    t = [buf.new(stored(a, SAMPLE)) for a in (q, k, v)]
    out, with_lse, lse = buf.empty(q.size), buf.empty(q.size), buf.empty(B * Sq * H)
    ops.attention_forward(*t, out, None, B, Sq, Sk, H, KH, dh)
    ops.attention_forward(*t, with_lse, lse, B, Sq, Sk, H, KH, dh)
    np.testing.assert_array_equal(host(out), host(with_lse))


def test_attention_large_scores(gpu):
    """Scores of hundreds: the maximum is taken out before the exponential."""
    rng = np.random.default_rng(6)
    B, S, H, dh = 1, 96, 1, 64
    q, k, v, do = (rng.standard_normal((B, S, dh)).astype(np.float32) for _ in range(4))
    q *= 30
    k *= 3
    got = att_run(Buffers(), (q, k, v), dict(causal=False, k_len=None, q_start=None, rows=REF), (B, S, S, H, H, dh), do)
    d = lambda x: per_head(x.astype(np.float64), 1)  # noqa: E731
    want = ref.attention(d(q), d(k), d(v), ref.allowed(B, S, S, False, None, None), dh ** -0.5, d(do))
    for name, (w, lim) in want.items():
        x = got[name].transpose(0, 2, 1) if name == "lse" else per_head(got[name], 1)
        print("  ", name, ref.check(name, x, w, lim))


# ---------------------------------------------------- Linear + cross-entropy
CE = [  # N, D, V, bias, targets, reduction, accumulate
    (1, 1, 1, False, "all", "mean", False), (1, 64, 1000, True, "all", "mean", False), (3, 5, 2, True, "some", "sum", True),
    (64, 32, 100, False, "some", "mean", False), (32, 65, 300, True, "some", "mean", True), (33, 130, 1000, False, "all", "sum", True),
    (17, 513, 4100, True, "some", "mean", False), (65, 33, 257, True, "some", "mean", True),
    (130, 100, 1001, True, "all", "sum", False), (257, 128, 512, False, "none", "mean", True),
    (300, 256, 4096, True, "some", "mean", False), (513, 96, 333, True, "some", "mean", True),
    (1024, 64, 2048, False, "some", "mean", False),
]


@pytest.mark.parametrize("N,D,V,bias,kind,reduction,acc", CE)
def test_linear_ce(gpu, N, D, V, bias, kind, reduction, acc):
    print(f"[linear ce] N={N} D={D} V={V} bias={bias} {kind} {reduction} accumulate={acc}", flush=True)
    rng = np.random.default_rng(N + D * 3 + V)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    X, W, b = f(N, D), f(D, V) / np.float32(np.sqrt(D)), f(V) if bias else None
    t = rng.integers(0, V, N).astype(np.int32)
    if kind == "none":
        t[:] = -100
    elif kind == "some":
        t[rng.random(N) < 0.3] = -1
        t[rng.random(N) < 0.1] = V
        t[rng.random(N) < 0.1] = np.iinfo(np.int32).min
    base = (f(D, V), f(V) if bias else np.zeros(V, np.float32))
    buf = Buffers()
    x, w, tt, oob = buf.new(X.T), buf.new(W.T), buf.new(t, np.int32), buf.new([2], np.int32)
    bb = buf.new(b) if bias else None
    loss, lse, dX = buf.empty(1), buf.empty(N), buf.empty(N * D)
    dW = buf.new(base[0].T) if acc else buf.empty(D * V)
    db = (buf.new(base[1]) if acc else buf.empty(V)) if bias else None
    ops.linear_ce_head(x, w, bb, tt, loss, lse, dX, dW, db, N, D, V, reduction, acc, oob)
    d = lambda a: None if a is None else a.astype(np.float64)  # noqa: E731
    want = ref.linear_ce(d(X), d(W), d(b), t, reduction == "mean", tuple(map(d, base)) if acc else None)
    got = {"loss": host(loss), "lse": host(lse), "dX": host(dX).reshape(D, N).T, "dW": host(dW).reshape(V, D).T}
    if bias:
        got["db"] = host(db)
    for name, a in got.items():
        print("  ", name, ref.check(name, a, *want[name]))
    assert host(oob)[0] == 2 + (t >= V).sum()
    loss2, lse2 = buf.empty(1), buf.empty(N)
    ops.linear_ce_forward(x, w, bb, tt, loss2, lse2, N, D, V, reduction)
    ref.check("loss of the forward", host(loss2), *want["loss"])
    ref.check("lse of the forward", host(lse2), *want["lse"])
    buf.intact()


# ------------------------------------------------------- all of them together
def lm_step(buf, B, S, V, D, H, rows, ids, t, W, Wqkv, Wo, call=lambda f: f()):
    """One training step of a one-block language model with tied weights: its
    loss and gradients.  Returns a function of no arguments that runs it."""
    N, dh, scale = B * S, D // H, float(np.sqrt(D))
    x, qkv, a, lse, h, da, dqkv, dx, dh_ = (buf.empty(n * N) for n in (D, 3 * D, D, H, D, D, 3 * D, D, D))
    loss, hl = buf.empty(1), buf.empty(N)
    gW, gWqkv, gWo = buf.empty(V * D), buf.empty(3 * D * D), buf.empty(D * D)
    part = lambda m, i: m[i * D * N:(i + 1) * D * N]  # noqa: E731

    def step():
        ops.token_embedding_forward(ids, W, x, B, S, V, D, scale, rows=rows)
        ops.linear_forward(x, Wqkv, None, qkv, N, D, 3 * D)
        ops.attention_forward(part(qkv, 0), part(qkv, 1), part(qkv, 2), a, lse, B, S, S, H, H, dh, True, rows=rows)
        ops.linear_forward_act(a, Wo, None, h, x, N, D, D, "residual")
        ops.linear_ce_head(h, W, None, t, loss, hl, dh_, gW, None, N, D, V)
        ops.linear_backward(a, Wo, dh_, gWo, None, da, N, D, D, accumulate=False)
        ops.attention_backward(part(qkv, 0), part(qkv, 1), part(qkv, 2), a, lse, da, part(dqkv, 0), part(dqkv, 1),
                               part(dqkv, 2), B, S, S, H, H, dh, True, rows=rows)
        ops.linear_backward_act(x, Wqkv, dqkv, gWqkv, None, dx, dh_, N, D, 3 * D, "residual")
        ops.token_embedding_backward(ids, dx, gW, B, S, V, D, scale, True, rows)
    return step, (loss, gW, gWqkv, gWo)


@pytest.mark.parametrize("rows", [REF, SAMPLE])
def test_language_model_step(gpu, rows):
    """Loss and gradients of a whole step against 64-bit autograd: each gradient
    within 2e-5 of its size.  The chain has ten products; their bounds g(n) of
    at most 2 (1000 + 8) u = 1.2e-4 of the absolute sums leave room for
    rounding that all points one way, and random rounding stays below a
    twentieth of it."""
    B, S, V, D, H = 3, 37, 211, 64, 4
    rng = np.random.default_rng(11)
    f = lambda *s: (rng.standard_normal(s) / np.sqrt(D)).astype(np.float32)  # noqa: E731
    W, Wqkv, Wo = f(V, D), f(3 * D, D), f(D, D)
    ids, t = rng.integers(0, V, B * S).astype(np.int32), rng.integers(0, V, B * S).astype(np.int32)
    t[rng.random(B * S) < 0.2] = -1
    buf = Buffers()
    step, outs = lm_step(buf, B, S, V, D, H, rows, buf.new(ids, np.int32), buf.new(t, np.int32), buf.new(W),
                         buf.new(Wqkv), buf.new(Wo))
    step()
    got = [host(o) for o in outs]
    p = [torch.tensor(m, dtype=torch.float64, requires_grad=True) for m in (W, Wqkv, Wo)]
    order = torch.tensor(ids if rows == REF else ids.reshape(S, B).T.ravel()).long()
    x = p[0][order] * np.sqrt(D)
    split = (lambda m: m.view(S, B, H, D // H).permute(1, 2, 0, 3)) if rows == REF else \
        (lambda m: m.view(B, S, H, D // H).permute(0, 2, 1, 3))
    q, k, v = (split(m) for m in (x @ p[1].T).split(D, 1))
    s = (q @ k.transpose(2, 3) / np.sqrt(D // H)).masked_fill(torch.ones(S, S).triu(1).bool(), -np.inf)
    o = torch.softmax(s, 3) @ v
    o = (o.permute(2, 0, 1, 3) if rows == REF else o.permute(0, 2, 1, 3)).reshape(B * S, D)
    z = torch.log_softmax((o @ p[2].T + x) @ p[0].T, 1)
    at = torch.tensor(t).long()
    loss = -z[torch.arange(B * S), at.clamp(min=0)][at >= 0].mean()
    want = [loss.detach().reshape(1)] + list(torch.autograd.grad(loss, p))
    for name, a, w in zip(("loss", "gW", "gWqkv", "gWo"), got, want):
        w = w.numpy().ravel()
        rel = np.linalg.norm(a - w) / np.linalg.norm(w)
        print("  ", name, rel)
        assert rel < 2e-5, name
    buf.intact()


def test_language_model_step_in_a_graph(gpu):
    """The step captured on one stream and replayed between eager steps gives
    the eager bits every time."""
    B, S, V, D, H = 2, 70, 300, 64, 2
    rng = np.random.default_rng(12)
    f = lambda *s: (rng.standard_normal(s) / np.sqrt(D)).astype(np.float32)  # noqa: E731
    buf = Buffers()
    ids, t = (buf.new(rng.integers(0, V, B * S), np.int32) for _ in range(2))
    step, outs = lm_step(buf, B, S, V, D, H, SAMPLE, ids, t, buf.new(f(V, D)), buf.new(f(3 * D, D)), buf.new(f(D, D)))
    st = torch.cuda.Stream()
    import ctypes
    lib, handle = _capi.load(), ctypes.c_void_p(st.cuda_stream)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        step()
        st.synchronize()
        want = [host(o).copy() for o in outs]
        _capi.check(lib.cnhip_graph_begin_capture(handle))
        step()
        graph = ctypes.c_void_p()
        _capi.check(lib.cnhip_graph_end_capture(handle, 1, ctypes.byref(graph)))
        for _ in range(3):
            for o in outs:
                o.fill_(float("nan"))
            _capi.check(lib.cnhip_graph_launch(graph, handle))
            st.synchronize()
            for a, w in zip(outs, want):
                np.testing.assert_array_equal(host(a), w)
            step()
            st.synchronize()
            for a, w in zip(outs, want):
                np.testing.assert_array_equal(host(a), w)
        _capi.check(lib.cnhip_graph_destroy(graph))
    buf.intact()


def test_language_model_steps_on_two_streams(gpu):
    """Two steps with other inputs on two streams at once: each gives what it gives alone."""
    B, S, V, D, H = 2, 128, 500, 128, 2
    rng = np.random.default_rng(13)
    f = lambda *s: (rng.standard_normal(s) / np.sqrt(D)).astype(np.float32)  # noqa: E731
    runs = []
    for _ in range(2):
        buf = Buffers()
        ids, t = (buf.new(rng.integers(0, V, B * S), np.int32) for _ in range(2))
        step, outs = lm_step(buf, B, S, V, D, H, SAMPLE, ids, t, buf.new(f(V, D)), buf.new(f(3 * D, D)), buf.new(f(D, D)))
        step()
        runs.append((torch.cuda.Stream(), step, outs, [host(o).copy() for o in outs]))
    torch.cuda.synchronize()
    for _ in range(4):
        for st, step, _, _ in runs:
            with torch.cuda.stream(st):
                step()
    torch.cuda.synchronize()
    for _, _, outs, want in runs:
        for a, w in zip(outs, want):
            np.testing.assert_array_equal(host(a), w)
