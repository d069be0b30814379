"""GPU tests of the language-model operators where their paths and their data
end: every path of the attention over caches that hold anything past the read
keys, blocks of very different size, row pieces of the cross-entropy, rows
without a target that hold anything, captured calls.  Forms and bounds are
those of lm_ops_ref.py."""
import numpy as np
import pytest
import torch

import lm_ops_ref as ref
from cppnet_amd import ops
from test_gpu_lm_ops import REF, SAMPLE, Buffers, att_run, host, per_head

pytestmark = pytest.mark.gpu


def wide(x, h):
    return per_head(x.astype(np.float64), h)


def att_check(dims, causal, k_len, q_start, rows, scale, q, k, v, do):
    B, Sq, Sk, H, KH, dh = dims
    ok = ref.allowed(B, Sq, Sk, causal, k_len, q_start)
    buf = Buffers()
    got = att_run(buf, (q, k, v), dict(causal=causal, k_len=k_len, q_start=q_start, rows=rows), dims, do, scale)
    read = ok.any(1)[:, :, None]
    want = ref.attention(wide(q, H), wide(np.where(read, k, 0), KH), wide(np.where(read, v, 0), KH), ok,
                         dh ** -0.5 if scale is None else scale, None if do is None else wide(do, H))
    for name, (w, lim) in want.items():
        x = got[name].transpose(0, 2, 1) if name == "lse" else per_head(got[name], KH if name in ("dk", "dv") else H)
        print("  ", name, ref.check(name, x, w, lim))
    buf.intact()
    return got


FEW = [  # B, Sq, Sk, H, KH, dh, causal, rows: one to nine query rows a key head
    (1, 1, 1, 1, 1, 1, False, SAMPLE), (2, 1, 31, 3, 1, 8, True, REF), (3, 1, 32, 4, 1, 32, False, SAMPLE),
    (1, 1, 33, 5, 1, 33, True, SAMPLE), (2, 2, 127, 2, 2, 64, True, SAMPLE), (1, 4, 129, 2, 1, 80, True, REF),
    (2, 1, 257, 8, 1, 96, False, SAMPLE), (1, 8, 300, 1, 1, 97, True, SAMPLE), (2, 1, 3001, 4, 1, 128, True, SAMPLE),
    (1, 3, 2050, 4, 2, 128, True, REF), (1, 1, 5000, 8, 1, 128, False, SAMPLE), (2, 7, 40, 2, 2, 100, True, SAMPLE),
    (2, 3, 90, 3, 1, 64, True, SAMPLE), (5, 1, 700, 6, 6, 40, True, SAMPLE), (2, 5, 3, 1, 1, 16, True, SAMPLE),
]


@pytest.mark.parametrize("B,Sq,Sk,H,KH,dh,causal,rows", FEW)
def test_attention_of_few_rows(gpu, B, Sq, Sk, H, KH, dh, causal, rows):
    print(f"[attention] B={B} {Sq}x{Sk} heads {H}/{KH} dh={dh} causal={causal} rows={rows}", flush=True)
    rng = np.random.default_rng(B + Sk + dh)
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v = f(B, Sq, H * dh), f(B, Sk, KH * dh), f(B, Sk, KH * dh)
    k_len = [int(n) for n in rng.integers(0, Sk + 1, B)]
    k_len[-1] = Sk
    for b in range(B):
        k[b, k_len[b]:], v[b, k_len[b]:] = np.nan, np.inf
    start = [n - Sq for n in k_len] if causal else None
    att_check((B, Sq, Sk, H, KH, dh), causal, k_len, start, rows, None, q, k, v, None)


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("Sq,H,KH,dh", [(1, 4, 2, 64), (3, 2, 1, 128), (20, 4, 2, 32), (70, 2, 1, 64), (130, 2, 2, 96)])
def test_attention_over_a_cache_with_anything_past_its_last_query(gpu, Sq, H, KH, dh, rows):
    print(f"[attention] cache {Sq} heads {H}/{KH} dh={dh} rows={rows}", flush=True)
    rng = np.random.default_rng(Sq)
    B, Sk = 4, 300
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v, do = f(B, Sq, H * dh), f(B, Sk, KH * dh), f(B, Sk, KH * dh), f(B, Sq, H * dh)
    start = [0, 299 - Sq, -Sq, 101]  # the third sample reads nothing
    for b in range(B):
        k[b, start[b] + Sq:], v[b, start[b] + Sq:] = np.inf, np.nan
    got = att_check((B, Sq, Sk, H, KH, dh), True, None, start, rows, None, q, k, v, do)
    for name in ("dk", "dv"):
        for b in range(B):
            assert (got[name][b, start[b] + Sq:] == 0).all()
    assert (got["out"][2] == 0).all() and (got["lse"][2] == -np.inf).all() and (got["dq"][2] == 0).all()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("S,H,KH,dh", [(160, 2, 1, 64), (200, 1, 1, 128), (40, 2, 2, 32)])
def test_attention_of_blocks_of_very_different_size(gpu, S, H, KH, dh, causal):
    print(f"[attention] blocks {S} heads {H}/{KH} dh={dh} causal={causal}", flush=True)
    rng = np.random.default_rng(S + dh)
    size = lambda *e: np.array(e)[np.arange(S) // 32 % len(e)].astype(np.float32)[None, :, None]  # noqa: E731
    f = lambda h: rng.standard_normal((2, S, h * dh)).astype(np.float32)  # noqa: E731
    q = f(H) * size(1.0, 2.0 ** -30, 4.0, 0.0, 2.0 ** -70)
    k = f(KH) * size(2.0 ** -20, 1.0, 0.0, 2.0)
    v = f(KH) * size(2.0 ** 40, 2.0 ** -40, 1.0, 0.0, 2.0 ** 20)
    do = f(H) * size(2.0 ** -50, 1.0, 2.0 ** 30, 0.0)
    att_check((2, S, S, H, KH, dh), causal, None, None, SAMPLE, None, q, k, v, do)


@pytest.mark.parametrize("which", ["q", "k", "v", "dout", "all"])
@pytest.mark.parametrize("S", [5, 40, 100])
def test_attention_of_zeros(gpu, S, which):
    rng = np.random.default_rng(S)
    x = {n: rng.standard_normal((2, S, 64)).astype(np.float32) for n in ("q", "k", "v", "dout")}
    for n in x:
        if which in (n, "all"):
            x[n][:] = 0
    att_check((2, S, S, 2, 2, 32), True, None, None, REF, None, x["q"], x["k"], x["v"], x["dout"])


@pytest.mark.parametrize("B,Sq,Sk", [(1, 1, 40), (1, 1, 4000), (2, 20, 30), (2, 20, 900), (64, 130, 140)])
def test_attention_of_scores_past_the_range(gpu, B, Sq, Sk):
    """Where every score that a query reads is -inf, its softmax is 0 / 0 in
    every path; other queries keep theirs, but for those packed with it, whose
    scale is that query's."""
    rng = np.random.default_rng(Sk)
    q, k, v = (np.abs(rng.standard_normal((B, s, 32))).astype(np.float32) + np.float32(0.5) for s in (Sq, Sk, Sk))
    k *= np.float32(-1e25)
    q *= np.float32(1e-25)
    q[:, 0] *= np.float32(1e38)
    q[:, 0] *= np.float32(1e7)  # scores below -1e43
    got = att_run(Buffers(), (q, k, v), dict(causal=False, k_len=None, q_start=None, rows=SAMPLE), (B, Sq, Sk, 1, 1, 32))
    assert np.isnan(got["out"][:, 0]).all() and not np.isfinite(got["lse"][:, 0]).any()
    want = ref.attention(wide(q[:, 1:], 1), wide(k, 1), wide(v, 1), np.ones((B, Sq - 1, Sk), bool), 32 ** -0.5) if 1 < Sq < 64 else {}
    for name, (w, lim) in want.items():
        x = got[name].transpose(0, 2, 1) if name == "lse" else per_head(got[name], 1)
        ref.check(name, x[:, :, 1:], w, lim)


@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0 ** -60, 1.5])
@pytest.mark.parametrize("S", [6, 45, 97])
def test_attention_gradients_at_any_scale(gpu, S, scale):
    rng = np.random.default_rng(S)
    q, k, v, do = (rng.standard_normal((2, S, 96)).astype(np.float32) for _ in range(4))
    att_check((2, S, S, 2, 2, 48), True, [S, S // 2], None, SAMPLE, scale, q, k, v, do)


@pytest.mark.parametrize("Sq", [1, 2, 20, 70])
def test_attention_gradient_is_the_slope(gpu, Sq):
    """Along a direction u, f = sum(out * dout) in 64 bits moves by the gradients.
    A step h of the central difference leaves h^2 / 6 of the third derivative.
    That of a row of out is a fourth joint cumulant of v and s' three times, s'
    = scale u k or scale q u: at most 2^4 + 3 * 2^4 of |v| |s'|^3, for values
    off their mean by twice their largest."""
    rng = np.random.default_rng(Sq)
    B, Sk, H, KH, dh, h = 1, 90, 2, 1, 32, 2.0 ** -14
    f = lambda s, h: rng.standard_normal((B, s, h * dh)).astype(np.float32)  # noqa: E731
    x, do = [f(Sq, H), f(Sk, KH), f(Sk, KH)], f(Sq, H)
    dims, kw = (B, Sq, Sk, H, KH, dh), dict(causal=True, k_len=None, q_start=None, rows=SAMPLE)
    got = att_run(Buffers(), x, kw, dims, do)
    ok = ref.allowed(B, Sq, Sk, True, None, None)
    wq, wk, wv = (wide(a, n) for a, n in zip(x, (H, KH, KH)))
    want = ref.attention(wq, wk, wv, ok, dh ** -0.5, wide(do, H))
    longest = max(np.linalg.norm(wq, axis=3).max(), np.linalg.norm(wk, axis=3).max())
    third = 64 * np.abs(do).sum() * np.abs(wv).max() * (dh ** -0.5 * longest) ** 3
    for i, name in enumerate(("dq", "dk", "dv")):
        u = rng.standard_normal((wq, wk, wv)[i].shape)
        u /= np.linalg.norm(u)
        def value(step):
            y = [wq, wk, wv]
            y[i] = y[i] + step * u
            return (ref.attention(*y, ok, dh ** -0.5)["out"][0] * wide(do, H)).sum()
        slope = (value(h) - value(-h)) / (2 * h)
        along = (wide(got[name], (H, KH, KH)[i]) * u).sum()
        lim = (want[name][1] * np.abs(u)).sum() + h * h / 6 * third + 1e-12 * np.abs(do).sum() / h
        assert abs(along - slope) <= lim, (name, along, slope, lim)


def ce_run(buf, X, W, b, t, reduction, base=None):
    N, D = X.shape
    V = W.shape[1]
    x, w, tt = buf.new(X.T), buf.new(W.T), buf.new(t, np.int32)
    loss, lse, dX = buf.empty(1), buf.empty(N), buf.empty(N * D)
    dW = buf.empty(D * V) if base is None else base
    bb, db = (None, None) if b is None else (buf.new(b), buf.empty(V))
    ops.linear_ce_head(x, w, bb, tt, loss, lse, dX, dW, db, N, D, V, reduction, base is not None)
    return {"loss": host(loss), "lse": host(lse), "dX": host(dX).reshape(D, N).T, "dW": host(dW).reshape(V, D).T,
            **({} if b is None else {"db": host(db)})}, dW, (x, w, bb, tt)


@pytest.mark.parametrize("N", [40, 100, 600])
@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf, 1e30, 3e38])
def test_linear_ce_rows_without_a_target_may_hold_anything(gpu, N, what):
    print(f"[linear ce] N={N} {what} in rows without a target", flush=True)
    rng = np.random.default_rng(N)
    D, V = 70, 700
    X, W = rng.standard_normal((N, D)).astype(np.float32), (rng.standard_normal((D, V)) / 8).astype(np.float32)
    b, t = rng.standard_normal(V).astype(np.float32), rng.integers(0, V, N).astype(np.int32)
    t[rng.random(N) < 0.4] = -1
    held = t >= 0
    plain = np.where(held[:, None], X, 0)
    X[~held, 3:9] = what
    buf = Buffers()
    got, _, (x, w, bb, tt) = ce_run(buf, X, W, b, t, "mean")
    d = lambda a: a.astype(np.float64)  # noqa: E731
    want = ref.linear_ce(d(plain), d(W), d(b), t, True)
    for name in ("loss", "dX", "dW", "db"):
        print("  ", name, ref.check(name, got[name], *want[name]))
    ref.check("lse", got["lse"][held], *(a[held] for a in want["lse"]))
    loss, lse = buf.empty(1), buf.empty(N)
    ops.linear_ce_forward(x, w, bb, tt, loss, lse, N, D, V)
    ref.check("loss of the forward", host(loss), *want["loss"])
    ref.check("lse of the forward", host(lse)[held], *(a[held] for a in want["lse"]))
    if not np.isfinite(what):  # such values count as zeros
        zeroed = ref.linear_ce(d(np.where(np.isfinite(X), X, 0)), d(W), d(b), t, True)["lse"]
        ref.check("lse of all", got["lse"], *zeroed)
        ref.check("lse of all, forward", host(lse), *zeroed)
    buf.intact()


def test_linear_ce_in_pieces_of_rows(gpu):
    """1100 rows of 131080 classes go through as 1024 and 76, as two calls over
    those rows do, the second adding to the first's gradient.  The parts that dX
    is summed in may be others where a call's largest piece is another."""
    rng = np.random.default_rng(8)
    N, D, V, R = 1100, 20, 131080, 1024
    X, W = rng.standard_normal((N, D)).astype(np.float32), (rng.standard_normal((D, V)) / 4).astype(np.float32)
    X[[0, R]] = 5.0  # the same largest value in both
    t = rng.integers(0, V, N).astype(np.int32)
    t[[3, 500, 1050]] = -1
    buf = Buffers()
    whole, _, (x, w, _, tt) = ce_run(buf, X, W, None, t, "sum")
    one, dW, _ = ce_run(buf, X[:R], W, None, t[:R], "sum")
    two, _, _ = ce_run(buf, X[R:], W, None, t[R:], "sum", dW)
    np.testing.assert_array_equal(whole["lse"], np.concatenate([one["lse"], two["lse"]]))
    np.testing.assert_array_equal(whole["dX"][:R], one["dX"])
    d = lambda a: a.astype(np.float64)  # noqa: E731
    sample = np.concatenate([np.arange(20), [3, 500], np.arange(R, R + 20), [1050]])
    want = ref.linear_ce(d(X[sample]), d(W), None, t[sample], False)
    ref.check("lse", whole["lse"][sample], *want["lse"])
    ref.check("dX", whole["dX"][sample], *want["dX"])
    ref.check("dX of two calls", np.concatenate([one["dX"], two["dX"]])[sample], *want["dX"])
    lse = np.concatenate([np.log(np.exp(d(X[i:i + 100]) @ d(W)).sum(1)) for i in range(0, N, 100)])
    held = t >= 0
    loss = (lse - (d(X) * d(W)[:, np.where(held, t, 0)].T).sum(1))[held].sum()
    bound = ref.g(D + V + N) * (np.abs(lse) + np.abs(d(X)).sum(1) * np.abs(W).max()).sum()
    assert abs(whole["loss"][0] - loss) <= bound and abs(one["loss"][0] + two["loss"][0] - loss) <= bound
    cols = np.unique(np.concatenate([t[held][:50], rng.integers(0, V, 50), [0, V - 1]]))
    z = d(X) @ d(W)[:, cols]
    P = np.exp(z - lse[:, None])
    G = np.where(held[:, None], P - (t[:, None] == cols), 0)
    # errors of z, lse and G as in the reference, with the rows' largest values
    ez = ref.g(D) * (np.abs(d(X)) @ np.abs(d(W)[:, cols])) + 2 * D * ref.F * np.abs(X).max() * np.abs(W).max()
    el = ref.g(D) * (np.abs(d(X)).sum(1) * np.abs(W).max()) + ref.g(V) + 16 * ref.U * np.abs(lse)
    eG = held[:, None] * (P * (ez + el[:, None] + ref.g(0)) + 4 * ref.U * np.abs(G) + ref.F)
    lim = np.abs(d(X)).T @ eG + ref.g(N) * (np.abs(d(X)).T @ np.abs(G)) + ref.F * 5.0 * np.abs(G).sum(0)
    for a in (whole, two):
        ref.check("dW", a["dW"][:, cols], d(X).T @ G, 1.05 * lim)
    loss, lse32 = buf.empty(1), buf.empty(N)
    ops.linear_ce_forward(x, w, None, tt, loss, lse32, N, D, V, "sum")
    ref.check("lse of the forward", host(lse32), lse, 1.05 * el)
    buf.intact()


@pytest.mark.parametrize("N", [65, 70, 257])
@pytest.mark.parametrize("D,V", [(1, 1), (1, 2), (2, 1), (17, 3), (3, 129), (700, 1), (33, 32)])
def test_linear_ce_of_few_features_and_classes(gpu, N, D, V):
    rng = np.random.default_rng(N + D)
    X, W = rng.standard_normal((N, D)).astype(np.float32), rng.standard_normal((D, V)).astype(np.float32)
    b, t = rng.standard_normal(V).astype(np.float32), rng.integers(-1, V + 1, N).astype(np.int32)
    buf = Buffers()
    got, _, (x, w, bb, tt) = ce_run(buf, X, W, b, t, "mean")
    want = ref.linear_ce(*(a.astype(np.float64) for a in (X, W, b)), t, True)
    for name, a in got.items():
        ref.check(name, a, *want[name])
    loss, lse, oob = buf.empty(1), buf.empty(N), buf.new([5], np.int32)
    ops.linear_ce_forward(x, w, bb, tt, loss, lse, N, D, V, "mean", oob)
    ref.check("loss of the forward", host(loss), *want["loss"])
    ref.check("lse of the forward", host(lse), *want["lse"])
    assert host(oob)[0] == 5 + (t == V).sum()
    buf.intact()


@pytest.mark.parametrize("scale", [-1.5, 0.0, 2.0 ** -130])
def test_token_embedding_at_any_scale(gpu, scale):
    rng = np.random.default_rng(3)
    B, S, V, D = 3, 70, 40, 33
    ids = rng.integers(-1, V + 1, B * S).astype(np.int32)
    W, dY = rng.standard_normal((V, D)).astype(np.float32), rng.standard_normal((B * S, D)).astype(np.float32)
    W[~np.isin(np.arange(V), ids)] = np.nan  # rows that no id names are not read
    buf = Buffers()
    tid, out, gW = buf.new(ids, np.int32), buf.empty(B * S * D), buf.empty(V * D)
    ops.token_embedding_forward(tid, buf.new(W), out, B, S, V, D, scale)
    held = (ids >= 0) & (ids < V)
    want = np.where(held[:, None], W[np.clip(ids, 0, V - 1)] * np.float32(scale), np.float32(0))
    np.testing.assert_array_equal(host(out).reshape(D, B * S).T, want)
    ops.token_embedding_backward(tid, buf.new(dY.T), gW, B, S, V, D, scale)
    want, lim = ref.embedding_grad(ids, dY.astype(np.float64), V, scale)
    ref.check("gW", host(gW).reshape(V, D), want, lim + 2.0 ** -149)  # below 2^-126 a rounding is to 2^-149
    buf.intact()


@pytest.mark.parametrize("Sq,N", [(1, 30), (40, 70), (96, 300)])
def test_captured_calls_replayed_over_new_data(gpu, Sq, N):
    """Attention and cross-entropy forward in one graph, replayed with eager
    calls of other sizes between the replays."""
    rng = np.random.default_rng(Sq)
    B, Sk, H, KH, dh, D, V = 2, 640, 4, 2, 64, 48, 900
    f = lambda n: torch.from_numpy(rng.standard_normal(n).astype(np.float32)).cuda()  # noqa: E731
    q, k, v = f(B * Sq * H * dh), f(B * Sk * KH * dh), f(B * Sk * KH * dh)
    X, W, t = f(N * D), f(D * V), torch.from_numpy(rng.integers(-1, V, N).astype(np.int32)).cuda()
    new = lambda: [torch.empty(n, device="cuda") for n in (q.numel(), B * Sq * H, 1, N)]  # noqa: E731
    got, want = new(), new()

    def run(out):
        ops.attention_forward(q, k, v, out[0], out[1], B, Sq, Sk, H, KH, dh, True)
        ops.linear_ce_forward(X, W, None, t, out[2], out[3], N, D, V)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(got)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(got)
    for _ in range(4):
        for x in (q, k, v, X):
            x.copy_(f(x.numel()))
        for x in got:
            x.fill_(float("nan"))
        run(want)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_attention_over_a_cache_past_32_bits(gpu):
    """One query over a cache of more than 2^31 values: 17 GB of keys and
    values.  Sums run in lanes, waves and blocks, 1024 tiles of 32 keys a block
    at most, so no chain of additions is longer than 2^12 and g(2^12) bounds
    them; out, lse, and dk and dv of the first and last keys, each a product of
    the one query."""
    dh, Sk = 128, 2 ** 24 + 77
    torch.manual_seed(1)
    k, v = torch.randn(dh, Sk, device="cuda"), torch.randn(dh, Sk, device="cuda")
    q, do = torch.randn(dh, device="cuda"), torch.randn(dh, device="cuda")
    out, lse = torch.full_like(q, float("nan")), torch.full((1,), float("nan"), device="cuda")
    dims, kw = (1, 1, Sk, 1, 1, dh), dict(causal=True, rows=SAMPLE)
    ops.attention_forward(q, k, v, out, lse, *dims, **kw)
    scale = dh ** -0.5
    s, es = [], 0.0
    for j in range(0, Sk, 1 << 20):
        part = k[:, j:j + (1 << 20)].double()
        s.append(q.double() @ part * scale)
        es = max(es, float((q.double().abs() @ part.abs()).max()) * ref.g(dh) * scale + 6 * ref.U * float(s[-1].abs().max()))
    s = torch.cat(s)
    es += 6 * ref.U * float(s.max())
    want_lse = torch.logsumexp(s, 0)
    P = torch.exp(s - want_lse)
    want, mag = torch.zeros(dh, device="cuda", dtype=torch.float64), torch.zeros(dh, device="cuda", dtype=torch.float64)
    for j in range(0, Sk, 1 << 20):
        part = v[:, j:j + (1 << 20)].double()
        want += part @ P[j:j + (1 << 20)]
        mag += part.abs() @ P[j:j + (1 << 20)]
    n = 2 ** 12
    el = es + ref.g(n) + 4 * ref.U * abs(float(want_lse))
    eo = (2 * es + 2 * ref.g(n)) * mag
    num = lambda t: t.cpu().double().numpy()  # noqa: E731
    ref.check("lse", num(lse), num(want_lse[None]), 1.05 * el)
    ref.check("out", num(out), num(want), num(1.05 * eo))
    dq, dk, dv = torch.empty_like(q), torch.full_like(k, float("nan")), torch.full_like(v, float("nan"))
    ops.attention_backward(q, k, v, out, lse, do, dq, dk, dv, *dims, **kw)
    delta = float((do.double() * want).sum())
    edelta = float((do.double().abs() * want.abs()).sum()) * ref.g(dh) + float((do.double().abs() * eo).sum())
    eb = 2 * es + el + ref.g(0)
    top = lambda x: float(x.abs().max())  # noqa: E731
    bound = 2 * float(do.double().norm()) * float(v.norm(dim=0).max())
    for at in (slice(0, 300), slice(Sk - 300, Sk)):
        p, part = P[at], v[:, at].double()
        dP = do.double() @ part
        dS = p * (dP - delta) * scale
        edP = ref.g(dh) * (do.double().abs() @ part.abs()) + 2 * dh * ref.F * top(do) * top(v)
        edS = scale * p * (edP + edelta + (eb + ref.g(0)) * (dP.abs() + abs(delta)))
        aq, ado = q.double().abs()[:, None], do.double().abs()[:, None]
        ek = aq * edS + ref.g(1) * aq * dS.abs() + 2 * scale * ref.F * bound * top(q) + ref.F * top(q) * dS.abs()
        ev = ado * p * (eb + ref.g(1)) + 3 * ref.F * top(do)
        ref.check("dk", num(dk[:, at]), num(q.double()[:, None] * dS), num(1.05 * ek))
        ref.check("dv", num(dv[:, at]), num(do.double()[:, None] * p), num(1.05 * ev))
    assert torch.isfinite(dq).all() and torch.isfinite(dk[:, ::1009]).all() and torch.isfinite(dv[:, ::1009]).all()


@pytest.mark.parametrize("N", [5, 70])
def test_tied_table_past_32_bits(gpu, N):
    """A table of more than 2^31 values, 9 GB, as the embedding's and as the
    Linear's weight.  Exponentials are summed over 128 classes at once, then in
    chains of 2^11 in sixteen waves: g(2^12) bounds them."""
    V, D = 2 ** 22 + 5, 520
    torch.manual_seed(2)
    W = torch.randn(V, D, device="cuda") / D ** 0.5
    X = torch.randn(D, N, device="cuda")
    t = torch.randint(0, V, (N,), device="cuda", dtype=torch.int32)
    t[0], t[1], t[2] = V - 1, 0, V
    loss, lse, dX = (torch.full((n,), float("nan"), device="cuda") for n in (1, N, N * D))
    dW = torch.full_like(W, float("nan"))
    ops.linear_ce_head(X, W, None, t, loss, lse, dX, dW, None, N, D, V, "sum")
    x, step = X.double().t(), 1 << 18
    z = torch.cat([x @ W[v:v + step].double().t() for v in range(0, V, step)], 1)
    mag = max(float((x.abs() @ W[v:v + step].double().abs().t()).max()) for v in range(0, V, step))
    want = torch.logsumexp(z, 1)
    top = lambda a: float(a.abs().max())  # noqa: E731
    ez = ref.g(D) * mag + 2 * D * ref.F * top(X) * top(W)
    el = ez + 12 * ref.U * top(z) + ref.g(2 ** 12) + 4 * ref.U * top(want)
    num = lambda a: a.cpu().double().numpy()  # noqa: E731
    ref.check("lse", num(lse), num(want), 1.05 * el)
    held = t < V
    at = torch.where(held, t, 0).long()
    rows = torch.where(held, want - z.gather(1, at[:, None])[:, 0], 0.0)
    ref.check("loss", num(loss), num(rows.sum()[None]), 1.05 * N * (el + ez + 4 * ref.U * top(rows)) + ref.g(N) * float(rows.sum()))
    for cols in (slice(0, 300), slice(V - 300, V)):
        P = torch.exp(z[:, cols] - want[:, None])
        G = torch.where(held[:, None], P - (t[:, None] == torch.arange(V, device="cuda")[cols]).double(), 0.0)
        eG = held[:, None] * (P * (ez + el + ref.g(0)) + 4 * ref.U * G.abs() + ref.F)
        lim = eG.t() @ x.abs() + ref.g(N) * (G.abs().t() @ x.abs()) + ref.F * top(X) * G.abs().sum(0)[:, None]
        ref.check("dW", num(dW[cols]), num(G.t() @ x), num(1.05 * lim))
    assert torch.isfinite(dX).all() and torch.isfinite(dW.view(-1)[::1009]).all()
    # the embedding of the same table, its gradient added to the Linear's
    ids = torch.tensor([V - 1, 0, V - 2, V - 1, V, -1], device="cuda", dtype=torch.int32)
    out, dY = torch.full((D, 6), float("nan"), device="cuda"), torch.randn(D, 6, device="cuda")
    ops.token_embedding_forward(ids, W, out, 1, 6, V, D)
    assert torch.equal(out[:, :4].t(), W[ids[:4].long()]) and (out[:, 4:] == 0).all()
    before = dW[[V - 1, V - 2, 0, V - 3]].clone()
    ops.token_embedding_backward(ids, dY, dW, 1, 6, V, D, 1.0, True)
    assert torch.equal(dW[[V - 1, V - 2, 0, V - 3]],
                       before + torch.stack([dY[:, 0] + dY[:, 3], dY[:, 2], dY[:, 1], torch.zeros_like(dY[:, 0])]))
