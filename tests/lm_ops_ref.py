"""Plain 64-bit forms of the language-model operators on logical matrices, with
the error that an fp32 implementation may have in each output.

Bounds.  u = 2^-24 is the rounding of fp32.  A sum of n products in any order
is off by at most g(n) = 2 (n + 8) u times the sum of the absolute products:
one rounding per product and per addition, doubled because the matrix cores cut
the low bits of a sum where an fp32 adder rounds them, and 8 more for the few
roundings around the sum (scales, exponentials to 2 ulp, a division).  Errors
of intermediate values are carried to the outputs to first order, exactly as
the formulas chain them; second-order terms are covered by a factor 1.05.

Where an operand is held as a pair of fp16 terms (cppnet_amd/csrc/mfma_pair.hpp)
a value is kept to 2^-22 of itself, which the 8 more in g cover (2 * 8 u =
2^-20), but not closer than F = 2^-39 of the operand's largest: the largest is
scaled to at least 2^14, and the second term is rounded on fp16's subnormal grid
of 2^-24, so by 2^-25 at most.  The cross-entropy's gradient is scaled by 2^15.

In the attention, operands are blocks of 32 rows of a sample and head.
Probabilities are scaled by 2^14, and dS by the power of two that takes its
block's bound 2 max ||dout_i|| max ||v_j|| (i in the block) to 2^14 at least.
In sums over blocks, P and dS also carry by how much the other factor's block,
x, is smaller than the largest block up to there, X: by 2^-d, the quotient of the
two blocks' powers of two.  Scaled, x and X both lie in [2^14, 2^15), so 2^d < 2 X
/ x.  P and dS are off by F at most (times dS's bound), so their product with a
value |y| <= x by F 2^d |y| < 2 F X.  A pair of a query and a key is off by at most
2 F max |v| in out, 2 F bound_i max |k| in dq, 2 F max |dout| in dv, 2 F max (bound
|q|) in dk (2^-25 2^15 in scaled units, of which bound and |q| each are 2^14 or
more), where the last two are over the blocks of queries from that on which the
first of the 128 keys around it is read by."""
import numpy as np

U = 2.0 ** -24
F = 2.0 ** -39


def g(n):
    return 2.0 * (n + 8) * U


def embedding(ids, W, scale):
    """[N] ids, W [V, D] -> out [N, D]; ids outside the table read zeros."""
    held = (ids >= 0) & (ids < W.shape[0])
    out = np.zeros((ids.size, W.shape[1]))
    out[held] = W[ids[held]] * scale
    return out


def embedding_grad(ids, dY, V, scale, base=None):
    """Gradient of W [V, D] and its bound."""
    grad = np.zeros((V, dY.shape[1])) if base is None else base.astype(np.float64).copy()
    mag, n = np.abs(grad), np.zeros(V)
    for p, i in enumerate(ids):
        if 0 <= i < V:
            grad[i] += scale * dY[p]
            mag[i] += abs(scale) * np.abs(dY[p])
            n[i] += 1
    return grad, np.array([g(k + 1) for k in n])[:, None] * mag


def allowed(B, Sq, Sk, causal, k_len, q_start):
    n = np.full(B, Sk) if k_len is None else np.clip(np.asarray(k_len), 0, Sk)
    ok = np.broadcast_to(np.arange(Sk)[None, None, :] < n[:, None, None], (B, Sq, Sk)).copy()
    if causal:
        first = np.full(B, Sk - Sq) if q_start is None else np.asarray(q_start, np.int64)
        ok &= np.arange(Sk)[None, None, :] <= first[:, None, None] + np.arange(Sq)[None, :, None]
    return ok


def attention(q, k, v, ok, scale, dout=None):
    """q [B, H, Sq, dh], k, v [B, KH, Sk, dh] (values at keys that no query of
    the sample reads may be anything), ok [B, Sq, Sk].  Returns {name: (value,
    bound)} for out, lse and, given dout, dq, dk, dv."""
    B, H, Sq, dh = q.shape
    KH, Sk = k.shape[1], k.shape[2]
    G = H // KH
    used = ok.any(1)[:, None, :, None]
    k0, v0 = np.where(used, k, 0.0), np.where(used, v, 0.0)
    K, Vv = np.repeat(k0, G, 1), np.repeat(v0, G, 1)
    T = lambda x: np.swapaxes(x, 2, 3)  # noqa: E731
    m = ok[:, None]
    s = np.where(m, scale * (q @ T(K)), -np.inf)
    top = s.max(3, keepdims=True)
    top = np.where(np.isfinite(top), top, 0.0)
    p = np.exp(s - top)
    l = p.sum(3, keepdims=True)
    some = l > 0
    P = p / np.where(some, l, 1.0)
    with np.errstate(divide="ignore"):
        lse = (top + np.log(l))[..., 0]
    out = P @ Vv
    # scores: the contraction, and the roundings of scale * log2(e) and of the
    # exponent's difference; from the score's and the maximum's size
    es = np.where(m, g(dh) * abs(scale) * (np.abs(q) @ T(np.abs(K))) + 6 * U * np.abs(np.where(m, s, 0)), 0.0)

    def block(x):  # every row's block's largest
        x = np.abs(x).max(3)
        top = np.maximum.reduceat(x, np.arange(0, x.shape[2], 32), 2)
        return np.repeat(top, 32, 2)[:, :, :x.shape[2], None]

    aq, aK = np.abs(q), np.abs(K)
    mq, mk, mv = block(q), block(K), block(Vv)
    row = lambda x: x.sum(3, keepdims=True)  # noqa: E731
    most = lambda x: x.max(2, keepdims=True)  # noqa: E731
    reads = m.sum(3, keepdims=True)
    es = es + np.where(m, abs(scale) * F * (mq * T(row(aK)) + T(mk) * row(aq)), 0.0)
    es = es.max(3, keepdims=True) + 6 * U * np.abs(top)
    eP = 2 * es + g(Sk)  # relative, of every probability of a row
    aV = P @ np.abs(Vv)
    eo = eP * aV + g(Sk) * aV + F * (P @ mv) + 2 * F * reads * most(mv)
    el = (es + g(Sk) + 4 * U * np.abs(np.where(np.isfinite(lse), lse, 0))[..., None])[..., 0]
    res = {"out": (out, 1.05 * eo), "lse": (lse, 1.05 * el)}
    if dout is None:
        return res
    do, ado = dout, np.abs(dout)
    dP = do @ T(Vv)
    norm = lambda x: np.sqrt((x * x).sum(3, keepdims=True))  # noqa: E731
    mdo, bound = block(do), 2 * block(norm(do)) * most(norm(Vv))
    edP = g(dh) * (ado @ T(np.abs(Vv))) + F * (mdo * T(row(np.abs(Vv))) + T(mv) * row(ado))
    delta = (do * out).sum(3, keepdims=True)
    edelta = g(dh) * (ado * np.abs(out)).sum(3, keepdims=True) + (ado * eo).sum(3, keepdims=True)
    dS = P * (dP - delta) * scale
    eb = 2 * es + el[..., None] + g(0)  # of the probability formed again from lse
    edS = abs(scale) * P * (edP + edelta + (eb + g(0)) * (np.abs(dP) + np.abs(delta)))
    edS = np.where(m, edS, 0.0)
    aS = np.abs(dS)
    dq, eq = dS @ K, edS @ np.abs(K) + g(Sk) * (aS @ np.abs(K)) + F * (aS @ mk)
    eq = eq + 2 * abs(scale) * F * bound * most(mk) * reads
    # the first of the queries' blocks for each key, and the largest from there on
    read = ok.reshape(B, Sq, Sk).any(1)
    lead = np.arange(Sk) // 128 * 128
    first = np.where(read, ok.argmax(1), Sq - 1)[:, lead] // 32 * 32
    after = lambda x: np.take_along_axis(np.maximum.accumulate(x[:, :, ::-1], 2)[:, :, ::-1],  # noqa: E731
                                         np.broadcast_to(first[:, None, :, None], (B, H, Sk, 1)), 2)
    taken = np.broadcast_to(T(m).sum(3, keepdims=True), (B, H, Sk, 1))
    share = lambda x: x.reshape(B, KH, G, Sk, dh).sum(2)  # noqa: E731
    n = Sq * G
    dk = share(T(dS) @ q)
    ek = share(T(edS) @ np.abs(q) + g(n) * (T(aS) @ np.abs(q)) + F * (T(aS) @ mq) + 2 * abs(scale) * F * taken * after(bound * mq))
    dv = share(T(P) @ do)
    ev = share(T(P * eb) @ ado + g(n) * (T(P) @ ado) + F * (T(P) @ mdo) + 2 * F * taken * after(mdo))
    res.update(dq=(dq, 1.05 * eq), dk=(dk, 1.05 * ek), dv=(dv, 1.05 * ev))
    return res


def linear_ce(X, W, b, t, mean, acc=None):
    """X [N, D], W [D, V], b [V] or None, t [N].  {name: (value, bound)} for
    loss, lse, dX, dW, db; acc = (dW, db) that the gradients are added to."""
    N, D = X.shape
    V = W.shape[1]
    held = (t >= 0) & (t < V)
    count = max(1, held.sum()) if mean else 1
    bb = np.zeros(V) if b is None else b
    z = X @ W + bb
    aW, aX = np.abs(W), np.abs(X)
    mx = np.where(held, aX[held].max() if held.any() else 0.0, aX.max(1))[:, None]
    ez = g(D) * (aX @ aW + np.abs(bb)) + F * (mx * aW.sum(0) + aW.max() * aX.sum(1, keepdims=True))
    top = z.max(1, keepdims=True)
    p = np.exp(z - top)
    l = p.sum(1, keepdims=True)
    lse = (top + np.log(l))[:, 0]
    es = ez.max(1) + 6 * U * (np.abs(top[:, 0]) + np.abs(z).max(1))
    el = es + g(V) + 4 * U * np.abs(lse)
    at = np.where(held, t, 0)
    rows = np.where(held, lse - z[np.arange(N), at], 0.0)
    erow = np.where(held, el + es + 2 * U * np.abs(rows), 0.0)
    loss, eloss = rows.sum() / count, (erow.sum() + g(N) * np.abs(rows).sum()) / count
    P = p / l
    G = P.copy()
    G[np.arange(N)[held], t[held]] -= 1.0
    G = np.where(held[:, None], G, 0.0) / count
    eG = np.where(held[:, None], P * (es + el + g(0))[:, None], 0.0) / count + 4 * U * np.abs(G)
    aG = np.abs(G)
    eG = eG + np.where(held[:, None], F / count, 0.0)
    dX, eX = G @ W.T, eG @ aW.T + g(V) * (aG @ aW.T) + F * aW.max() * aG.sum(1, keepdims=True)
    dW, eW = X.T @ G, aX.T @ eG + g(N) * (aX.T @ aG) + F * mx.max(where=held[:, None], initial=0.0) * aG.sum(0)
    db, eb = G.sum(0), eG.sum(0) + g(N) * np.abs(G).sum(0)
    if acc is not None:
        dW, db = dW + acc[0], db + acc[1]
        eW, eb = eW + 2 * U * np.abs(dW), eb + 2 * U * np.abs(db)
    return {"loss": (np.array([loss]), np.array([1.05 * eloss])), "lse": (lse, 1.05 * el), "dX": (dX, 1.05 * eX),
            "dW": (dW, 1.05 * eW), "db": (db, 1.05 * eb)}


def check(name, got, want, bound, tiny=1e-37):
    """got within bound of want, infinities equal; `tiny`: below fp32's normal range."""
    got = np.asarray(got, np.float64)
    assert got.shape == want.shape, f"{name}: shape {got.shape}, not {want.shape}"
    fine = np.isfinite(want)
    assert np.array_equal(got[~fine], want[~fine]), f"{name}: infinities differ"
    assert np.isfinite(got[fine]).all(), f"{name}: {(~np.isfinite(got[fine])).sum()} values are not finite"
    err, lim = np.abs(got[fine] - want[fine]), np.broadcast_to(bound, want.shape)[fine] + U * np.abs(want[fine]) + tiny
    bad = err > lim
    if bad.any():
        i = int(np.argmax(err - lim))
        raise AssertionError(f"{name}: {bad.sum()} of {bad.size} outside; worst off by {err[i]:.3g}, bound {lim[i]:.3g}, "
                             f"value {want[fine][i]:.6g}")
    return float((err / lim).max()) if err.size else 0.0
