"""Plain 64-bit forms of the operators of a recurrent language model's block on
logical arrays, with the error that an fp32 implementation may have in each output.

Bounds.  u = 2^-24 is the rounding of fp32, G(n) = 2 (n + 8) u that of a sum of n
products in any order (lm_ops_ref.py).  Errors are carried to first order, a factor
1.05 covers the rest.

The exponential of a sigmoid is zero where it is below fp32's normal range (2^-126):
SiLU is then off by 2^-126 |z|, its derivative by 2^-126 (1 + |z|); LOW covers both.

A sigmoid (and 1 minus it) is off by at most 8 u of itself: exp to 1 ulp (2 u), the
sum 1 + e, the reciprocal to 1 ulp (2 u), a product, and what those leave in the sum.

Recurrence.  M_t = a M_{t-1} + w |x| is the sum of the absolute terms.  Every step
adds what is off in its factor, 8 u (1 - a) M_{t-1} (the factor is held in two
floats, so it is off by as much as 1 - a is), and in its term, 10 u w |x|, and rounds
twice, 4 u M_t; these decay as the state does.  The state that enters a lane's steps
has also passed up to 4 + 6 + 1 + 16 joined maps, each of which rounds its sum twice:
64 u M_t covers them."""
import numpy as np

from lm_ops_ref import F, U, check, g as G  # noqa: F401


LOW = 2.0 ** -126


def sigmoid(z):
    z = np.asarray(z, np.float64)
    e = np.exp(-np.abs(z))
    return np.where(z >= 0, 1.0, e) / (1.0 + e)


def recurrence(x, f, i=None, h0=None, lengths=None, dh=None, dh_last=None):
    """x, f, i, dh [B, S, D], h0, dh_last [B, D].  {name: (value, bound)} for h and
    last, and given dh for dx, df, di, dh0."""
    B, S, D = x.shape
    a, off = sigmoid(f), sigmoid(-f)
    w, woff = (sigmoid(i), sigmoid(-i)) if i is not None else (off, None)
    n = np.full(B, S) if lengths is None else np.clip(lengths, 0, S)
    state = np.zeros((B, D)) if h0 is None else h0.astype(np.float64)
    M, E = np.abs(state), np.zeros((B, D))
    h, eh, before, ebefore = (np.zeros((B, S, D)) for _ in range(4))
    x = np.where(np.arange(S)[None, :, None] < n[:, None, None], x, 0.0)
    for t in range(S):
        on = (t < n)[:, None]
        before[:, t], ebefore[:, t] = state, E + 64 * U * M
        m1 = a[:, t] * M + w[:, t] * np.abs(x[:, t])
        e1 = a[:, t] * E + U * (8 * off[:, t] * M + 10 * w[:, t] * np.abs(x[:, t]) + 4 * m1)
        new = a[:, t] * state + w[:, t] * x[:, t]
        state, M, E = np.where(on, new, state), np.where(on, m1, M), np.where(on, e1, E)
        h[:, t], eh[:, t] = np.where(on, state, 0.0), np.where(on, E + 64 * U * M, 0.0)
    res = {"h": (h, 1.05 * eh), "last": (state, 1.05 * (E + 64 * U * M))}
    if dh is None:
        return res
    into = np.zeros((B, D)) if dh_last is None else dh_last.astype(np.float64)
    M, E = np.abs(into), np.zeros((B, D))
    grads = {k: (np.zeros((B, S, D)), np.zeros((B, S, D))) for k in (("dx", "df") if i is None else ("dx", "df", "di"))}
    for t in reversed(range(S)):
        on = (t < n)[:, None]
        at, ot, wt, xt, prev = a[:, t], off[:, t], w[:, t], x[:, t], before[:, t]
        d = np.where(on, dh[:, t], 0.0)
        gt, mg = into + d, M + np.abs(d)
        eg = E + U * mg + 64 * U * mg
        arm = prev if i is not None else prev - xt
        earm = ebefore[:, t] + (0.0 if i is not None else U * (np.abs(prev) + np.abs(xt)))
        vals = {"dx": (wt * gt, wt * (eg + 10 * U * mg)),
                "df": (at * ot * gt * arm, at * ot * (eg * np.abs(arm) + mg * earm + 20 * U * mg * np.abs(arm)))}
        if i is not None:
            vals["di"] = (wt * woff[:, t] * gt * xt, wt * woff[:, t] * np.abs(xt) * (eg + 20 * U * mg))
        for k, (v, e) in vals.items():
            grads[k][0][:, t], grads[k][1][:, t] = np.where(on, v, 0.0), np.where(on, 1.05 * e, 0.0)
        into = np.where(on, at * gt, into)
        E = np.where(on, at * (E + U * mg) + U * (8 * ot + 4) * mg, E)
        M = np.where(on, at * mg, M)
    return res | grads | {"dh0": (into, 1.05 * (E + 64 * U * M))}


# ------------------------------------------------------------------ dropout
def kept(n, p, seed, position):
    """The documented generator: entry j is kept where the top 24 bits of
    splitmix64(seed + (position + j) golden), over 2^24, are below 1 - p in fp32."""
    with np.errstate(over="ignore"):
        z = np.uint64(seed) + (np.uint64(position) + np.arange(n, dtype=np.uint64)) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    top = ((z ^ (z >> np.uint64(31))) >> np.uint64(40)).astype(np.float32)
    return top * np.float32(2.0 ** -24) < np.float32(1) - np.float32(p)


def dropped(x, p, seed, position):
    """fp32, bit for bit; x flat."""
    scale = np.float32(1) / (np.float32(1) - np.float32(p))
    return np.where(kept(x.size, p, seed, position), x * scale, np.float32(0)).astype(np.float32)


# --------------------------------------------------------------------- norm
def rms_norm(s, gamma, eps, dy=None, dsum=None, base=None):
    """s [N, F] as the kernel holds it.  {name: (value, bound)} for rstd and y, and
    given dy for ds and dgamma."""
    s, gamma = s.astype(np.float64), gamma.astype(np.float64)
    r = 1.0 / np.sqrt((s * s).mean(1) + float(np.float32(eps)))
    n = s * r[:, None]
    y = n * gamma
    res = {"rstd": (r, 1.05 * 2 * U * r), "y": (y, 1.05 * 5 * U * np.abs(y))}
    if dy is None:
        return res
    dy = dy.astype(np.float64)
    d = dy * gamma
    c, mag = (d * n).mean(1)[:, None], np.abs(d * n).mean(1)[:, None]
    skip = 0.0 if dsum is None else dsum.astype(np.float64)
    ds = skip + r[:, None] * (d - n * c)
    # n: rstd (2 u) and a product; d a product; their products are summed in 64 bits, c rounds once
    eds = r[:, None] * (6 * U * (np.abs(d) + np.abs(n * c)) + np.abs(n) * 7 * U * mag) + 3 * U * (np.abs(ds) + np.abs(skip))
    terms = np.abs(dy * n)
    b = 0.0 if base is None else base.astype(np.float64)
    dg = b + (dy * n).sum(0)
    return res | {"ds": (ds, 1.05 * eds), "dgamma": (dg, 1.05 * ((G(s.shape[0] + 1) + 4 * U) * (terms.sum(0) + np.abs(b))))}


# ------------------------------------------------------ gated feed-forward
def gate(act, z):
    """act(z), act'(z) and the sum of act''s absolute terms."""
    if act == "gelu":
        from scipy.special import ndtr
        cdf, pdf = ndtr(z), np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi)
        return z * cdf, cdf + z * pdf, cdf + np.abs(z) * pdf
    if act == "relu":
        on = (z > 0).astype(np.float64)
        return z * on, on, on
    s, o = sigmoid(z), sigmoid(-z)
    return (z * s, s * (1 + z * o), s * (1 + np.abs(z) * o)) if act == "silu" else (s, s * o, s * o)


def ffn_forward(X, W, b, act):
    """X [N, D], W [D, 2 F], b [2 F].  {name: (value, bound)} for Z and H.  A sum of
    pairs is kept to 2^-39 of the largest of X's row and of 32 columns of W."""
    X, W = X.astype(np.float64), W.astype(np.float64)
    Fh = W.shape[1] // 2
    bias = 0.0 if b is None else b.astype(np.float64)
    Z = X @ W + bias
    aX, aW = np.abs(X), np.abs(W)
    top = np.maximum.reduceat(aW.max(0).reshape(2, Fh), np.arange(0, Fh, 32), 1)
    top = np.repeat(top, 32, 1)[:, :Fh].reshape(-1)  # of the 32 columns that are packed together
    ez = G(X.shape[1]) * (aX @ aW) + F * (aX.max(1)[:, None] * aW.sum(0) + aX.sum(1)[:, None] * top) + 2 * U * (np.abs(Z) + np.abs(bias))
    y, d, _ = gate(act, Z[:, :Fh])
    H = y * Z[:, Fh:]
    eg, eu = ez[:, :Fh], ez[:, Fh:]
    # (ReLU and its like: a value next to the border moves by no more than its error)
    eh = np.maximum(np.abs(d), 1.0 if act == "relu" else 0.0) * eg * np.abs(Z[:, Fh:]) + eg * eg * np.abs(Z[:, Fh:]) + np.abs(y) * eu \
        + 16 * U * np.abs(H) + LOW * (1 + np.abs(Z[:, :Fh])) * np.abs(Z[:, Fh:])
    return {"Z": (Z, 1.05 * ez), "H": (H, 1.05 * eh)}


def ffn_backward(X, W, Z, dH, act, baseW=None, baseb=None):
    """From Z as the kernel is given it: dX, dW, db."""
    X, W, Z, dH = (t.astype(np.float64) for t in (X, W, Z, dH))
    Fh = dH.shape[1]
    y, d, md = gate(act, Z[:, :Fh])
    up = Z[:, Fh:]
    dZ = np.concatenate([dH * up * d, dH * y], 1)
    far = LOW * (1 + np.abs(Z[:, :Fh]))
    eZ = np.concatenate([np.abs(dH * up) * (16 * U * md + far), np.abs(dH) * (16 * U * np.abs(y) + far)], 1)
    aX, aW, aZ = np.abs(X), np.abs(W), np.abs(dZ)
    # dZ's scale is that of a bound of its largest, up to 8 times it here: |act| and |act'| are bounded by
    # max(z, 1) and 1.13 (z >= 0) and by (1 + |z|) e^z or (1 + |z|) e^(-z^2 / 2) (z < 0)
    mx, mw, mz = aX.max(), aW.max(), 8 * aZ.max()
    eX = G(2 * Fh) * (aZ @ aW.T) + eZ @ aW.T + F * (mz * aW.sum(1)[None, :] + mw * aZ.sum(1)[:, None])
    eW = G(X.shape[0]) * (aX.T @ aZ) + aX.T @ eZ + F * (mx * aZ.sum(0)[None, :] + mz * aX.sum(0)[:, None])
    bW = 0.0 if baseW is None else baseW.astype(np.float64)
    bb = 0.0 if baseb is None else baseb.astype(np.float64)
    dX, dW, db = dZ @ W.T, X.T @ dZ + bW, dZ.sum(0) + bb
    return {"dX": (dX, 1.05 * (eX + 2 * U * np.abs(dX))), "dW": (dW, 1.05 * (eW + 2 * U * (np.abs(dW) + np.abs(bW)))),
            "db": (db, 1.05 * (G(X.shape[0] + 1) * (aZ.sum(0) + np.abs(bb)) + eZ.sum(0)))}
