"""GPU tests of the Linear with cross-entropy where logits are far from zero."""
import numpy as np
import pytest

import lm_ops_ref as ref
from cppnet_amd import ops
from test_gpu_lm_ops import Buffers, host
from test_gpu_lm_ops_edges import ce_run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("level", [0.0, 2.0 ** 20, -2.0 ** 26, 2.0 ** 100])
@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("N,D,V", [(1, 5, 40), (40, 20, 700), (64, 33, 129), (65, 20, 700), (300, 70, 1500)])
def test_logits_at_any_level(gpu, N, D, V, reduction, level):
    """Rows of zeros: the logits are the bias, exactly, here `level` plus small
    multiples of its last place.  Softmax and loss take that as it is: they are
    off by the sum's rounding and the exponential's alone, at any level."""
    print(f"[linear ce] {N} rows {D} -> {V} {reduction} level {level}", flush=True)
    rng = np.random.default_rng(N + V)
    step = max(0.25, 2.0 ** -23 * abs(level))
    b = (level + step * rng.integers(-3, 4, V)).astype(np.float32)
    X, W = np.zeros((N, D), np.float32), rng.standard_normal((D, V)).astype(np.float32)
    t = rng.integers(-1, V, N).astype(np.int32)
    t[0] = 0
    buf = Buffers()
    got, _, (x, w, bb, tt) = ce_run(buf, X, W, b, t, reduction)
    z = b.astype(np.float64) - b.max()
    held, count = t >= 0, (t >= 0).sum() if reduction == "mean" else 1
    l = np.exp(z).sum()
    rows = np.where(held, np.log(l) - z[np.where(held, t, 0)], 0.0)
    # a row: the log sum's error, and the roundings of it and of its sum with the
    # difference of two logits, which is itself rounded
    row_lim = np.where(held, ref.g(V) + 4 * ref.U * (np.log(l) - z[np.where(held, t, 0)]), 0.0)
    loss_lim = (row_lim.sum() + ref.g(N) * np.abs(rows).sum()) / count
    ref.check("loss", got["loss"], np.array([rows.sum() / count]), np.array([loss_lim]))
    P = np.exp(z) / l
    G = np.where(held[:, None], P - (t[:, None] == np.arange(V)), 0) / count
    # a probability: its sum's error, and what its exponent's rounding and log2(e)'s make
    eG = (held[:, None] * (P * (ref.g(V) + 6 * ref.U * (np.log(l) - z)) + ref.F) + 4 * ref.U * np.abs(G) * count) / count
    ref.check("db", got["db"], G.sum(0), eG.sum(0) + ref.g(N) * np.abs(G).sum(0))
    Wd = W.astype(np.float64)
    ref.check("dX", got["dX"], G @ Wd.T, eG @ np.abs(Wd).T + ref.g(V) * (np.abs(G) @ np.abs(Wd).T) + ref.F * np.abs(Wd).max() * np.abs(G).sum(1, keepdims=True))
    assert (got["dW"] == 0).all()
    loss, lse = buf.empty(1), buf.empty(N)
    ops.linear_ce_forward(x, w, bb, tt, loss, lse, N, D, V, reduction)
    ref.check("loss of the forward", host(loss), np.array([rows.sum() / count]), np.array([loss_lim]))
    for a in (got["lse"], host(lse)):
        ref.check("lse", a, np.full(N, b.max() + np.log(l)), ref.g(V) + 4 * ref.U * (abs(level) + np.log(l)))
    buf.intact()
