"""The 64-bit forms that the GPU tests of the language-model operators use,
against autograd and differences (no GPU)."""
import numpy as np
import pytest
import torch

import lm_ops_ref as ref


@pytest.mark.parametrize("causal,k_len,q_start", [(False, None, None), (True, None, None), (True, [6, 0], [-2, 3]), (False, [4, 7], None)])
def test_attention_gradients(causal, k_len, q_start):
    B, H, KH, Sq, Sk, dh, scale = 2, 4, 2, 5, 7, 3, 0.6
    rng = np.random.default_rng(1)
    q, do = rng.standard_normal((2, B, H, Sq, dh))
    k, v = rng.standard_normal((2, B, KH, Sk, dh))
    ok = ref.allowed(B, Sq, Sk, causal, k_len, q_start)
    want = ref.attention(q, k, v, ok, scale, do)
    t = [torch.tensor(x, requires_grad=True) for x in (q, k, v)]
    wide = [t[0]] + [x.repeat_interleave(H // KH, 1) for x in t[1:]]
    mask = torch.tensor(ok)[:, None]
    e = torch.exp(scale * wide[0] @ wide[1].transpose(2, 3)) * mask
    l = e.sum(3, keepdim=True)
    out = (e / torch.where(l > 0, l, 1.0)) @ wide[2]
    np.testing.assert_allclose(want["out"][0], out.detach().numpy(), atol=1e-13)
    np.testing.assert_allclose(np.exp(want["lse"][0]), l[..., 0].detach().numpy(), rtol=1e-12)
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, t, torch.tensor(do))):
        np.testing.assert_allclose(want[name][0], g.numpy(), atol=1e-13)
    # along a direction, against a central difference
    for i, name in enumerate(("dq", "dk", "dv")):
        d = rng.standard_normal(t[i].shape)
        h = 1e-6
        side = []
        for s in (h, -h):
            x = [q, k, v]
            x[i] = x[i] + s * d
            side.append((ref.attention(*x, ok, scale)["out"][0] * do).sum())
        assert abs((side[0] - side[1]) / (2 * h) - (want[name][0] * d).sum()) < 1e-7


@pytest.mark.parametrize("mean", [True, False])
def test_linear_ce_gradients(mean):
    rng = np.random.default_rng(2)
    N, D, V = 6, 4, 9
    X, W, b, t = rng.standard_normal((N, D)), rng.standard_normal((D, V)), rng.standard_normal(V), np.array([3, -1, 8, 0, 9, 5])
    want = ref.linear_ce(X, W, b, t, mean)
    p = [torch.tensor(x, requires_grad=True) for x in (X, W, b)]
    z = torch.log_softmax(p[0] @ p[1] + p[2], 1)
    rows = [0, 2, 3, 5]
    loss = -z[rows, torch.tensor(t[rows])].sum() / (len(rows) if mean else 1)
    np.testing.assert_allclose(want["loss"][0], [loss.item()], rtol=1e-13)
    for name, g in zip(("dX", "dW", "db"), torch.autograd.grad(loss, p)):
        np.testing.assert_allclose(want[name][0], g.numpy(), atol=1e-14)
    d, h = rng.standard_normal(W.shape), 1e-6
    side = [ref.linear_ce(X, W + s * d, b, t, mean)["loss"][0][0] for s in (h, -h)]
    assert abs((side[0] - side[1]) / (2 * h) - (want["dW"][0] * d).sum()) < 1e-8


def test_embedding_gradient():
    ids, dY = np.array([2, -1, 0, 2, 5]), np.arange(10.0).reshape(5, 2)
    grad, _ = ref.embedding_grad(ids, dY, 4, 0.5)
    np.testing.assert_array_equal(grad, [[2, 2.5], [0, 0], [3, 4], [0, 0]])
    np.testing.assert_array_equal(ref.embedding(ids, np.eye(4), 2.0)[[0, 1, 4]], [[0, 0, 2, 0], [0] * 4, [0] * 4])


def test_check_sees_a_planted_error():
    X = np.ones((3, 4))
    ref.check("x", X, X, 1e-6)
    off = X.copy()
    off[1, 2] += 3e-6
    with pytest.raises(AssertionError, match="1 of 12 outside"):
        ref.check("x", off, X, 1e-6)
    off[1, 2] = np.nan
    with pytest.raises(AssertionError, match="not finite"):
        ref.check("x", off, X, 1e-6)
