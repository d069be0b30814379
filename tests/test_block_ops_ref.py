"""The 64-bit forms that the GPU tests of a recurrent block's operators use, against
autograd and differences (no GPU)."""
import numpy as np
import pytest
import torch

import block_ops_ref as ref


def differences(f, args, i, want, rng, tol, h=1e-6):
    d = rng.standard_normal(args[i].shape)
    side = []
    for s in (h, -h):
        a = list(args)
        a[i] = a[i] + s * d
        side.append(f(*a))
    assert abs((side[0] - side[1]) / (2 * h) - (want * d).sum()) < tol


@pytest.mark.parametrize("gate", [True, False])
@pytest.mark.parametrize("lengths", [None, [7, 0, 3]])
def test_recurrence_gradients(gate, lengths):
    rng = np.random.default_rng(1)
    B, S, D = 3, 7, 4
    x, f, i, dh = rng.standard_normal((4, B, S, D))
    h0, dl = rng.standard_normal((2, B, D))
    i = i if gate else None
    want = ref.recurrence(x, f, i, h0, lengths, dh, dl)
    t = [torch.tensor(v, requires_grad=True) for v in (x, f, h0)] + ([torch.tensor(i, requires_grad=True)] if gate else [])
    a = torch.sigmoid(t[1])
    w = torch.sigmoid(t[3]) if gate else 1 - a
    n, state, out = [S] * B if lengths is None else lengths, t[2], []
    for s in range(S):
        on = torch.tensor([[s < m] for m in n])
        state = torch.where(on, a[:, s] * state + w[:, s] * t[0][:, s], state)
        out.append(torch.where(on, state, torch.zeros_like(state)))
    h = torch.stack(out, 1)
    np.testing.assert_allclose(want["h"][0], h.detach().numpy(), atol=1e-14)
    np.testing.assert_allclose(want["last"][0], state.detach().numpy(), atol=1e-14)
    grads = torch.autograd.grad((h * torch.tensor(dh)).sum() + (state * torch.tensor(dl)).sum(), t)
    for name, g in zip(("dx", "df", "dh0", "di"), grads):
        np.testing.assert_allclose(want[name][0], g.numpy(), atol=1e-13)

    def loss(x, f, h0, i):
        r = ref.recurrence(x, f, i, h0, lengths)
        return (r["h"][0] * dh).sum() + (r["last"][0] * dl).sum()
    for k, name in enumerate(("dx", "df", "dh0") + (("di",) if gate else ())):
        differences(loss, [x, f, h0, i], k, want[name][0], rng, 1e-7)


def test_sigmoid_keeps_both_tails():
    z = np.array([-700.0, -40.0, -1.0, 0.0, 1.0, 40.0])
    np.testing.assert_allclose(ref.sigmoid(z), torch.sigmoid(torch.tensor(z)).numpy(), rtol=1e-14)


@pytest.mark.parametrize("skip", [True, False])
def test_norm_gradients(skip):
    rng = np.random.default_rng(2)
    N, F = 5, 6
    s, dy, dsum = rng.standard_normal((3, N, F))
    g = rng.standard_normal(F)
    want = ref.rms_norm(s, g, 1e-3, dy, dsum if skip else None)
    t = [torch.tensor(s, requires_grad=True), torch.tensor(g, requires_grad=True)]
    y = t[0] * torch.rsqrt((t[0] ** 2).mean(1, keepdim=True) + float(np.float32(1e-3))) * t[1]
    np.testing.assert_allclose(want["y"][0], y.detach().numpy(), rtol=1e-13)
    total = (y * torch.tensor(dy)).sum() + ((t[0] * torch.tensor(dsum)).sum() if skip else 0)
    for name, grad in zip(("ds", "dgamma"), torch.autograd.grad(total, t)):
        np.testing.assert_allclose(want[name][0], grad.numpy(), atol=1e-13)
    loss = lambda s, g: (ref.rms_norm(s, g, 1e-3)["y"][0] * dy).sum() + ((s * dsum).sum() if skip else 0)  # noqa: E731
    differences(loss, [s, g], 0, want["ds"][0], rng, 1e-7)
    differences(loss, [s, g], 1, want["dgamma"][0], rng, 1e-7)


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
def test_ffn_gradients(act):
    rng = np.random.default_rng(3)
    N, D, F = 5, 4, 3
    X, W, b, dH = rng.standard_normal((N, D)), rng.standard_normal((D, 2 * F)), rng.standard_normal(2 * F), rng.standard_normal((N, F))
    fwd = ref.ffn_forward(X, W, b, act)
    want = ref.ffn_backward(X, W, fwd["Z"][0], dH, act)
    t = [torch.tensor(v, requires_grad=True) for v in (X, W, b)]
    z = t[0] @ t[1] + t[2]
    fn = {"silu": torch.nn.functional.silu, "gelu": torch.nn.functional.gelu, "sigmoid": torch.sigmoid, "relu": torch.relu}[act]
    H = fn(z[:, :F]) * z[:, F:]
    np.testing.assert_allclose(fwd["H"][0], H.detach().numpy(), atol=1e-13)
    for name, g in zip(("dX", "dW", "db"), torch.autograd.grad((H * torch.tensor(dH)).sum(), t)):
        np.testing.assert_allclose(want[name][0], g.numpy(), atol=1e-13)
    loss = lambda X, W, b: (ref.ffn_forward(X, W, b, act)["H"][0] * dH).sum()  # noqa: E731
    for k, name in enumerate(("dX", "dW", "db")):
        differences(loss, [X, W, b], k, want[name][0], rng, 1e-7)


def test_mask_is_the_documented_one():
    """splitmix64's published output for a state of 0 and its step, and the fp32 border."""
    def word(z):
        M = (1 << 64) - 1
        z = ((z ^ (z >> 30)) * 0xBF58476D1CE4E5B9) & M
        z = ((z ^ (z >> 27)) * 0x94D049BB133111EB) & M
        return z ^ (z >> 31)
    golden = 0x9E3779B97F4A7C15
    assert word(golden) == 0xE220A8397B1DCDAF and word(2 * golden & ((1 << 64) - 1)) == 0x6E789E6AA1B965F4
    for p in (0.0, 0.3, 0.999):
        want = [np.float32(word((77 + (5 + j) * golden) & ((1 << 64) - 1)) >> 40) * np.float32(2.0 ** -24)
                < np.float32(1) - np.float32(p) for j in range(300)]
        np.testing.assert_array_equal(ref.kept(300, p, 77, 5), want)
