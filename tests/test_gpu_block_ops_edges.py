"""GPU tests of a recurrent block's operators where their ranges end, on what is not finite,
and at positions past 32 bits."""
import numpy as np
import pytest
import torch

import block_ops_ref as ref
from cppnet_amd import ops
from test_gpu_block_ops import Ffn, Recurrence
from test_gpu_lm_ops import REF, SAMPLE

pytestmark = pytest.mark.gpu
U = ref.U


# --------------------------------------------------------------- recurrence
SHAPES = [(5, 1, 9), (5, 30, 9), (5, 600, 9), (2, 40000, 2)]  # the last in segments of its steps


def same(got, plain, where):
    for name in ("h", "dx", "df", "di"):
        if name in got:
            np.testing.assert_array_equal(got[name][where], plain[name][where])


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("B,S,D", SHAPES)
def test_recurrence_inputs_that_are_not_finite(gpu, B, S, D, gate, rows):
    """x at a step reaches h from there on and its own and later gates' gradients; f the
    gradients of earlier steps too.  No other sequence, and no step that it does not reach,
    changes a bit."""
    print(f"[recurrence] {B}x{S} D={D} rows={rows} gate={gate}", flush=True)
    r = Recurrence(B, S, D, rows, gate, True, None)
    plain, at = r.run(), S // 2
    r.x[1, at, 0], r.f[0, at, 1] = np.nan, np.nan
    got = r.run()
    clean = np.ones((B, S, D), bool)
    clean[1, :, 0] = clean[0, :, 1] = False
    same(got, plain, clean)
    for b, d in ((1, 0), (0, 1)):
        np.testing.assert_array_equal(got["h"][b, :at, d], plain["h"][b, :at, d])
        assert np.isnan(got["h"][b, at:, d]).all() and np.isnan(got["last"][b, d])
    np.testing.assert_array_equal(got["dx"][1, :, 0], plain["dx"][1, :, 0])  # has neither x nor h
    np.testing.assert_array_equal(got["dh0"][1, 0], plain["dh0"][1, 0])
    np.testing.assert_array_equal(got["df"][1, :at, 0], plain["df"][1, :at, 0])
    assert np.isnan(got["df"][1, at + (1 if gate else 0):, 0]).all()
    np.testing.assert_array_equal(got["dx"][0, at + 1:, 1], plain["dx"][0, at + 1:, 1])
    assert np.isnan(got["df"][0, :, 1]).all() and np.isnan(got["dx"][0, :at, 1]).all() and np.isnan(got["dh0"][0, 1])


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("B,S,D", SHAPES)
def test_recurrence_gradients_that_are_not_finite(gpu, B, S, D, gate, rows):
    """dh at a step reaches that step and the earlier ones of its sequence, dh_last all of
    them, and nothing else changes a bit."""
    print(f"[recurrence] {B}x{S} D={D} rows={rows} gate={gate}", flush=True)
    r = Recurrence(B, S, D, rows, gate, True, None)
    plain, at = r.run(), S // 2
    r.dh[1, at, 0], r.dh[0, at, 0], r.dl[1, 1] = np.nan, -np.inf, np.inf
    got = r.run()
    np.testing.assert_array_equal(got["h"], plain["h"])
    clean = np.ones((B, S, D), bool)
    clean[1, :at + 1, 0] = clean[0, :at + 1, 0] = clean[1, :, 1] = False
    same(got, plain, clean)
    for name in ("dx", "df", "di") if gate else ("dx", "df"):
        assert not np.isfinite(got[name][~clean]).any(), name
    assert not np.isfinite(got["dh0"][[1, 0, 1], [0, 0, 1]]).any()
    others = np.ones((B, D), bool)
    others[[1, 0, 1], [0, 0, 1]] = False
    np.testing.assert_array_equal(got["dh0"][others], plain["dh0"][others])


@pytest.mark.parametrize("rows", [REF, SAMPLE])
def test_recurrence_infinite_gates_in_segments(gpu, rows):
    """-inf drops the state and takes the input, +inf keeps the state, over every border."""
    B, S, D = 2, 40000, 2
    r = Recurrence(B, S, D, rows, False, True, None)
    r.f[:, 1::2], r.f[:, 0::2] = np.inf, -np.inf
    got = r.run()
    np.testing.assert_array_equal(got["h"], np.repeat(r.x[:, 0::2], 2, 1))
    assert (got["df"] == 0).all() and (got["dh0"] == 0).all() and (got["dx"][:, 1::2] == 0).all()
    r.f[:] = np.inf
    got = r.run()
    np.testing.assert_array_equal(got["h"], np.broadcast_to(r.h0[:, None], (B, S, D)))
    assert (got["dx"] == 0).all() and (got["df"] == 0).all()


# ------------------------------------------------------ gated feed-forward
@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("gate,up,dh", [
    (0.0, 3.2e38, 1.0),   # dgate = up / 2, but the largest |act'| times up is past the range
    (-0.0, -3.2e38, 1.0), (0.25, 3.1e38, -1.0),
    (1.2, 0.0, 3.0e38),   # dup = 0.77 (SiLU) or 0.88 (GELU) gate dh, but gate dh is past it
])
def test_ffn_gradients_next_to_the_end_of_the_range(gpu, act, gate, up, dh):
    """Z's gradient is finite where a multiple of it is not.  X and W are small enough for
    every product of it."""
    c = Ffn(300, 40, 64, act, True)
    c.X, c.W = (np.clip(t, -2, 2) / np.float32(8) for t in (c.X, c.W))
    c.Z[5, 7], c.Z[5, 64 + 7], c.dH[5, 7] = gate, up, dh
    got, want = c.backward(), ref.ffn_backward(c.X, c.W, c.Z, c.dH, act)
    for name, value in got.items():
        assert np.isfinite(value).all(), name
        ref.check(name, value, *want[name])
    c.buf.intact()


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("gate", [-10.0, -6.0, 0.125, 3.0])
def test_ffn_scale_of_the_gradient(gpu, act, gate):
    """Packed, dup is kept to F = 2^-39 of 2 times its largest at most: the documented bound.
    Rows of 2^-20 of the largest show it; each has one element of dup, so that no sum hides
    it.  Beside F: dup itself (16 u), what the pairs leave of a product and of a sum with
    zeros (g(0) = 16 u), two roundings."""
    N, D, F = 300, 40, 64
    c = Ffn(N, D, F, act, False)
    rng = np.random.default_rng(3)
    c.Z[:, :F], c.Z[:, F:] = gate, 0.0
    c.W = rng.uniform(0.5, 1.0, c.W.shape).astype(np.float32)
    c.dH[:] = 0
    rows, at = np.arange(N), np.arange(N) % F
    c.dH[rows, at] = np.where(rows == 0, 1.0, rng.uniform(0.5, 1.0, N) * 2.0 ** -20)
    got = c.backward()["dX"]
    y = ref.gate(act, np.float64(gate))[0] * c.dH[rows, at].astype(np.float64)
    want = y[:, None] * c.W[:, F + at].T.astype(np.float64)
    bound = 1.05 * (34 * U * np.abs(want) + 2 * ref.F * np.abs(y).max() * c.W.max())
    print("  worst share of the bound", ref.check("dX", got, want, bound))
    c.buf.intact()


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
@pytest.mark.parametrize("N,D,F", [(20, 8, 40), (300, 1100, 700)])  # fp32 MFMAs and the Linear's backward; packed
def test_ffn_gates_of_any_size(gpu, act, N, D, F):
    """Gates up to 1e30, whose squares are past fp32's range."""
    c = Ffn(N, D, F, act, True)
    far = np.float32(10.0) ** np.linspace(2, 30, F // 2).astype(np.float32)
    c.b = np.concatenate([far, -far, np.full(F, 3.0)]).astype(np.float32)
    c.X[:] = 0
    got, want = c.forward(), ref.ffn_forward(c.X, c.W, c.b, act)
    c.Z = np.broadcast_to(c.b, (N, 2 * F)).astype(np.float32).copy()
    c.X = np.random.default_rng(1).standard_normal(c.X.shape).astype(np.float32)
    want |= ref.ffn_backward(c.X, c.W, c.Z, c.dH, act)
    for name, value in (got | c.backward()).items():
        assert np.isfinite(value).all(), name
        ref.check(name, value, *want[name])
    c.buf.intact()


# ----------------------------------------------------- positions past 32 bits
def spare(gib):
    if torch.cuda.mem_get_info()[0] < gib << 30:
        pytest.skip(f"needs {gib} GiB of free device memory")


def filled(n, value):
    """n floats, filled in parts."""
    t = torch.empty(n, device="cuda")
    for i in range(0, n, 1 << 28):
        t[i:i + (1 << 28)] = value
    return t


@pytest.mark.parametrize("F", [1024, 2048])  # rows held, tiles
def test_norm_backward_past_32_bits(gpu, F):
    """2^31 + 2^21 values.  dy is one in the last column and zero elsewhere,
    so every element has a value of its own form:  n = s r, c = gamma n_last / F,
    ds_last = r (gamma - n_last c), ds_j = -r n_j c.  A value passes fewer than ten roundings;
    one of dgamma's terms fewer than 2000 (32 rows of a block, or 256, then up to 66000 blocks
    over 64 sums side by side, or 4100 over 8)."""
    spare(60)
    N = ((1 << 31) + (1 << 21)) // F
    tail = 5000
    s = filled(N * F, 1.0)
    s[-tail:] = 2.0  # the last rows' last feature
    size = np.where(np.arange(N) < N - tail, 1.0, 2.0)
    r = 1 / np.sqrt((F - 1 + size ** 2) / F + float(np.float32(1e-5)))
    rstd, gamma = torch.from_numpy(r.astype(np.float32)).cuda(), torch.full((F,), 3.0, device="cuda")
    dy = filled(N * F, 0.0)
    dy[-N:] = 1.0
    dx, dg = torch.empty(N * F, device="cuda"), torch.empty(F, device="cuda")
    ops.rms_norm_backward(s, rstd, gamma, dy, None, dx, None, dg, N, F)
    c = 3 * size * r / F
    np.testing.assert_allclose(dx[-N:].cpu().numpy(), r * (3 - size * r * c), rtol=20 * U)
    for f in (0, 511, F - 2):
        np.testing.assert_allclose(dx[f * N:(f + 1) * N].cpu().numpy(), -r * r * c, rtol=20 * U)
    got = dg.cpu().numpy()
    assert (got[:-1] == 0).all()
    np.testing.assert_allclose(got[-1], (size * r).sum(), rtol=2000 * U)


@pytest.mark.parametrize("rows", [REF, SAMPLE])
def test_recurrence_backward_past_32_bits(gpu, rows):
    """Four chains of 2^29 + 2^19 steps whose gate is one half: every value is a power of two
    times a small number, and exact."""
    spare(70)
    B, D = 2, 2
    n = (1 << 31) + (1 << 21)
    S = n // 4
    zero, h, dh = filled(n, 0.0), filled(n, 0.0), filled(n, 0.0)
    at = lambda b, t, d: b + B * t + B * S * d if rows == REF else t + S * b + B * S * d  # noqa: E731
    dh[at(0, 2, 0)], dh[at(1, S - 1, 1)], dh[at(0, S - 2, 1)] = 16.0, 64.0, 32.0
    h[at(1, S - 2, 1)], h[at(0, 0, 0)] = 8.0, 4.0
    last = torch.tensor([0.0, 128.0, 0.0, 0.0], device="cuda")  # [B, D] as it is stored: b + B d
    dx, df, dh0 = filled(n, 7.0), filled(n, 7.0), torch.empty(4, device="cuda")
    ops.linear_recurrence_backward(zero, zero, None, None, h, dh, last, dx, df, None, dh0, B, S, D, rows=rows)
    # g halves from step to step towards the first; dx = g / 2, df = g h_{t-1} / 4
    for b, t, d, g in ((0, 2, 0, 16.0), (1, S - 1, 1, 64.0), (0, S - 2, 1, 32.0), (1, S - 1, 0, 128.0)):
        for k in range(3):
            assert float(dx[at(b, t - k, d)]) == g / 2 ** k / 2, (b, t, d, k)
    for b, t, d in ((0, 3, 0), (0, S - 1, 1), (0, S - 1, 0), (0, S // 2, 0), (1, 0, 0), (1, 1, 1)):
        assert float(dx[at(b, t, d)]) == 0
    assert float(df[at(1, S - 1, 1)]) == 64.0 * 8 / 4 and float(df[at(0, 1, 0)]) == 8.0 * 4 / 4
    df[at(1, S - 1, 1)] = df[at(0, 1, 0)] = 0
    assert sum(float(df[i:i + (1 << 28)].abs().max()) for i in range(0, n, 1 << 28)) == 0
    np.testing.assert_array_equal(dh0.cpu().numpy(), [2.0, 0.0, 0.0, 0.0])


def test_ffn_past_32_bits(gpu):
    """2^20 + 3 rows and 1025 hidden features, so that Z has more than 2^31 values; all of them
    small whole numbers, and every sum below 2^24, so that both directions are exact.
      Z = (n % 3) (1 + j % 2) + 1 + j % 3 (ReLU keeps it), dH = 1 or -1 in turn."""
    spare(40)
    N, D, F = (1 << 20) + 3, 2, 1025
    n, j = torch.arange(N, device="cuda"), torch.arange(2 * F, device="cuda")
    X = torch.stack([n % 3, torch.ones_like(n)]).float()                     # (D, N)
    W = torch.stack([1 + j % 2, j % 3], 1).float().contiguous()              # (2 F, D)
    b = torch.ones(2 * F, device="cuda")
    H, Z = torch.empty(F, N, device="cuda"), torch.empty(2 * F, N, device="cuda")
    ops.gated_ffn_forward(X, W, b, H, Z, N, D, F, act="relu")

    def z_of(a, e):
        return X[0] * W[a:e, :1] + (W[a:e, 1:] + 1)
    step = 41  # 1025 = 25 41
    for a in range(0, F, step):
        g, u = z_of(a, a + step), z_of(F + a, F + a + step)
        assert torch.equal(Z[a:a + step], g) and torch.equal(Z[F + a:F + a + step], u)
        assert torch.equal(H[a:a + step], g * u)
    dH = H
    for f in range(F):
        dH[f] = 1 - 2 * ((n + f) % 2)
    dX, dW, db = torch.empty(D, N, device="cuda"), torch.empty(2 * F, D, device="cuda"), torch.empty(2 * F, device="cuda")
    ops.gated_ffn_backward(X, W, Z, dH, dX, dW, db, N, D, F, act="relu")
    wX = torch.zeros(D, N, device="cuda", dtype=torch.float64)
    for a in range(0, F, step):
        dg, du = (dH[a:a + step] * z_of(F + a, F + a + step)).double(), (dH[a:a + step] * z_of(a, a + step)).double()
        for at, dz in ((a, dg), (F + a, du)):
            w = W[at:at + step].double()
            for d in range(D):
                wX[d] += (dz * w[:, d:d + 1]).sum(0)
                assert torch.equal(dW[at:at + step, d].double(), (dz * X[d].double()).sum(1))
            assert torch.equal(db[at:at + step].double(), dz.sum(1))
    assert torch.equal(dX.double(), wX)
