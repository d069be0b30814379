"""GPU tests of a recurrent block's operators where their ranges end."""
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
