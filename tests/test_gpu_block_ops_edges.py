"""GPU tests of a recurrent block's operators where their ranges end."""
import numpy as np
import pytest

import block_ops_ref as ref
from test_gpu_block_ops import Ffn

pytestmark = pytest.mark.gpu
U = ref.U


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
