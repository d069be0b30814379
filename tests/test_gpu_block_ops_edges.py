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
