"""GPU tests of the operators of a recurrent language model's block against their
64-bit forms in block_ops_ref.py, whose bounds are derived there."""
import numpy as np
import pytest
import torch

import block_ops_ref as ref
from cppnet_amd import ops
from test_gpu_lm_ops import REF, SAMPLE, Buffers, host, logical, stored

pytestmark = pytest.mark.gpu
U = ref.U


# --------------------------------------------------------------- recurrence
REC = [  # B, S, D, rows, input gate, state, lengths
    (1, 1, 1, SAMPLE, False, False, None), (8, 1, 33, SAMPLE, False, True, None), (8, 1, 33, REF, True, True, [1, 0] * 4),
    (3, 2, 5, SAMPLE, True, True, None), (3, 3, 70, SAMPLE, False, False, [3, 0, 2]), (5, 17, 9, SAMPLE, False, True, None),
    (2, 64, 11, SAMPLE, True, False, None), (2, 127, 7, SAMPLE, False, True, [127, 64]), (3, 128, 40, SAMPLE, False, False, None),
    (3, 129, 5, SAMPLE, False, True, [129, 128, 1]), (2, 256, 6, SAMPLE, True, True, None), (2, 257, 6, SAMPLE, False, True, None),
    (4, 1001, 3, SAMPLE, True, True, [1001, 0, 512, 513]), (1, 1024, 3, REF, False, True, None),
    (2, 5003, 4, SAMPLE, False, False, [5003, 4097]), (70, 300, 61, SAMPLE, False, False, None),  # a wave a chain
    (1, 40001, 3, SAMPLE, False, True, None), (2, 35000, 2, SAMPLE, True, True, [35000, 20001]),  # in segments
    (2, 1, 3, REF, False, True, None), (2, 31, 5, REF, True, True, None), (2, 301, 5, REF, False, True, [301, 100]),
    (5, 1001, 7, REF, True, True, [1001, 0, 7, 512, 999]), (32, 40, 6, REF, False, False, None), (33, 17, 3, REF, False, True, None),
    (64, 40, 3, REF, True, False, None), (70, 33, 4, REF, False, True, [33, 0] * 35), (130, 9, 2, REF, True, True, None),
    (21, 70, 300, REF, False, True, None), (2, 20001, 2, REF, False, True, [20001, 11111]),  # in segments
    (40, 3001, 1, REF, True, True, None), (1, 2, 4096, REF, False, False, None),
]


class Recurrence:
    """Operands of one case on logical arrays and on the device; steps past a sample's
    length hold NaN everywhere."""

    def __init__(self, B, S, D, rows, gate, state, lengths, seed=0, f=None):
        rng = np.random.default_rng(seed + B * 7 + S * 3 + D)
        draw = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.dims, self.rows, self.lengths = (B, S, D), rows, lengths
        self.x, self.i, self.dh = draw(B, S, D), draw(B, S, D) if gate else None, draw(B, S, D)
        self.f = (2 + 1.5 * draw(B, S, D)) if f is None else np.broadcast_to(np.float32(f), (B, S, D)).copy()
        self.h0, self.dl = (draw(B, D), draw(B, D)) if state else (None, None)
        n = np.full(B, S) if lengths is None else np.clip(lengths, 0, S)
        self.past = np.broadcast_to(np.arange(S)[None, :, None] >= n[:, None, None], (B, S, D))
        self.buf = Buffers()

    def seq(self, a):
        if a is None:
            return None
        a = np.where(self.past, np.float32(np.nan), a)
        return self.buf.new(stored(a, self.rows))

    def state(self, a):
        return None if a is None else self.buf.new(a.T)

    def run(self, what=("forward", "backward")):
        B, S, D = self.dims
        how = {"rows": self.rows}
        if self.lengths is not None:
            how["seq_len"] = self.buf.new(self.lengths, np.int32)
        x, f, i, h0 = self.seq(self.x), self.seq(self.f), self.seq(self.i), self.state(self.h0)
        h, last = self.buf.empty(B * S * D), self.buf.empty(B * D)
        ops.linear_recurrence_forward(x, f, i, h0, h, last, B, S, D, **how)
        out = {"h": self.logical(h), "last": host(last).reshape(D, B).T}
        if "backward" in what:
            dx, df, di = (self.buf.empty(B * S * D) for _ in range(3))
            di = di if i is not None else None
            dh0 = self.buf.empty(B * D)
            ops.linear_recurrence_backward(x, f, i, h0, h, self.seq(self.dh), self.state(self.dl), dx, df, di, dh0, B, S, D, **how)
            out |= {"dx": self.logical(dx), "df": self.logical(df), "dh0": host(dh0).reshape(D, B).T}
            if di is not None:
                out["di"] = self.logical(di)
        self.buf.intact()
        return out

    def logical(self, t):
        return logical(host(t), *self.dims, self.rows)

    def want(self):
        return ref.recurrence(self.x, self.f, self.i, self.h0, self.lengths, self.dh, self.dl)


@pytest.mark.parametrize("B,S,D,rows,gate,state,lengths", REC)
def test_recurrence(gpu, B, S, D, rows, gate, state, lengths):
    print(f"[recurrence] {B}x{S} D={D} rows={rows} gate={gate} state={state}", flush=True)
    r = Recurrence(B, S, D, rows, gate, state, lengths)
    got, want = r.run(), r.want()
    for name, (value, bound) in want.items():
        print(f"  {name}: worst share of the bound", ref.check(name, got[name], value, bound))
    for name in ("h", "dx", "df", "di"):
        if name in got:
            assert (got[name][r.past] == 0).all(), f"{name}: steps past the length are not zero"
    again = r.run()
    for name in got:
        np.testing.assert_array_equal(got[name], again[name])


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("f", [-30.0, -8.0, 8.0, 12.0, 16.0, 30.0])
def test_recurrence_gates_far_out(gpu, f, rows):
    """Gates that forget or remember nearly everything, alike at every step: an error in
    the factor would add up over all of them."""
    r = Recurrence(2, 9001, 2, rows, False, True, None, f=f)
    r.x = np.ones_like(r.x)
    got, want = r.run(), r.want()
    for name, (value, bound) in want.items():
        ref.check(name, got[name], value, bound)
    # towards 1 as far as the gate lets it
    assert np.abs(got["h"] - want["h"][0]).max() < 100 * U * max(1.0, np.abs(r.h0).max())


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("S", [5, 200, 700])
def test_recurrence_infinite_gates(gpu, S, rows):
    """-inf drops the state and takes the input, +inf keeps the state."""
    B, D = 3, 4
    r = Recurrence(B, S, D, rows, False, True, None)
    r.f[:, 1::2], r.f[:, 0::2] = np.inf, -np.inf
    got = r.run()
    want = np.repeat(r.x[:, 0::2], 2, 1)[:, :S]
    np.testing.assert_array_equal(got["h"], want)
    assert (got["df"] == 0).all() and (got["dh0"] == 0).all()
    r.f[:] = np.inf
    got = r.run()
    np.testing.assert_array_equal(got["h"], np.broadcast_to(r.h0[:, None], (B, S, D)))
    assert (got["dx"] == 0).all() and (got["df"] == 0).all()


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("S", [1, 30, 200, 600])
def test_recurrence_keeps_what_is_not_finite_to_its_sequence(gpu, S, rows):
    r = Recurrence(5, S, 9, rows, False, True, None)
    plain = r.run()
    at = S // 2
    r.x[1, at, 3], r.f[2, at, 4], r.x[3, at, :] = np.nan, np.nan, np.inf
    got = r.run()
    touched = np.zeros((5, S, 9), bool)
    touched[1, at:, 3] = touched[2, at:, 4] = touched[3, at:, :] = True
    np.testing.assert_array_equal(got["h"][~touched], plain["h"][~touched])
    assert np.isnan(got["h"][1, at:, 3]).all() and np.isnan(got["h"][2, at:, 4]).all()
    assert not np.isfinite(got["h"][3, at:]).any()
    untouched = [(b, d) for b in range(5) for d in range(9) if (b, d) not in ((1, 3), (2, 4)) and b != 3]
    for b, d in untouched:
        for name in ("dx", "df"):
            np.testing.assert_array_equal(got[name][b, :, d], plain[name][b, :, d])


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("S,D", [(1, 40), (50, 7), (3000, 3), (40000, 2)])
def test_recurrence_states_in_place(gpu, S, D, rows):
    """h_last over h0 and dh0 over dh_last, and steps one after the other as one call."""
    B = 2
    r = Recurrence(B, S, D, rows, True, True, [S, max(0, S - 3)])
    got = r.run()
    x, f, i, dh = (r.seq(t) for t in (r.x, r.f, r.i, r.dh))
    n = r.buf.new(r.lengths, np.int32)
    s, ds, h = r.state(r.h0), r.state(r.dl), r.buf.empty(B * S * D)
    ops.linear_recurrence_forward(x, f, i, s, h, s, B, S, D, seq_len=n, rows=rows)
    np.testing.assert_array_equal(host(s).reshape(D, B).T, got["last"])
    np.testing.assert_array_equal(r.logical(h), got["h"])
    g = [r.buf.empty(B * S * D) for _ in range(3)]
    ops.linear_recurrence_backward(x, f, i, r.state(r.h0), h, dh, ds, *g, ds, B, S, D, seq_len=n, rows=rows)
    np.testing.assert_array_equal(host(ds).reshape(D, B).T, got["dh0"])
    np.testing.assert_array_equal(r.logical(g[1]), got["df"])
    r.buf.intact()


@pytest.mark.parametrize("rows", [REF, SAMPLE])
def test_recurrence_step_by_step_is_the_whole_sequence(gpu, rows):
    B, S, D = 3, 40, 20
    r = Recurrence(B, S, D, rows, False, True, None)
    want = r.want()["h"]
    state = r.state(r.h0)
    for t in range(S):
        x, f = (r.buf.new(a[:, t].T) for a in (r.x, r.f))
        h = r.buf.empty(B * D)
        ops.linear_recurrence_forward(x, f, None, state, h, state, B, 1, D, rows=rows)
        ref.check(f"h[{t}]", host(h).reshape(D, B).T, want[0][:, t], want[1][:, t])
        np.testing.assert_array_equal(host(h), host(state))
    # the backward the same way: u goes from step to step
    whole = r.want()
    u = r.state(r.dl)
    hist = np.concatenate([r.h0[:, None], want[0][:, :-1].astype(np.float32)], 1)
    for t in reversed(range(S)):
        x, f, dh, h0 = (r.buf.new(a[:, t].T) for a in (r.x, r.f, r.dh, hist))
        dx, df = r.buf.empty(B * D), r.buf.empty(B * D)
        ops.linear_recurrence_backward(x, f, None, h0, r.buf.new(want[0][:, t].T), dh, u, dx, df, None, u, B, 1, D, rows=rows)
        ref.check(f"dx[{t}]", host(dx).reshape(D, B).T, whole["dx"][0][:, t], whole["dx"][1][:, t])
        ref.check(f"df[{t}]", host(df).reshape(D, B).T, whole["df"][0][:, t], whole["df"][1][:, t])
    r.buf.intact()


def test_recurrence_lengths_past_the_ends(gpu):
    """Lengths below 0 and above S are cut; without a state a sample of no steps ends in zeros."""
    r = Recurrence(4, 150, 3, SAMPLE, False, False, [-5, 400, 0, np.iinfo(np.int32).max])
    got, want = r.run(), r.want()
    for name, (value, bound) in want.items():
        ref.check(name, got[name], value, bound)
    assert (got["last"][[0, 2]] == 0).all()


# ------------------------------------------------------------------ dropout
@pytest.mark.parametrize("n", [1, 3, 4, 1025, 70001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.999])
def test_dropout_seeded(gpu, n, p):
    rng = np.random.default_rng(n)
    x = rng.standard_normal(n).astype(np.float32)
    seed, offset, count = (1 << 63) + 12345, 77, (1 << 40) + 5
    buf = Buffers()
    t, y = buf.new(x), buf.empty(n)
    ops.dropout_seeded(t, y, p, seed, offset)
    want = ref.dropped(x, p, seed, offset)
    np.testing.assert_array_equal(host(y), want)
    # the stored mask's call draws the same
    z, mask = buf.empty(n), torch.empty(n, dtype=torch.uint8, device="cuda")
    ops.dropout_forward(t, z, mask, p, seed, offset)
    np.testing.assert_array_equal(host(z), host(y))
    counter = torch.tensor([count], dtype=torch.int64, device="cuda")
    ops.dropout_seeded(t, y, p, seed, offset, counter)
    np.testing.assert_array_equal(host(y), ref.dropped(x, p, seed, offset + count))
    ops.dropout_seeded(t, t, p, seed, offset)  # in place
    np.testing.assert_array_equal(host(t), want)
    buf.intact()


def test_dropout_drops_what_is_not_finite(gpu):
    n, p = 5000, 0.5
    keep = ref.kept(n, p, 3, 0)
    x = np.where(keep, np.float32(2), np.float32(np.nan)).astype(np.float32)
    x[~keep & (np.arange(n) % 2 == 0)] = np.inf
    y = torch.empty(n, device="cuda")
    ops.dropout_seeded(torch.from_numpy(x).cuda(), y, p, 3)
    got = host(y)
    np.testing.assert_array_equal(got, np.where(keep, np.float32(4), np.float32(0)))
    assert not np.signbit(got).any()


def test_dropout_counter_goes_on_and_wraps(gpu):
    c = torch.tensor([5], dtype=torch.int64, device="cuda")
    ops.dropout_advance(c, 1 << 40)
    assert host(c)[0] == 5 + (1 << 40)
    ops.dropout_advance(c, (1 << 64) - 10)
    assert host(c)[0] == (1 << 40) - 5
    x, y, z = (torch.ones(4096, device="cuda") for _ in range(3))
    ops.dropout_seeded(x, y, 0.5, 9, (1 << 64) - 100)  # positions run past 2^64
    np.testing.assert_array_equal(host(y), ref.dropped(np.ones(4096, np.float32), 0.5, 9, (1 << 64) - 100))


def test_dropout_long(gpu):
    """More elements than one round of the grid, and the share that is kept."""
    n, p = 40_000_003, 0.3
    x, y = torch.ones(n, device="cuda"), torch.empty(n, device="cuda")
    ops.dropout_seeded(x, y, p, 11)
    scale = np.float32(1) / (np.float32(1) - np.float32(p))
    got = host(y)
    assert set(np.unique(got)) == {np.float32(0), scale}
    assert abs((got > 0).mean() - (1 - p)) < 6 * np.sqrt(p * (1 - p) / n)
    np.testing.assert_array_equal(got[-1000:] > 0, ref.kept(1000, p, 11, n - 1000))


# --------------------------------------------------------------------- norm
NORM = [  # N, F, p, residual, dsum
    (1, 1, 0.0, False, False), (1, 512, 0.0, True, True), (3, 7, 0.3, True, True), (2, 4096, 0.0, True, False),
    (8, 512, 0.1, True, True), (17, 100, 0.0, False, True), (32, 33, 0.5, True, True), (33, 1024, 0.0, True, True),
    (64, 513, 0.1, False, True), (257, 512, 0.1, True, True), (100, 2000, 0.0, True, True), (1000, 40, 0.0, True, False),
    (45, 4099, 0.1, True, True), (70, 2049, 0.0, True, True), (5, 20001, 0.2, True, True), (20000, 12, 0.0, True, True),
    (16500, 64, 0.1, True, True), (1300, 6001, 0.1, True, True), (2100, 8300, 0.0, True, False),  # several tiles a block
    # features a multiple of 8, up to 1024, and next to that
    (34, 8, 0.0, True, True), (95, 24, 0.2, True, True), (63, 128, 0.0, False, False), (65, 136, 0.1, True, True),
    (100, 256, 0.0, True, True), (131, 336, 0.1, True, False), (96, 384, 0.0, False, True), (70, 520, 0.0, True, True),
    (47, 768, 0.3, True, True), (6001, 1024, 0.1, True, True), (6040, 776, 0.0, True, True), (700, 640, 0.0, True, True),
    (300, 1032, 0.0, True, True), (1000, 39, 0.1, True, True), (20000, 13, 0.0, True, True), (16500, 65, 0.1, True, True),
    (77, 9, 0.0, True, True), (300, 333, 0.1, True, True), (513, 517, 0.0, True, False), (6100, 1021, 0.1, True, True),
    (90, 771, 0.0, True, True), (20000, 5, 0.1, True, True), (70, 3, 0.0, False, True),
]


def sum_of(x, residual, p, seed, position):
    """s, bit for bit; [N, F] with positions along the rows first."""
    d = ref.dropped(np.ascontiguousarray(x.T).ravel(), p, seed, position).reshape(x.T.shape).T if p else x
    return d if residual is None else (residual + d).astype(np.float32)


class Norm:
    def __init__(self, N, F, p, residual, dsum, seed=0):
        rng = np.random.default_rng(seed + N * 3 + F)
        draw = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.N, self.F, self.p = N, F, p
        self.x, self.gamma, self.dy, self.base = draw(N, F), 1 + draw(F), draw(N, F), draw(F)
        self.residual = 3 * draw(N, F) if residual else None
        self.dsum = draw(N, F) if dsum else None
        self.seed, self.offset, self.count = 99, 1234, (1 << 33) + 1
        self.buf = Buffers()

    def mat(self, a):
        return None if a is None else self.buf.new(a.T)

    def logical(self, t):
        return host(t).reshape(self.F, self.N).T

    def run(self, eps=1e-5, accumulate=False):
        N, F, new, empty = self.N, self.F, self.buf.new, self.buf.empty
        counter = torch.tensor([self.count], dtype=torch.int64, device="cuda")
        how = {"p": self.p, "seed": self.seed, "offset": self.offset, "counter": counter} if self.p else {}
        y, s, rstd, gamma = empty(N * F), empty(N * F), empty(N), new(self.gamma)
        ops.rms_norm_forward(self.mat(self.x), self.mat(self.residual), gamma, y, s, rstd, N, F, eps, **how)
        dx, dr, dg = empty(N * F), empty(N * F), new(self.base) if accumulate else empty(F)
        ops.rms_norm_backward(s, rstd, gamma, self.mat(self.dy), self.mat(self.dsum), dx, dr, dg, N, F, accumulate=accumulate, **how)
        self.buf.intact()
        return {"sum": self.logical(s), "y": self.logical(y), "rstd": host(rstd).copy(), "dx": self.logical(dx),
                "ds": self.logical(dr), "dgamma": host(dg).copy()}


@pytest.mark.parametrize("N,F,p,residual,dsum", NORM)
def test_norm(gpu, N, F, p, residual, dsum):
    print(f"[norm] {N}x{F} p={p}", flush=True)
    c = Norm(N, F, p, residual, dsum)
    for accumulate in (False, True):
        got = c.run(accumulate=accumulate)
        s = sum_of(c.x, c.residual, p, c.seed, c.offset + c.count)
        np.testing.assert_array_equal(got["sum"], s)
        want = ref.rms_norm(s, c.gamma, 1e-5, c.dy, c.dsum, c.base if accumulate else None)
        for name, (value, bound) in want.items():
            print(f"  {name}: worst share of the bound", ref.check(name, got[name], value, bound))
        np.testing.assert_array_equal(got["dx"], sum_of(got["ds"], None, p, c.seed, c.offset + c.count))
        again = c.run(accumulate=accumulate)
        for name in got:
            np.testing.assert_array_equal(got[name], again[name])


@pytest.mark.parametrize("N,F", [(3, 40), (40, 300), (50, 3000)])
def test_norm_optional_outputs(gpu, N, F):
    """Without sum, rstd and dresidual, over the residual in place, and as two calls."""
    c = Norm(N, F, 0.25, True, True)
    full = c.run()
    how = {"p": c.p, "seed": c.seed, "offset": c.offset + c.count}
    y, gamma = c.buf.empty(N * F), c.buf.new(c.gamma)
    ops.rms_norm_forward(c.mat(c.x), c.mat(c.residual), gamma, y, None, None, N, F, **how)
    np.testing.assert_array_equal(c.logical(y), full["y"])
    stream = c.mat(c.residual)
    ops.rms_norm_forward(c.mat(c.x), stream, gamma, y, stream, None, N, F, **how)
    np.testing.assert_array_equal(c.logical(y), full["y"])
    np.testing.assert_array_equal(c.logical(stream), full["sum"])
    d, rstd = c.buf.empty(N * F), c.buf.empty(N)
    ops.dropout_seeded(c.mat(c.x), d, c.p, c.seed, c.offset + c.count)
    ops.rms_norm_forward(d, c.mat(c.residual), gamma, y, stream, rstd, N, F)
    np.testing.assert_array_equal(c.logical(y), full["y"])
    dx, dg = c.buf.empty(N * F), c.buf.empty(F)
    ops.rms_norm_backward(stream, rstd, gamma, c.mat(c.dy), c.mat(c.dsum), dx, None, dg, N, F, **how)
    np.testing.assert_array_equal(c.logical(dx), full["dx"])
    np.testing.assert_array_equal(host(dg), full["dgamma"])
    c.buf.intact()


@pytest.mark.parametrize("F", [64, 3000])
@pytest.mark.parametrize("size", [1e-30, 1e-8, 1e15, 3e37])
def test_norm_of_any_size(gpu, size, F):
    c = Norm(37, F, 0.0, False, False)
    c.x *= np.float32(size)
    c.x[5] = 0
    got = c.run(eps=1e-5)
    want = ref.rms_norm(c.x, c.gamma, 1e-5, c.dy, None)
    for name, (value, bound) in want.items():
        # what fp32 holds of values below its normal range, times what they are multiplied with
        ref.check(name, got[name], value, bound + 2.0 ** -149 * (1 + np.abs(c.gamma).max()) * (np.abs(c.x).max() + 1))
    assert (got["y"][5] == 0).all()


def test_norm_rows_that_are_not_finite_stay_alone(gpu):
    c = Norm(70, 300, 0.0, True, True)
    plain = c.run()
    c.x[3, 7], c.x[40, 200], c.x[66, 0] = np.nan, np.inf, -np.inf
    got = c.run()
    others = np.setdiff1d(np.arange(70), [3, 40, 66])
    for name in ("y", "sum", "rstd", "dx", "ds"):
        np.testing.assert_array_equal(got[name][others], plain[name][others])
    assert np.isnan(got["y"][[3, 40, 66]]).all()
    # and a dropped NaN is nobody's
    c = Norm(70, 300, 0.5, True, True)
    keep = ref.kept(70 * 300, 0.5, c.seed, c.offset + c.count).reshape(300, 70).T
    plain = c.run()
    c.x = np.where(keep, c.x, np.float32(np.nan))
    got = c.run()
    for name in got:
        np.testing.assert_array_equal(got[name], plain[name])


# ------------------------------------------------------ gated feed-forward
FFN = [  # N, D, F, activation, bias
    (1, 1, 1, "silu", False), (1, 512, 2048, "silu", False), (4, 33, 17, "gelu", True), (16, 130, 64, "relu", True),
    (17, 300, 100, "sigmoid", False), (33, 64, 65, "silu", True), (64, 257, 31, "gelu", True), (65, 33, 31, "silu", True),
    (100, 64, 128, "gelu", False), (130, 1, 40, "silu", True), (70, 40, 1, "relu", False), (257, 100, 300, "silu", True),
    (300, 513, 97, "gelu", True), (1021, 257, 130, "silu", False), (1300, 96, 64, "sigmoid", True), (2050, 40, 33, "relu", True),
    (70, 1100, 33, "silu", True), (9, 1500, 12, "gelu", False), (600, 33, 400, "silu", False),
    # the forward on packed operands too
    (1021, 257, 1300, "silu", False), (2050, 300, 700, "relu", True), (3000, 130, 1000, "gelu", True),
    (700, 1100, 600, "sigmoid", False), (5000, 33, 1900, "silu", True), (513, 1000, 999, "gelu", False),
    # every size of tile, with sums that are split and whole
    (520, 2100, 260, "relu", True), (300, 4100, 260, "sigmoid", False), (1000, 130, 4000, "silu", True),
    (1000, 4100, 1050, "gelu", False), (4100, 4100, 20, "silu", True), (65, 2100, 4000, "gelu", True),
    (4100, 130, 4000, "relu", False),
]


class Ffn:
    def __init__(self, N, D, F, act, bias, seed=0):
        rng = np.random.default_rng(seed + N + 5 * D + F)
        draw = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        self.N, self.D, self.F, self.act = N, D, F, act
        self.X, self.W, self.b = draw(N, D), draw(D, 2 * F) / np.float32(np.sqrt(D)), 0.3 * draw(2 * F) if bias else None
        self.dH, self.Z, self.baseW, self.baseb = draw(N, F), 1.5 * draw(N, 2 * F), draw(D, 2 * F), draw(2 * F)
        self.buf = Buffers()

    def mat(self, a):
        return None if a is None else self.buf.new(a.T)

    def out(self, t, cols):
        return host(t).reshape(cols, -1).T

    def forward(self, keep=True):
        N, D, F = self.N, self.D, self.F
        H, Z = self.buf.empty(N * F), self.buf.empty(N * 2 * F) if keep else None
        ops.gated_ffn_forward(self.mat(self.X), self.mat(self.W), None if self.b is None else self.buf.new(self.b), H, Z, N, D, F,
                              act=self.act)
        return {"H": self.out(H, F)} | ({"Z": self.out(Z, 2 * F)} if keep else {})

    def backward(self, accumulate=False):
        N, D, F = self.N, self.D, self.F
        dX = self.buf.empty(N * D)
        dW = self.mat(self.baseW) if accumulate else self.buf.empty(D * 2 * F)
        db = None if self.b is None else self.buf.new(self.baseb) if accumulate else self.buf.empty(2 * F)
        ops.gated_ffn_backward(self.mat(self.X), self.mat(self.W), self.mat(self.Z), self.mat(self.dH), dX, dW, db, N, D, F,
                               act=self.act, accumulate=accumulate)
        got = {"dX": self.out(dX, D), "dW": self.out(dW, 2 * F)}
        return got | ({} if db is None else {"db": host(db).copy()})

    def check(self, accumulate=False):
        got, want = self.forward(), ref.ffn_forward(self.X, self.W, self.b, self.act)
        back = self.backward(accumulate)
        want |= ref.ffn_backward(self.X, self.W, self.Z, self.dH, self.act, self.baseW if accumulate else None,
                                 self.baseb if accumulate else None)
        for name, value in (got | back).items():
            print(f"  {name}: worst share of the bound", ref.check(name, value, *want[name]))
        self.buf.intact()
        return got | back


@pytest.mark.parametrize("N,D,F,act,bias", FFN)
def test_ffn(gpu, N, D, F, act, bias):
    print(f"[ffn] {N}x{D} -> {F} {act} bias={bias}", flush=True)
    c = Ffn(N, D, F, act, bias)
    got = c.check()
    again = c.forward() | c.backward()
    for name in got:
        np.testing.assert_array_equal(got[name], again[name])
    np.testing.assert_array_equal(c.forward(keep=False)["H"], got["H"])
    c.check(accumulate=True)


@pytest.mark.parametrize("N,D,F", [(20, 70, 96), (200, 70, 96), (1100, 260, 1312)])
def test_ffn_rows_and_columns_of_any_size(gpu, N, D, F):
    """Forward: a row of X and a block of W's columns have scales of their own."""
    c = Ffn(N, D, F, "silu", False)
    c.X *= np.float32(2.0) ** np.random.default_rng(1).integers(-60, 30, (N, 1)).astype(np.float32)
    c.W[:, :32] *= np.float32(2.0 ** -40)
    c.W[:, F:F + 32] *= np.float32(2.0 ** 20)
    got, want = c.forward(), ref.ffn_forward(c.X, c.W, None, "silu")
    for name in got:
        ref.check(name, got[name], *want[name])


@pytest.mark.parametrize("act", ["silu", "gelu", "sigmoid", "relu"])
def test_ffn_gates_far_out(gpu, act):
    """Pre-activations from -120 to 120, zero among them, and what is left of them."""
    c = Ffn(66, 8, 40, act, True)
    c.X[:], c.W[:] = 0, 0
    c.b = np.concatenate([np.linspace(-120, 119.9, 40), np.full(40, 3.0)]).astype(np.float32)
    c.b[20] = 0
    c.Z = np.broadcast_to(c.b, (66, 80)).astype(np.float32).copy()
    c.W = np.random.default_rng(0).standard_normal(c.W.shape).astype(np.float32)
    c.check()


def test_ffn_rows_that_are_not_finite_stay_alone(gpu):
    for N, D, F in ((30, 40, 50), (300, 40, 50), (1100, 260, 1300)):
        c = Ffn(N, D, F, "silu", True)
        plain = c.forward()
        c.X[7, 3], c.X[20, :] = np.nan, np.inf
        got = c.forward()
        others = np.setdiff1d(np.arange(N), [7, 20])
        for name in ("H", "Z"):
            np.testing.assert_array_equal(got[name][others], plain[name][others])
            assert not np.isfinite(got[name][[7, 20]]).any()


@pytest.mark.parametrize("last", [777, 2])
def test_ffn_in_pieces(gpu, last):
    """More values of dZ than one piece holds: a million rows of 40 hidden features go
    through in two, each with scales of its own; checked against calls on the parts."""
    D, F, act = 2, 40, "silu"
    piece = (1 << 27) // 128 // 256 * 256  # 40 features are packed as 64
    N = piece + last
    g = torch.Generator(device="cuda").manual_seed(5)
    new = lambda n: torch.randn(n, generator=g, device="cuda")  # noqa: E731
    X, W, Z, dH = new(N * D), new(D * 2 * F), new(N * 2 * F), new(N * F)
    dX, dW, db = torch.empty(N * D, device="cuda"), torch.empty(D * 2 * F, device="cuda"), torch.empty(2 * F, device="cuda")
    ops.gated_ffn_backward(X, W, Z, dH, dX, dW, db, N, D, F, act=act)
    cut = lambda t, cols, a, b: t.view(cols, N)[:, a:b].contiguous().view(-1)  # noqa: E731
    sW, sb, parts = torch.zeros_like(dW), torch.zeros_like(db), []
    for a, b in ((0, piece), (piece, N)):
        parts.append(torch.empty((b - a) * D, device="cuda"))
        ops.gated_ffn_backward(cut(X, D, a, b), W, cut(Z, 2 * F, a, b), cut(dH, F, a, b), parts[-1], sW, sb, b - a, D, F, act=act,
                               accumulate=True)
    assert torch.equal(parts[0], cut(dX, D, 0, piece))
    # the last rows' sums may be split otherwise in a call of their own: both are off by their bound
    x, z, dh = (host(cut(t, k, piece, N)).reshape(k, last).T for t, k in ((X, D), (Z, 2 * F), (dH, F)))
    want = ref.ffn_backward(x, host(W).reshape(2 * F, D).T, z, dh, act)
    ref.check("dX", host(cut(dX, D, piece, N)).reshape(D, last).T, *want["dX"])
    for one, other, bound in ((sW, dW, want["dW"][1].T), (sb, db, want["db"][1])):
        one, other = host(one).astype(np.float64), host(other).astype(np.float64)
        assert (np.abs(one - other) <= 2 * bound.ravel() + 2 * U * np.abs(other)).all()


# ------------------------------------------------------------- differences
def test_gradients_against_differences(gpu):
    """Central differences of the GPU's forward along a direction.  Their distance from the
    gradient is at most the distance of the 64-bit differences from the 64-bit gradient
    (third derivatives) and both sides' errors: the bounds of the outputs, over the step."""
    h = np.float32(1.0 / 64)

    def compare(grad, egrad, fwd, want, arrays, k, direction):
        """fwd and want: arrays -> sum of outputs with fixed weights (want: value, bound)."""
        sides, exact, err = [], [], 0.0
        for s in (h, -h):
            moved = list(arrays)
            moved[k] = (arrays[k] + s * direction).astype(np.float32)
            sides.append(fwd(*moved))
            v, e = want(*moved)
            exact.append(v)
            err += e
        step = 2 * float(h)
        g64 = (egrad[0] * direction).sum()
        slack = abs((exact[0] - exact[1]) / step - g64) + err / step + (egrad[1] * np.abs(direction)).sum()
        assert abs((sides[0] - sides[1]) / step - (grad.astype(np.float64) * direction).sum()) <= slack

    rng = np.random.default_rng(8)
    unit = lambda *s: rng.choice([-1.0, 1.0], s).astype(np.float32)  # noqa: E731  (a step of h is exact beside values near 1)

    r = Recurrence(2, 70, 3, SAMPLE, False, True, None)
    got, want = r.run(), r.want()

    def rec_gpu(x, f):
        r.x, r.f = x, f
        o = r.run(("forward",))
        return (o["h"].astype(np.float64) * r.dh).sum() + (o["last"].astype(np.float64) * r.dl).sum()

    def rec_64(x, f):
        o = ref.recurrence(x, f, None, r.h0)
        return ((o["h"][0] * r.dh).sum() + (o["last"][0] * r.dl).sum(),
                (o["h"][1] * np.abs(r.dh)).sum() + (o["last"][1] * np.abs(r.dl)).sum())
    arrays = [r.x, r.f]
    for k, name in enumerate(("dx", "df")):
        compare(got[name], want[name], rec_gpu, rec_64, arrays, k, unit(*r.x.shape))

    c = Ffn(70, 20, 24, "silu", True)
    fw = ref.ffn_forward(c.X, c.W, c.b, "silu")
    c.Z = fw["Z"][0].astype(np.float32)
    got, want = c.backward(), ref.ffn_backward(c.X, c.W, c.Z, c.dH, "silu")

    def ffn_gpu(X, W):
        c.X, c.W = X, W
        return (c.forward()["H"].astype(np.float64) * c.dH).sum()

    def ffn_64(X, W):
        o = ref.ffn_forward(X, W, c.b, "silu")["H"]
        return (o[0] * c.dH).sum(), (o[1] * np.abs(c.dH)).sum()
    arrays = [c.X, c.W]
    for k, name in enumerate(("dX", "dW")):
        compare(got[name], want[name], ffn_gpu, ffn_64, arrays, k, unit(*arrays[k].shape))

    m = Norm(9, 30, 0.0, False, True)
    got, want = m.run(), ref.rms_norm(m.x, m.gamma, 1e-5, m.dy, m.dsum)

    def norm_gpu(x, gamma):
        m.x, m.gamma = x, gamma
        o = m.run()
        return (o["y"].astype(np.float64) * m.dy).sum() + (o["sum"].astype(np.float64) * m.dsum).sum()

    def norm_64(x, gamma):
        o = ref.rms_norm(x, gamma, 1e-5)["y"]
        return (o[0] * m.dy).sum() + (x.astype(np.float64) * m.dsum).sum(), (o[1] * np.abs(m.dy)).sum()
    arrays = [m.x, m.gamma]
    compare(got["ds"], want["ds"], norm_gpu, norm_64, arrays, 0, unit(9, 30))
    compare(got["dgamma"], want["dgamma"], norm_gpu, norm_64, arrays, 1, unit(30))
