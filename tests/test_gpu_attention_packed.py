"""GPU tests of the attention's forward on packed operands, which takes over
from 64 queries and 8192 query rows over all samples and heads on: values of out
and lse, and the gradients that follow from them, against the 64-bit form and
the bounds of lm_ops_ref.py.  Then, in every path, operands at the ends of the
range: scores far from zero, values that are not finite, operands whose sizes
multiply past it, queries that read nothing."""
import numpy as np
import pytest

import lm_ops_ref as ref
from test_gpu_lm_ops import REF, SAMPLE, Buffers, att_run, per_head
from test_gpu_lm_ops_edges import att_check, wide

pytestmark = pytest.mark.gpu


def packed(B, Sq, H):
    return Sq >= 64 and B * H * Sq >= 8192


PACKED = [  # B, Sq, Sk, H, KH, dh, causal, k_len, q_start, rows, scale
    (8, 128, 128, 8, 8, 64, True, None, None, SAMPLE, None),
    (8, 130, 140, 8, 4, 32, True, None, None, SAMPLE, None),
    (7, 147, 147, 8, 8, 96, True, None, None, REF, None),
    (9, 129, 129, 8, 2, 128, False, None, None, SAMPLE, None),
    (33, 64, 64, 4, 4, 128, True, None, None, REF, None),
    (4, 260, 33, 8, 8, 40, False, None, None, SAMPLE, None),         # keys of one tile and one more
    (4, 260, 31, 8, 1, 64, True, None, None, SAMPLE, None),          # 229 queries read nothing
    (3, 700, 1, 4, 4, 17, False, None, None, REF, None),             # one key
    (2, 1100, 257, 4, 2, 100, True, None, [0, 100], SAMPLE, None),
    (6, 200, 300, 8, 4, 64, False, [300, 0, 1, 31, 32, 33], None, SAMPLE, None),
    (6, 200, 300, 8, 2, 33, True, [300, 0, 3, 64, 299, 129], None, REF, None),
    (6, 200, 300, 8, 8, 128, True, [300, 300, 70, 0, 5, 400], [100, -150, 60, 7, 299, -300], SAMPLE, None),
    (5, 300, 200, 6, 3, 80, False, [200, 199, 128, 97, 65], None, REF, None),
    (8, 150, 150, 8, 8, 64, True, None, None, SAMPLE, -0.3),
    (8, 150, 150, 8, 4, 48, False, None, None, REF, -1.5),
    (8, 150, 150, 8, 8, 1, True, None, None, SAMPLE, 0.0),
    (8, 150, 150, 8, 8, 32, True, None, None, SAMPLE, 2.0 ** -60),
    (1, 1200, 1300, 7, 1, 128, True, None, None, SAMPLE, None),      # seven heads on one, rows past a tile
    (1, 2049, 65, 4, 4, 66, True, None, [-1], REF, None),
]
BORDER = [  # B, Sq, H: just below the rule and just on it
    (64, 64, 2), (65, 63, 2), (43, 95, 2), (64, 127, 1), (64, 128, 1), (1, 8191, 1), (1, 8192, 1),
]


def test_the_cases_run_packed():
    assert all(packed(c[0], c[1], c[3]) for c in PACKED)
    assert [packed(*c) for c in BORDER] == [True, False, False, False, True, False, True]


def data(rng, B, Sq, Sk, H, KH, dh, causal, k_len, q_start):
    """Operands with NaN and infinities at every key that no query of its sample reads."""
    f = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
    q, k, v, do = f(B, Sq, H * dh), f(B, Sk, KH * dh), f(B, Sk, KH * dh), f(B, Sq, H * dh)
    unread = ~ref.allowed(B, Sq, Sk, causal, k_len, q_start).any(1)
    k[unread], v[unread] = np.nan, np.inf
    return q, k, v, do


@pytest.mark.parametrize("B,Sq,Sk,H,KH,dh,causal,k_len,q_start,rows,scale", PACKED)
def test_values(gpu, B, Sq, Sk, H, KH, dh, causal, k_len, q_start, rows, scale):
    print(f"[attention] B={B} {Sq}x{Sk} heads {H}/{KH} dh={dh} causal={causal} {k_len} {q_start} rows={rows} {scale}", flush=True)
    rng = np.random.default_rng(Sq + 7 * Sk + dh)
    x = data(rng, B, Sq, Sk, H, KH, dh, causal, k_len, q_start)
    att_check((B, Sq, Sk, H, KH, dh), causal, k_len, q_start, rows, scale, *x)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,Sq,H", BORDER)
def test_values_on_both_sides_of_the_rule(gpu, B, Sq, H, causal):
    print(f"[attention] B={B} {Sq}x50 heads {H} causal={causal}", flush=True)
    rng = np.random.default_rng(Sq)
    x = data(rng, B, Sq, 50, H, 1, 32, causal, None, [50 - Sq] * B if causal else None)
    att_check((B, Sq, 50, H, 1, 32), causal, None, None, SAMPLE, None, *x)


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,S,H,KH,dh", [(16, 160, 4, 2, 64), (11, 200, 4, 4, 128), (30, 70, 4, 1, 32)])
def test_blocks_of_very_different_size(gpu, B, S, H, KH, dh, causal):
    """The sums' scale follows the largest block of values so far."""
    print(f"[attention] blocks {B}x{S} heads {H}/{KH} dh={dh} causal={causal}", flush=True)
    rng = np.random.default_rng(S + dh)
    size = lambda *e: np.array(e)[np.arange(S) // 32 % len(e)].astype(np.float32)[None, :, None]  # noqa: E731
    f = lambda h: rng.standard_normal((B, S, h * dh)).astype(np.float32)  # noqa: E731
    q = f(H) * size(1.0, 2.0 ** -30, 4.0, 0.0, 2.0 ** -70)
    k = f(KH) * size(2.0 ** -20, 1.0, 0.0, 2.0)
    v = f(KH) * size(2.0 ** 40, 2.0 ** -40, 1.0, 0.0, 2.0 ** 20)
    do = f(H) * size(2.0 ** -50, 1.0, 2.0 ** 30, 0.0)
    assert packed(B, S, H)
    att_check((B, S, S, H, KH, dh), causal, None, None, SAMPLE, None, q, k, v, do)
    v = f(KH) * size(2.0 ** -40, 2.0 ** 20, 2.0 ** -45, 1.0, 2.0 ** 40)  # growing, and far below what came before
    att_check((B, S, S, H, KH, dh), causal, None, None, REF, None, q, k, v, do)


def sharp(rng, B, Sq, Sk, H, KH, dh, level):
    """Operands whose scores lie around `level` and vary by some 1e7: 64 exact
    units in feature 0 carry the level, the other features the variation."""
    q, k = (rng.standard_normal((B, s, h * dh)).astype(np.float32) * np.float32(2e3) for s, h in ((Sq, H), (Sk, KH)))
    q[:, :, ::dh], k[:, :, ::dh] = np.float32(8192), np.float32(level / 8192)
    return q, k


@pytest.mark.parametrize("level", [0.0, 7e7, -7e7, 1e9, -1e9])
@pytest.mark.parametrize("B,Sq,Sk,H,KH,dh,causal", [(2, 1, 300, 4, 2, 32, False), (2, 20, 300, 4, 2, 64, True),
                                                    (8, 130, 200, 8, 4, 64, True), (9, 128, 100, 8, 8, 128, False)])
def test_scores_far_from_zero(gpu, B, Sq, Sk, H, KH, dh, causal, level):
    """Where a query's largest score leads by more than the scores' errors, out
    is that key's value; no finite score gives anything that is not finite.  A
    probability of another key is below e^-40."""
    print(f"[attention] B={B} {Sq}x{Sk} heads {H}/{KH} dh={dh} causal={causal} level {level}", flush=True)
    rng = np.random.default_rng(Sk + dh)
    q, k = sharp(rng, B, Sq, Sk, H, KH, dh, level)
    v = rng.standard_normal((B, Sk, KH * dh)).astype(np.float32)
    got = att_run(Buffers(), (q, k, v), dict(causal=causal, k_len=None, q_start=None, rows=SAMPLE), (B, Sq, Sk, H, KH, dh), None, 1.0)
    assert np.isfinite(got["out"]).all() and np.isfinite(got["lse"]).all()
    wq, wk, wv = wide(q, H), np.repeat(wide(k, KH), H // KH, 1), np.repeat(wide(v, KH), H // KH, 1)
    ok = ref.allowed(B, Sq, Sk, causal, None, None)[:, None]
    s = np.where(ok, wq @ wk.transpose(0, 1, 3, 2), -np.inf)
    es = ref.g(dh) * np.where(ok, np.abs(wq) @ np.abs(wk).transpose(0, 1, 3, 2), 0).max(3)
    es += 2 * dh * ref.F * np.abs(wq).max() * np.abs(wk).max() + 12 * ref.U * np.abs(s.max(3))
    best = s.argmax(3)
    others = np.where(np.arange(Sk) == best[..., None], -np.inf, s).max(3)
    leads = s.max(3) - others > 2 * es + 40
    assert leads.mean() > 0.5, leads.mean()
    want = np.take_along_axis(wv, best[..., None], 2)
    lim = (ref.g(Sk) + Sk * np.exp(-40.0)) * np.abs(wv).max()
    off = np.abs(per_head(got["out"], H) - want).max(3)[leads]
    assert off.max() <= lim, (off.max(), lim)
    off = np.abs(got["lse"].transpose(0, 2, 1) - s.max(3))
    assert (off <= es + 4 * ref.U * np.abs(s.max(3)) + np.log(Sk)).all()


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("level", [0.0, 7e7, -1e9])
@pytest.mark.parametrize("Sq,Sk,H,KH,dh,causal", [(1, 1, 2, 2, 32, False), (40, 70, 4, 2, 64, True), (200, 150, 2, 1, 128, False), (70, 70, 3, 3, 96, True)])
def test_gradients_of_scores_far_from_zero(gpu, Sq, Sk, H, KH, dh, causal, level, rows):
    """The probabilities formed again from lse are off by 2^-22 |lse| of
    themselves and the like of the scores' own errors, which at scores of 1e7 and
    more says little about them; but each is held to 1, so dv of a key is at most
    the sum of |dout| over the queries that read it, and the other gradients are
    finite.  Level 0: scores of moderate size whose terms cancel."""
    print(f"[attention] {Sq}x{Sk} heads {H}/{KH} dh={dh} causal={causal} level {level} rows={rows}", flush=True)
    rng = np.random.default_rng(Sk + dh)
    B = 2
    q, k = sharp(rng, B, Sq, Sk, H, KH, dh, level)
    if level == 0.0:
        half = dh // 2
        for x, h, sign in ((q, H, 1), (k, KH, -1)):
            y = x.reshape(B, -1, h, dh)
            y[..., half:] = sign * y[..., :half]
    v, do = (rng.standard_normal((B, s, h * dh)).astype(np.float32) for s, h in ((Sk, KH), (Sq, H)))
    got = att_run(Buffers(), (q, k, v), dict(causal=causal, k_len=None, q_start=None, rows=rows), (B, Sq, Sk, H, KH, dh), do, 1.0)
    for name, x in got.items():
        assert np.isfinite(x).all(), name
    ok = ref.allowed(B, Sq, Sk, causal, None, None)[:, None]
    most = (ok.transpose(0, 1, 3, 2) @ np.abs(wide(do, H))).reshape(B, KH, H // KH, Sk, dh).sum(2)
    dv = np.abs(per_head(got["dv"], KH).astype(np.float64))
    assert (dv <= most * (1 + ref.g(Sq * H)) + 4 * Sq * ref.F * np.abs(do).max()).all(), (dv - most).max()


@pytest.mark.parametrize("what", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("B,Sq,Sk,H,KH,dh", [(2, 1, 100, 2, 2, 32), (2, 20, 100, 2, 1, 64), (8, 130, 100, 8, 4, 64), (16, 128, 70, 4, 4, 32)])
def test_values_that_are_not_finite_among_small_ones(gpu, B, Sq, Sk, H, KH, dh, what):
    """A block of values that are zeros but for one that is not finite: its
    feature of out is not finite either, however small the block's others are
    beside those of the blocks before; other features are as without it."""
    print(f"[attention] B={B} {Sq}x{Sk} heads {H}/{KH} dh={dh} {what}", flush=True)
    rng = np.random.default_rng(Sk + dh)
    f = lambda s, h: rng.standard_normal((B, s, h * dh)).astype(np.float32)  # noqa: E731
    q, k, v = f(Sq, H), f(Sk, KH), f(Sk, KH)
    v[:, 32:64] = 0
    v[:, 40, 3] = what  # feature 3 of the first key head
    dims, kw = (B, Sq, Sk, H, KH, dh), dict(causal=False, k_len=None, q_start=None, rows=SAMPLE)
    got = att_run(Buffers(), (q, k, v), kw, dims)
    out = per_head(got["out"], H)
    readers = slice(0, H // KH)
    assert not np.isfinite(out[:, readers, :, 3]).any()
    v[:, 40, 3] = 0
    want = ref.attention(wide(q, H), wide(k, KH), wide(v, KH), ref.allowed(B, Sq, Sk, False, None, None), dh ** -0.5)
    hit = np.zeros(out.shape, bool)
    hit[:, readers, :, 3] = True
    ref.check("out", np.where(hit, 0, out), np.where(hit, 0, want["out"][0]), want["out"][1])
    ref.check("lse", got["lse"].transpose(0, 2, 1), *want["lse"])
    v[:, 32:64] = what  # and a block of nothing else
    assert not np.isfinite(att_run(Buffers(), (q, k, v), kw, dims)["out"]).any()


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("B,Sq,Sk,H,KH,dh", [(2, 1, 100, 2, 2, 32), (2, 20, 100, 2, 1, 64), (2, 70, 90, 2, 1, 64), (8, 130, 100, 8, 4, 64)])
def test_large_operands_that_do_not_meet(gpu, B, Sq, Sk, H, KH, dh, causal):
    """Queries of 2^80 in one feature and keys of 2^80 in another: every score is
    an exact 0.  Values and gradients are those of the same operands at 1, dq and
    dk times 2^80."""
    print(f"[attention] B={B} {Sq}x{Sk} heads {H}/{KH} dh={dh} causal={causal}", flush=True)
    rng = np.random.default_rng(Sk + dh)
    q, k = np.zeros((B, Sq, H, dh), np.float32), np.zeros((B, Sk, KH, dh), np.float32)
    q[..., 1], k[..., 2] = 1, 1
    q, k = q.reshape(B, Sq, H * dh), k.reshape(B, Sk, KH * dh)
    v, do = (rng.standard_normal((B, s, h * dh)).astype(np.float32) for s, h in ((Sk, KH), (Sq, H)))
    big = np.float32(2.0 ** 80)
    dims, kw = (B, Sq, Sk, H, KH, dh), dict(causal=causal, k_len=None, q_start=None, rows=SAMPLE)
    got = att_run(Buffers(), (q * big, k * big, v), kw, dims, do)
    want = ref.attention(wide(q, H), wide(k, KH), wide(v, KH), ref.allowed(B, Sq, Sk, causal, None, None), dh ** -0.5, wide(do, H))
    for name, (w, lim) in want.items():
        x = got[name].transpose(0, 2, 1) if name == "lse" else per_head(got[name], KH if name in ("dk", "dv") else H)
        print("  ", name, ref.check(name, x * 2.0 ** -80 if name in ("dq", "dk") else x, w, lim))


@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("B,Sq,Sk,H,KH,dh", [(2, 3, 50, 2, 2, 32), (2, 40, 70, 2, 1, 64), (8, 130, 100, 8, 4, 64)])
def test_scale_of_minus_zero(gpu, B, Sq, Sk, H, KH, dh, rows):
    rng = np.random.default_rng(Sk)
    k_len, start = [Sk - 9] * B, [Sk - Sq - 9] * B
    x = data(rng, B, Sq, Sk, H, KH, dh, True, k_len, start)
    got = att_check((B, Sq, Sk, H, KH, dh), True, k_len, start, rows, -0.0, *x)
    assert (got["dq"] == 0).all() and (got["dk"] == 0).all()


@pytest.mark.parametrize("what", [np.nan, np.inf, 1e30])
@pytest.mark.parametrize("rows", [REF, SAMPLE])
@pytest.mark.parametrize("B,Sq,Sk,H,KH,dh", [(3, 4, 60, 2, 2, 32), (3, 40, 600, 2, 1, 64), (3, 70, 90, 2, 1, 64), (9, 130, 100, 8, 4, 64),
                                             (9, 257, 140, 4, 4, 128)])
def test_queries_that_read_nothing_may_hold_anything(gpu, B, Sq, Sk, H, KH, dh, rows, what):
    """The first queries of a sample that begins before its keys, and all of a
    sample without keys, give zero rows and reach no gradient."""
    print(f"[attention] B={B} {Sq}x{Sk} heads {H}/{KH} dh={dh} rows={rows} {what}", flush=True)
    rng = np.random.default_rng(Sk + dh)
    f = lambda s, h: rng.standard_normal((B, s, h * dh)).astype(np.float32)  # noqa: E731
    q, k, v, do = f(Sq, H), f(Sk, KH), f(Sk, KH), f(Sq, H)
    start = [(-(Sq // 2), 3, -1)[b % 3] for b in range(B)]
    k_len = [(Sk, 0, Sk - 5)[b % 3] for b in range(B)]
    ok = ref.allowed(B, Sq, Sk, True, k_len, start)
    reads = ok.any(2)[:, :, None]
    assert not reads.all() and reads.any()
    dims, kw = (B, Sq, Sk, H, KH, dh), dict(causal=True, k_len=k_len, q_start=start, rows=rows)
    buf = Buffers()
    got = att_run(buf, (np.where(reads, q, np.float32(what)), k, v), kw, dims, np.where(reads, do, np.float32(what)))
    read = ok.any(1)[:, :, None]
    want = ref.attention(wide(np.where(reads, q, 0), H), wide(np.where(read, k, 0), KH), wide(np.where(read, v, 0), KH), ok,
                         dh ** -0.5, wide(np.where(reads, do, 0), H))
    for name, (w, lim) in want.items():
        x = got[name].transpose(0, 2, 1) if name == "lse" else per_head(got[name], KH if name in ("dk", "dv") else H)
        print("  ", name, ref.check(name, x, w, lim))
    for name in ("out", "dq"):
        assert (got[name][~reads[:, :, 0]] == 0).all()
    buf.intact()
    # nor does a key or value that only the others read reach their rows
    k[:, 0], v[:, 0] = what, what
    got = att_run(Buffers(), (q, k, v), kw, dims, do)
    for name in ("out", "dq"):
        assert (got[name][~reads[:, :, 0]] == 0).all()
    assert (got["lse"][~reads[:, :, 0]] == -np.inf).all()
