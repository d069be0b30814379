"""The operators of a recurrent block together, as a training step and as generation
use them: eager, captured and replayed, over two streams; and at sizes whose positions
pass 32 bits."""
import numpy as np
import pytest
import torch

import block_ops_ref as ref
from cppnet_amd import ops
from test_gpu_lm_ops import REF, SAMPLE

pytestmark = pytest.mark.gpu


def f32(t):
    return t.to(device="cuda", dtype=torch.float32).contiguous()


class Block:
    """A language model of one block over the framework's operators:
      r0 = embedding;  n1 = norm(r0);  [x f] = n1 Wxf;  h = recurrence(x, f)
      r1, n2 = norm of r0 + dropout(h Wo);  u = gated_ffn(n2);  r2, n3 = norm of r1 + dropout(u Wd)
      loss = cross-entropy of n3 E^T with the embedding's own table.
    Rows by sample.  step() leaves the loss and every gradient in self.out."""
    P = 0.25
    SEED = 77

    def __init__(self, B=3, S=37, V=150, D=48, F=80, seed=0):
        self.dims = (B, S, V, D, F)
        g = torch.Generator().manual_seed(seed)
        r = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
        # storage of a ColMajor [in, out] weight is (out, in)
        self.w64 = {"E": r(V, D) / D ** 0.5, "Wxf": r(2 * D, D) / D ** 0.5, "Wo": r(D, D) / D ** 0.5,
                    "Wg": r(2 * F, D) / D ** 0.5, "bg": 0.2 * r(2 * F), "Wd": r(D, F) / F ** 0.5,
                    "g1": 1 + 0.2 * r(D), "g2": 1 + 0.2 * r(D), "g3": 1 + 0.2 * r(D)}
        self.w64 = {k: v.float().double() for k, v in self.w64.items()}
        self.w = {k: f32(v) for k, v in self.w64.items()}
        self.ids = torch.randint(0, V, (S, B), generator=g, dtype=torch.int32).cuda().view(-1)       # ColMajor [B, S]
        self.targets = torch.randint(-1, V, (B * S,), generator=g, dtype=torch.int32).cuda()          # rows by sample
        self.counter = torch.zeros(1, dtype=torch.int64, device="cuda")
        N = B * S
        e = lambda *s: torch.empty(s, device="cuda")  # noqa: E731
        self.t = {k: e(n * N) for k, n in {"r0": D, "n1": D, "x": 2 * D, "h": D, "o": D, "r1": D, "n2": D, "H": F, "Z": 2 * F,
                                           "d": D, "r2": D, "n3": D}.items()}
        self.t |= {k: e(N) for k in ("s1", "s2", "s3", "lse")}
        self.g = {k: torch.empty_like(v) for k, v in self.w.items()}
        self.d = {k: e(n * N) for k, n in {"n3": D, "r2": D, "d": D, "H": F, "n2": D, "r1": D, "o": D, "h": D, "xf": 2 * D,
                                           "n1": D, "r0": D}.items()}
        self.loss = e(1)
        self.out = [self.loss] + [self.g[k] for k in sorted(self.g)]

    def step(self):
        B, S, V, D, F = self.dims
        N, t, w, g, d = B * S, self.t, self.w, self.g, self.d
        n = N * D
        drop = lambda k: {"p": self.P, "seed": self.SEED, "offset": k * n, "counter": self.counter}  # noqa: E731
        ops.token_embedding_forward(self.ids, w["E"], t["r0"], B, S, V, D, rows=SAMPLE)
        ops.rms_norm_forward(t["r0"], None, w["g1"], t["n1"], None, t["s1"], N, D)
        ops.linear_forward(t["n1"], w["Wxf"], None, t["x"], N, D, 2 * D)
        x, f = t["x"][:n], t["x"][n:]
        ops.linear_recurrence_forward(x, f, None, None, t["h"], None, B, S, D, rows=SAMPLE)
        ops.linear_forward(t["h"], w["Wo"], None, t["o"], N, D, D)
        ops.rms_norm_forward(t["o"], t["r0"], w["g2"], t["n2"], t["r1"], t["s2"], N, D, **drop(0))
        ops.gated_ffn_forward(t["n2"], w["Wg"], w["bg"], t["H"], t["Z"], N, D, F)
        ops.linear_forward(t["H"], w["Wd"], None, t["d"], N, F, D)
        ops.rms_norm_forward(t["d"], t["r1"], w["g3"], t["n3"], t["r2"], t["s3"], N, D, **drop(1))
        ops.linear_ce_head(t["n3"], w["E"], None, self.targets, self.loss, t["lse"], d["n3"], g["E"], None, N, D, V)
        ops.rms_norm_backward(t["r2"], t["s3"], w["g3"], d["n3"], None, d["d"], d["r2"], g["g3"], N, D, **drop(1))
        ops.linear_backward(t["H"], w["Wd"], d["d"], g["Wd"], None, d["H"], N, F, D, accumulate=False)
        ops.gated_ffn_backward(t["n2"], w["Wg"], t["Z"], d["H"], d["n2"], g["Wg"], g["bg"], N, D, F)
        ops.rms_norm_backward(t["r1"], t["s2"], w["g2"], d["n2"], d["r2"], d["o"], d["r1"], g["g2"], N, D, **drop(0))
        ops.linear_backward(t["h"], w["Wo"], d["o"], g["Wo"], None, d["h"], N, D, D, accumulate=False)
        ops.linear_recurrence_backward(x, f, None, None, t["h"], d["h"], None, d["xf"][:n], d["xf"][n:], None, None, B, S, D,
                                       rows=SAMPLE)
        ops.linear_backward(t["n1"], w["Wxf"], d["xf"], g["Wxf"], None, d["n1"], N, D, 2 * D, accumulate=False)
        ops.rms_norm_backward(t["r0"], t["s1"], w["g1"], d["n1"], d["r1"], d["r0"], None, g["g1"], N, D)
        ops.token_embedding_backward(self.ids, d["r0"], g["E"], B, S, V, D, accumulate=True, rows=SAMPLE)
        ops.dropout_advance(self.counter, 2 * n)

    def reference(self, position):
        """The same by autograd in 64 bits."""
        B, S, V, D, F = self.dims
        N, n = B * S, B * S * D
        w = {k: v.clone().requires_grad_(True) for k, v in self.w64.items()}
        scale = 1.0 / (1.0 - self.P)

        def drop(x, k):  # positions run along the rows first
            keep = ref.kept(n, self.P, self.SEED, position + k * n).reshape(D, N).T
            return x * torch.tensor(keep * scale)

        def norm(x, gamma):
            return gamma * x * torch.rsqrt(x.square().mean(1, keepdim=True) + float(np.float32(1e-5)))
        ids = self.ids.cpu().view(S, B).T.reshape(-1).long()
        r0 = w["E"][ids]
        xf = norm(r0, w["g1"]) @ w["Wxf"].T
        a = torch.sigmoid(xf[:, D:]).view(B, S, D)
        x = xf[:, :D].view(B, S, D)
        state, out = torch.zeros(B, D, dtype=torch.float64), []
        for s in range(S):
            state = a[:, s] * state + (1 - a[:, s]) * x[:, s]
            out.append(state)
        r1 = r0 + drop(torch.stack(out, 1).reshape(N, D) @ w["Wo"].T, 0)
        z = norm(r1, w["g2"]) @ w["Wg"].T + w["bg"]
        u = torch.nn.functional.silu(z[:, :F]) * z[:, F:]
        r2 = r1 + drop(u @ w["Wd"].T, 1)
        logits = norm(r2, w["g3"]) @ w["E"].T
        held = self.targets.cpu() >= 0
        loss = torch.nn.functional.cross_entropy(logits[held], self.targets.cpu()[held].long())
        grads = torch.autograd.grad(loss, [w[k] for k in sorted(w)])
        return [loss.detach().reshape(1)] + list(grads)


def close(got, want):
    """A whole step's outputs within 2e-5 of the 64-bit ones (norm over norm): about twenty operators in a
    row, each off by some 2^-22 of its largest sums (1e-6 at most in the tests of each)."""
    for a, b in zip(got, want):
        a, b = a.double().cpu().view(-1), b.double().view(-1)
        assert torch.isfinite(a).all()
        assert (a - b).norm() <= 2e-5 * b.norm(), float((a - b).norm() / b.norm())


@pytest.mark.parametrize("size", [{}, {"B": 2, "S": 300, "V": 500, "D": 96, "F": 200}, {"B": 1, "S": 5, "V": 40, "D": 16, "F": 24}])
def test_training_step(gpu, size):
    b = Block(**size)
    position = 0
    for _ in range(2):  # the second step draws other masks
        b.step()
        torch.cuda.synchronize()
        close(b.out, b.reference(position))
        position = int(b.counter)
    n = 2 * b.dims[0] * b.dims[1] * b.dims[3]
    assert position == 2 * n


def test_training_step_captured(gpu):
    """Every replay of a captured step draws new masks from the counter, as the eager
    steps do, and gives their bits, with eager work of other sizes on the stream between."""
    b, eager, other = Block(), Block(), Block(B=2, S=90, V=300, D=64, F=100, seed=3)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        b.step()
        other.step()
    torch.cuda.synchronize()
    eager.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        b.step()
    seen = []
    for turn in range(4):
        for t in b.out:
            t.fill_(float("nan"))
        with torch.cuda.stream(stream):
            graph.replay()
            other.step()
        eager.step()
        torch.cuda.synchronize()
        for x, y in zip(b.out, eager.out):
            assert torch.equal(x, y)
        assert int(b.counter) == int(eager.counter)
        seen.append(b.out[1].clone())
    assert not torch.equal(seen[0], seen[1])
    close(b.out, b.reference(int(b.counter) - 2 * b.dims[0] * b.dims[1] * b.dims[3]))


def test_two_streams_at_once(gpu):
    """Two steps under way on streams of their own, with workspaces of their own."""
    blocks = [Block(B=4, S=200, V=400, D=128, F=256, seed=i) for i in range(2)]
    alone = []
    for b in blocks:
        b.step()
        torch.cuda.synchronize()
        alone.append([t.clone() for t in b.out])
        b.counter.zero_()
    streams = [torch.cuda.Stream() for _ in blocks]
    torch.cuda.synchronize()
    for _ in range(3):
        for b, s in zip(blocks, streams):
            with torch.cuda.stream(s):
                b.step()
                b.counter.zero_()
    torch.cuda.synchronize()
    for b, want in zip(blocks, alone):
        for x, y in zip(b.out, want):
            assert torch.equal(x, y)


def test_generation_is_the_training_forward(gpu):
    """Token by token with a carried state, as a whole prompt gives it (no dropout)."""
    B, S, D, F = 3, 12, 40, 56
    rng = np.random.default_rng(4)
    new = lambda *s: torch.from_numpy(rng.standard_normal(s).astype(np.float32)).cuda()  # noqa: E731
    x, f, gamma, W = new(D, B, S), new(D, B, S), new(D), new(2 * F, D) / D ** 0.5
    h, last = torch.empty(D * B * S, device="cuda"), torch.empty(D * B, device="cuda")
    ops.linear_recurrence_forward(x.view(-1), f.view(-1), None, None, h, last, B, S, D, rows=SAMPLE)
    y, H = torch.empty_like(h), torch.empty(F * B * S, device="cuda")
    ops.rms_norm_forward(h, x.view(-1), gamma, y, None, None, B * S, D)
    ops.gated_ffn_forward(y, W.view(-1), None, H, None, B * S, D, F)
    state = torch.zeros(D * B, device="cuda")
    for t in range(S):
        xt, ft = x[:, :, t].contiguous().view(-1), f[:, :, t].contiguous().view(-1)
        ht, yt, Ht = torch.empty(D * B, device="cuda"), torch.empty(D * B, device="cuda"), torch.empty(F * B, device="cuda")
        ops.linear_recurrence_forward(xt, ft, None, state, ht, state, B, 1, D)
        ops.rms_norm_forward(ht, xt, gamma, yt, None, None, B, D)
        ops.gated_ffn_forward(yt, W.view(-1), None, Ht, None, B, D, F)
        for a, whole, n in ((ht, h, D), (yt, y, D), (Ht, H, F)):
            want = whole.view(n, B, S)[:, :, t].reshape(-1)
            assert (a - want).norm() <= 1e-5 * want.norm()
    assert (state - last).norm() <= 1e-6 * last.norm()


def test_positions_past_32_bits(gpu):
    """2^31 + 2^21 values: a row of the last column, the last steps, the last elements."""
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("needs 80 GiB of free device memory")
    n = (1 << 31) + (1 << 21)
    x = torch.empty(n, device="cuda")
    for i in range(0, n, 1 << 28):
        x[i:i + (1 << 28)] = 1.0
    y = torch.empty(n, device="cuda")
    tail = 5000
    ops.dropout_seeded(x, y, 0.5, 5)
    keep = ref.kept(tail, 0.5, 5, n - tail)
    np.testing.assert_array_equal(y[-tail:].cpu().numpy(), np.where(keep, np.float32(2), np.float32(0)))
    # norm: columns of 2^21 + 2^11 rows
    F = 1024
    N = n // F
    gamma, rstd = torch.full((F,), 3.0, device="cuda"), torch.empty(N, device="cuda")
    x[-tail:] = 2.0  # the last rows' last feature
    ops.rms_norm_forward(x, None, gamma, y, None, rstd, N, F)
    want = 1 / np.sqrt((F - 1 + 4) / F + float(np.float32(1e-5)))
    got = y[-tail:].cpu().numpy()
    np.testing.assert_allclose(got, 6 * want, rtol=1e-6)
    np.testing.assert_allclose(rstd[-tail:].cpu().numpy(), want, rtol=1e-6)
    assert abs(float(y[0]) - 3 / np.sqrt(1 + 1e-5)) < 1e-5
    # recurrence: four chains of 2^29 + 2^19 steps with a gate of one half
    S = n // 4
    for i in range(0, n, 1 << 28):
        x[i:i + (1 << 28)] = 0.0
    h, last = y, torch.empty(4, device="cuda")
    one = torch.zeros(n, device="cuda")  # sigmoid(0) = 1 / 2
    x[S - 3], x[n - 2], x[n - 1] = 8.0, 4.0, 16.0
    ops.linear_recurrence_forward(x, one, None, None, h, last, 2, S, 2, rows=SAMPLE)
    np.testing.assert_array_equal(last.cpu().numpy(), [1.0, 0.0, 0.0, 9.0])
    np.testing.assert_array_equal(h[S - 4:S].cpu().numpy(), [0.0, 4.0, 2.0, 1.0])
    np.testing.assert_array_equal(h[-3:].cpu().numpy(), [0.0, 2.0, 9.0])


def test_more_chains_than_a_launch_takes(gpu):
    """2^29 + 2^16 chains of one step: a second launch has the last of them."""
    B, D = 1 << 16, (1 << 13) + 1
    n = B * D
    x, f, h = (torch.empty(n, device="cuda") for _ in range(3))
    f.zero_()  # a = 1 / 2
    h.fill_(-1.0)
    last = torch.full((n,), 6.0, device="cuda")
    for i in range(0, n, 1 << 24):
        k = min(1 << 24, n - i)
        x[i:i + k] = torch.arange(i % 1021, i % 1021 + k, device="cuda", dtype=torch.int32) % 1021
    ops.linear_recurrence_forward(x, f, None, last, h, last, B, 1, D)
    x.add_(6.0).mul_(0.5)
    assert torch.equal(h, x)
    assert torch.equal(last, x)
