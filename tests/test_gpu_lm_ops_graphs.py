"""GPU tests of the language-model operators in captured graphs: replays among
calls of other sizes and paths on the captured stream, and after calls that
needed more workspace than the graph's."""
import numpy as np
import pytest
import torch

from cppnet_amd import ops

pytestmark = pytest.mark.gpu


class Work:
    """Embedding, attention and cross-entropy, each with its gradients, over
    operands of one size; run() gives every output."""

    def __init__(self, seed, B, Sq, Sk, H, KH, dh, N, D, V):
        self.rng = np.random.default_rng(seed)
        f = lambda n: torch.from_numpy(self.rng.standard_normal(n).astype(np.float32)).cuda()  # noqa: E731
        i = lambda n, most: torch.from_numpy(self.rng.integers(-1, most, n).astype(np.int32)).cuda()  # noqa: E731
        nq, nk = B * Sq * H * dh, B * Sk * KH * dh
        self.dims, self.head, self.emb = (B, Sq, Sk, H, KH, dh), (N, D, V), (1, N, V, D)
        self.inputs = [f(n) for n in (nq, nk, nk, nq, N * D, V * D)]
        self.ids = i(N, V)
        self.sizes = (nq, B * Sq * H, nq, nk, nk, 1, N, N * D, V * D, N * D, V * D)

    def outputs(self):
        return [torch.full((n,), float("nan"), device="cuda") for n in self.sizes]

    def renew(self):
        for x in self.inputs:
            x.copy_(torch.from_numpy(self.rng.standard_normal(x.numel()).astype(np.float32)))

    def run(self, o):
        q, k, v, do, X, W = self.inputs
        ops.attention_forward(q, k, v, o[0], o[1], *self.dims, True)
        ops.attention_backward(q, k, v, o[0], o[1], do, *o[2:5], *self.dims, True)
        ops.linear_ce_head(X, W, None, self.ids, o[5], o[6], o[7], o[8], None, *self.head)
        ops.token_embedding_forward(self.ids, W, o[9], *self.emb)
        ops.token_embedding_backward(self.ids, X, o[10], *self.emb)


SMALL = dict(B=2, Sq=1, Sk=70, H=4, KH=2, dh=64, N=9, D=20, V=50)          # single tokens, few rows
MIDDLE = dict(B=2, Sq=40, Sk=300, H=2, KH=1, dh=96, N=100, D=48, V=900)    # keys split over blocks, packed rows
LARGE = dict(B=8, Sq=130, Sk=140, H=8, KH=8, dh=64, N=700, D=130, V=3000)  # everything packed


def capture(work, out, stream):
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        work.run(out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        work.run(out)
    return graph


def replay_and_compare(graph, work, got, want, stream):
    work.renew()
    for x in got:
        x.fill_(float("nan"))
    work.run(want)  # on the default stream, in its workspace
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("captured,others", [(MIDDLE, [SMALL]), (LARGE, [SMALL, MIDDLE])])
def test_replays_between_calls_of_other_sizes(gpu, captured, others):
    """On the captured stream, in the graph's own workspace."""
    work, stream = Work(1, **captured), torch.cuda.Stream()
    got, want = work.outputs(), work.outputs()
    graph = capture(work, got, stream)
    for turn in range(4):
        for i, size in enumerate(others):
            other = Work(10 * turn + i, **size)
            alone, among = other.outputs(), other.outputs()
            other.run(alone)
            torch.cuda.synchronize()
            with torch.cuda.stream(stream):
                other.run(among)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(alone, among))
        replay_and_compare(graph, work, got, want, stream)


def test_replays_after_calls_that_needed_more_workspace(gpu):
    """A graph keeps the workspace that it was captured with when a later call
    on its stream outgrows it, and so does one captured after that."""
    stream = torch.cuda.Stream()
    graphs = []
    for seed, size in enumerate((SMALL, MIDDLE, LARGE)):
        work = Work(seed, **size)
        got, want = work.outputs(), work.outputs()
        graphs.append((capture(work, got, stream), work, got, want))
        for _ in range(2):
            for g, w, a, b in graphs:
                replay_and_compare(g, w, a, b, stream)
    more = Work(9, **(LARGE | {"N": 3000, "V": 9000, "Sk": 600}))
    with torch.cuda.stream(stream):
        more.run(more.outputs())
    # others take what was given back, if anything was
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        more.run(more.outputs())
    torch.cuda.synchronize()
    for _ in range(3):
        for g, w, a, b in graphs:
            replay_and_compare(g, w, a, b, stream)
