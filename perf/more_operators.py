"""Performance cases of the operators of a recurrent language model's block: a
gated linear recurrence with its backward pass, a gated feed-forward layer (two
projections, an activation and their product) with its backward pass, a
root-mean-square norm over the sum of a residual and a dropped-out branch, and
dropout whose mask is never stored.

Everything is fp32 (the framework's only floating type).  Tensors follow the
framework's ColMajor layout: a [rows, cols] matrix is a torch tensor of shape
(cols, rows).  A sequence [B, S, D] is a [B*S, D] matrix whose rows are in the
reference order (row b + B*s) or by sample (row s + S*b).

`own` chooses what run() does: the framework's operators, or their plain form
in elementary torch operations.
"""
import math

import numpy as np
import torch

own = False

REF, BY_SAMPLE = 0, 1


# ------------------------------------------------------------------ helpers
def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 31)


def _randn(g, *shape):
    return torch.randn(shape, generator=g, device="cuda")


def _empty(*shape):
    return torch.empty(shape, device="cuda")


def _log(rng, lo, hi):
    """An integer spread over the logarithm of [lo, hi], odd ones among them."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _sigmoid(x):
    return 1.0 / (1.0 + torch.exp(-x))


# -------------------------------------------------- gated linear recurrence
#   a = sigmoid(f), w = sigmoid(i), or 1 - a where there is no i
#   h_t = a_t h_{t-1} + w_t x_t over the steps of each sample's length
def _rec_lengths(c):
    B, S = c["batch"], c["steps"]
    if not c["ragged"]:
        return [S] * B
    return [max(0, S - (b * 7919 + 13) % (S // 2 + 1)) for b in range(B)]


def _rec_prepare(c, g):
    B, S, D = c["batch"], c["steps"], c["dim"]
    n = B * S
    # gates of a trained model remember: a is 0.88 in the middle, 0.5 to 0.98 mostly
    s = {"x": _randn(g, D, n), "f": 2.0 + _randn(g, D, n), "i": _randn(g, D, n) if c["input_gate"] else None,
         "h0": _randn(g, D, B) if c["state"] else None, "h": _empty(D, n), "h_last": _empty(D, B)}
    s["len"] = torch.tensor(_rec_lengths(c), dtype=torch.int32, device="cuda") if c["ragged"] else None
    if c["train"]:
        s.update(dh=_randn(g, D, n), dh_last=_randn(g, D, B) if c["state"] else None, dx=_empty(D, n), df=_empty(D, n),
                 di=_empty(D, n) if c["input_gate"] else None, dh0=_empty(D, B) if c["state"] else None)
    return s


def _steps_last(c, t):
    """(D, B*S) storage -> [D, B, S]."""
    B, S, D = c["batch"], c["steps"], c["dim"]
    return t.view(D, S, B).transpose(1, 2) if c["rows"] == REF else t.view(D, B, S)


def _rec_stored(c, t):
    """[D, B, S] -> (D, B*S) storage."""
    return (t.transpose(1, 2) if c["rows"] == REF else t).reshape(c["dim"], -1)


def _scan(a, b):
    """y_t = a_t y_{t-1} + b_t along the last axis, y_{-1} = 0: every round
    joins runs twice as long."""
    k, n = 1, a.shape[-1]
    while k < n:
        b = torch.cat([b[..., :k], b[..., k:] + a[..., k:] * b[..., :-k]], -1)
        a = torch.cat([a[..., :k], a[..., k:] * a[..., :-k]], -1)
        k *= 2
    return b


def _from_state(a, b, y0):
    """b with the state before the first step entered."""
    return torch.cat([b[..., :1] + a[..., :1] * y0[..., None], b[..., 1:]], -1)


def _rec_plain(c, s):
    D, B, S = c["dim"], c["batch"], c["steps"]
    x, f = _steps_last(c, s["x"]), _steps_last(c, s["f"])
    i = _steps_last(c, s["i"]) if c["input_gate"] else None
    a, rest = _sigmoid(f), _sigmoid(-f)
    w = _sigmoid(i) if c["input_gate"] else rest
    h0 = s["h0"] if c["state"] else x.new_zeros(D, B)
    b = w * x
    if c["ragged"]:
        held = torch.arange(S, device=x.device)[None, :] < s["len"].long()[:, None]
        a, b = torch.where(held, a, torch.ones_like(a)), torch.where(held, b, torch.zeros_like(b))
    h = _scan(a, _from_state(a, b, h0))
    last = h[..., -1].contiguous()
    res = [_rec_stored(c, torch.where(held, h, torch.zeros_like(h)) if c["ragged"] else h), last]
    if not c["train"]:
        return res
    dh = _steps_last(c, s["dh"])
    dlast = s["dh_last"] if c["state"] else x.new_zeros(D, B)
    if c["ragged"]:
        dh = torch.where(held, dh, torch.zeros_like(dh))
    # u_t = a_t g_t is what the state before step t receives, g_t = dh_t + u_{t+1}
    ar = a.flip(-1)
    u = _scan(ar, _from_state(ar, ar * dh.flip(-1), dlast)).flip(-1)
    gr = dh + torch.cat([u[..., 1:], dlast[..., None]], -1)
    before = torch.cat([h0[..., None], h[..., :-1]], -1)
    dx = w * gr
    if c["input_gate"]:
        df, di = a * rest * gr * before, w * _sigmoid(-i) * gr * x
    else:
        df, di = a * rest * gr * (before - x), None
    grads = [dx, df] if di is None else [dx, df, di]
    if c["ragged"]:
        grads = [torch.where(held, t, torch.zeros_like(t)) for t in grads]
    res += [_rec_stored(c, t) for t in grads]
    return res + [u[..., 0].contiguous()] if c["state"] else res


def _rec_run(c, s):
    B, S, D = c["batch"], c["steps"], c["dim"]
    if own:
        from cppnet_amd import ops
        how = {"seq_len": s["len"], "rows": c["rows"]}
        ops.linear_recurrence_forward(s["x"], s["f"], s["i"], s["h0"], s["h"], s["h_last"], B, S, D, **how)
        if not c["train"]:
            return [s["h"], s["h_last"]]
        ops.linear_recurrence_backward(s["x"], s["f"], s["i"], s["h0"], s["h"], s["dh"], s["dh_last"], s["dx"], s["df"],
                                       s["di"], s["dh0"], B, S, D, **how)
        return [s[k] for k in ("h", "h_last", "dx", "df", "di", "dh0") if s[k] is not None]
    return _rec_plain(c, s)


def _rec_exact(c, s):
    """Step by step."""
    D, B, S = c["dim"], c["batch"], c["steps"]
    wide = {k: _steps_last(c, s[k]).double().permute(2, 0, 1).contiguous() for k in ("x", "f", "i", "dh")
            if s.get(k) is not None}
    f = wide["f"]
    a, x = torch.special.expit(f), wide["x"]
    w = torch.special.expit(wide["i"]) if c["input_gate"] else torch.special.expit(-f)
    n = torch.tensor(_rec_lengths(c), device=f.device)
    held = [n > t for t in range(S)] if c["ragged"] else None
    zero = f.new_zeros(D, B)
    state = s["h0"].double() if c["state"] else zero
    h = torch.zeros_like(f)
    before = torch.zeros_like(f)
    for t in range(S):
        before[t] = state
        new = a[t] * state + w[t] * x[t]
        if held is not None:
            h[t] = torch.where(held[t], new, zero)
            state = torch.where(held[t], new, state)
        else:
            h[t] = new
            state = new
    back = lambda t: _rec_stored(c, t.permute(1, 2, 0))  # noqa: E731
    res = [back(h), state]
    if not c["train"]:
        return res
    into = s["dh_last"].double() if c["state"] else zero
    total = torch.zeros_like(f)
    for t in reversed(range(S)):
        g = into + wide["dh"][t]
        if held is not None:
            total[t] = torch.where(held[t], g, zero)
            into = torch.where(held[t], a[t] * g, into)
        else:
            total[t] = g
            into = a[t] * g
    res += [back(total * w)]
    if c["input_gate"]:
        res += [back(total * before * a * (1 - a)), back(total * x * w * (1 - w))]
    else:
        res += [back(total * (before - x) * a * torch.special.expit(-f))]
    return res + [into] if c["state"] else res


def _rec_work(c):
    held, rows, B, D = sum(_rec_lengths(c)), c["batch"] * c["steps"], c["batch"], c["dim"]
    ins = 3 if c["input_gate"] else 2  # x, f (and i)
    state = 2 if c["state"] else 1     # h_last, and h0
    n = ins * held + rows + state * B
    if c["train"]:
        n += held + ins * rows + (2 * B if c["state"] else 0)  # dh, the gradients, dh_last and dh0
    return {"bytes": 4 * n * D, "flops": (30 if c["train"] else 12) * held * D}


# ------------------------------------------------- gated feed-forward layer
#   Z = X W + b, [batch, 2 hidden]: gate and up;  H = act(gate) * up
def _ffn_prepare(c, g):
    N, D, F = c["batch"], c["dim"], c["hidden"]
    s = {"X": _randn(g, D, N), "W": _randn(g, 2 * F, D) / math.sqrt(D), "b": 0.1 * _randn(g, 2 * F) if c["bias"] else None,
         "H": _empty(F, N), "Z": _empty(2 * F, N) if c["train"] else None}
    if c["train"]:
        s.update(dH=_randn(g, F, N) / N, dX=_empty(D, N), dW=_empty(2 * F, D), db=_empty(2 * F) if c["bias"] else None)
    return s


def _ffn_act(c, z):
    """The activation and its derivative."""
    if c["act"] == "silu":
        r = _sigmoid(z)
        return z * r, r * (1.0 + z * (1.0 - r))
    cdf = 0.5 * torch.special.erfc(z * -math.sqrt(0.5))
    return z * cdf, cdf + z * (torch.exp(-0.5 * z * z) / math.sqrt(2.0 * math.pi))


def _ffn_run(c, s):
    N, D, F = c["batch"], c["dim"], c["hidden"]
    if own:
        from cppnet_amd import ops
        ops.gated_ffn_forward(s["X"], s["W"], s["b"], s["H"], s["Z"], N, D, F, act=c["act"])
        if not c["train"]:
            return [s["H"]]
        ops.gated_ffn_backward(s["X"], s["W"], s["Z"], s["dH"], s["dX"], s["dW"], s["db"], N, D, F, act=c["act"])
        return [s[k] for k in ("H", "Z", "dX", "dW", "db") if s[k] is not None]
    Z = torch.matmul(s["W"], s["X"])
    if c["bias"]:
        Z = Z + s["b"][:, None]
    y, dy = _ffn_act(c, Z[:F])
    H = y * Z[F:]
    if not c["train"]:
        return [H]
    dZ = torch.cat([s["dH"] * Z[F:] * dy, s["dH"] * y])
    res = [H, Z, torch.matmul(s["W"].t(), dZ), torch.matmul(dZ, s["X"].t())]
    return res + [dZ.sum(1)] if c["bias"] else res


def _ffn_exact(c, s):
    F = c["hidden"]
    leaves = [t.double().requires_grad_(c["train"]) for t in (s["X"], s["W"], s["b"]) if t is not None]
    Z = torch.matmul(leaves[1], leaves[0])
    if c["bias"]:
        Z = Z + leaves[2][:, None]
    gate = Z[:F] * torch.special.expit(Z[:F]) if c["act"] == "silu" else Z[:F] * torch.special.ndtr(Z[:F])
    H = gate * Z[F:]
    if not c["train"]:
        return [H.detach()]
    return [H.detach(), Z.detach()] + list(torch.autograd.grad(H, leaves, s["dH"].double()))


def _ffn_work(c):
    N, D, F = c["batch"], c["dim"], c["hidden"]
    b = 2 * F if c["bias"] else 0
    if not c["train"]:
        return {"bytes": 4 * (N * D + 2 * D * F + b + N * F), "flops": 4 * N * D * F}
    # X, W, b, dH in; H, Z and the gradients out
    return {"bytes": 4 * (2 * N * D + 4 * D * F + 2 * b + 4 * N * F), "flops": 12 * N * D * F}


# ----------------------------- dropout by position, norm of a residual's sum
#   element j is kept where the top 24 bits of the mixed 64-bit word of (seed,
#   position + j) are below (1 - p) 2^24, and then times 1 / (1 - p)
SEED = 0x1234567


def _word(v):
    """A 64-bit constant as the signed number of the same bits."""
    return v - (1 << 64) if v >> 63 else v


def _kept(n, p, at):
    """Whether each of n elements from position `at` (a tensor) on is kept."""
    z = (at + torch.arange(n, device=at.device)) * _word(0x9E3779B97F4A7C15) + SEED
    z = (z ^ ((z >> 30) & ((1 << 34) - 1))) * _word(0xBF58476D1CE4E5B9)
    z = (z ^ ((z >> 27) & ((1 << 37) - 1))) * _word(0x94D049BB133111EB)
    top = ((z ^ ((z >> 31) & ((1 << 33) - 1))) >> 40) & ((1 << 24) - 1)
    return top < _limit(p)


def _limit(p):
    return math.ceil(float(np.float32(1) - np.float32(p)) * 2 ** 24)


def _dropped(x, kept, p):
    return torch.where(kept.view_as(x), x * (1.0 / (1.0 - p)), torch.zeros_like(x))


def _kept_exact(n, p, at):
    with np.errstate(over="ignore"):
        z = np.uint64(SEED) + (np.uint64(at) + np.arange(n, dtype=np.uint64)) * np.uint64(0x9E3779B97F4A7C15)
        z = (z ^ (z >> np.uint64(30))) * np.uint64(0xBF58476D1CE4E5B9)
        z = (z ^ (z >> np.uint64(27))) * np.uint64(0x94D049BB133111EB)
    u = ((z ^ (z >> np.uint64(31))) >> np.uint64(40)).astype(np.float32) / np.float32(2 ** 24)
    return u < np.float32(1) - np.float32(p)


def _factor_exact(shape, p, at):
    kept = torch.from_numpy(_kept_exact(math.prod(shape), p, at)).cuda().view(shape)
    return kept.double() / (1.0 - float(np.float32(p)))


def _drop_prepare(c, g):
    n = c["rows"] * c["dim"]
    s = {"x": _randn(g, n), "y": _empty(n),
         "counter": torch.randint(0, 1 << 40, (1,), generator=g, device="cuda", dtype=torch.int64)}
    if c["train"]:
        s.update(dy=_randn(g, n), dx=_empty(n))
    return s


def _drop_run(c, s):
    if own:
        from cppnet_amd import ops
        ops.dropout_seeded(s["x"], s["y"], c["p"], SEED, counter=s["counter"])
        if not c["train"]:
            return [s["y"]]
        ops.dropout_seeded(s["dy"], s["dx"], c["p"], SEED, counter=s["counter"])
        return [s["y"], s["dx"]]
    kept = _kept(s["x"].numel(), c["p"], s["counter"])
    y = _dropped(s["x"], kept, c["p"])
    return [y, _dropped(s["dy"], kept, c["p"])] if c["train"] else [y]


def _drop_exact(c, s):
    m = _factor_exact(s["x"].shape, c["p"], int(s["counter"]))
    return [s[k].double() * m for k in (("x", "dy") if c["train"] else ("x",))]


def _drop_work(c):
    n = c["rows"] * c["dim"] * (2 if c["train"] else 1)
    return {"bytes": 8 * n, "flops": n}


EPS = 1e-5


def _norm_prepare(c, g):
    N, F = c["rows"], c["dim"]
    # a residual stream is larger than what a block adds to it, and some features are larger than others
    s = {"x": _randn(g, F, N), "residual": 3.0 * _randn(g, F, N) * torch.exp(0.5 * _randn(g, F))[:, None],
         "gamma": 1.0 + 0.1 * _randn(g, F), "y": _empty(F, N), "sum": _empty(F, N), "rstd": _empty(N),
         "counter": torch.randint(0, 1 << 40, (1,), generator=g, device="cuda", dtype=torch.int64) if c["p"] else None}
    if c["train"]:
        s.update(dy=_randn(g, F, N), dsum=_randn(g, F, N), dx=_empty(F, N), dresidual=_empty(F, N) if c["p"] else None,
                 dgamma=_empty(F))
    return s


def _norm_run(c, s):
    N, F, p = c["rows"], c["dim"], c["p"]
    if own:
        from cppnet_amd import ops
        how = {"p": p, "seed": SEED, "counter": s["counter"]}
        ops.rms_norm_forward(s["x"], s["residual"], s["gamma"], s["y"], s["sum"], s["rstd"], N, F, eps=EPS, **how)
        if not c["train"]:
            return [s["sum"], s["y"]]
        ops.rms_norm_backward(s["sum"], s["rstd"], s["gamma"], s["dy"], s["dsum"], s["dx"], s["dresidual"], s["dgamma"],
                              N, F, **how)
        return [s[k] for k in ("sum", "y", "dx", "dresidual", "dgamma") if s[k] is not None]
    kept = _kept(F * N, p, s["counter"]) if p else None
    t = s["residual"] + (_dropped(s["x"], kept, p) if p else s["x"])
    r = 1.0 / torch.sqrt((t * t).mean(0) + EPS)
    unit = t * r
    y = unit * s["gamma"][:, None]
    if not c["train"]:
        return [t, y]
    dn = s["dy"] * s["gamma"][:, None]
    d = s["dsum"] + r * (dn - unit * (dn * unit).mean(0))
    dgamma = (s["dy"] * unit).sum(1)
    return [t, y, _dropped(d, kept, p), d, dgamma] if p else [t, y, d, dgamma]


def _norm_exact(c, s):
    leaves = [s[k].double().requires_grad_(c["train"]) for k in ("x", "residual", "gamma")]
    x = leaves[0] * _factor_exact(s["x"].shape, c["p"], int(s["counter"])) if c["p"] else leaves[0]
    t = leaves[1] + x
    y = leaves[2][:, None] * t * torch.rsqrt(t.square().mean(0, keepdim=True) + EPS)
    if not c["train"]:
        return [t.detach(), y.detach()]
    d = torch.autograd.grad([t, y], leaves, [s["dsum"].double(), s["dy"].double()])
    return [t.detach(), y.detach()] + ([d[0], d[1], d[2]] if c["p"] else [d[1], d[2]])


def _norm_work(c):
    n, N, F = c["rows"] * c["dim"], c["rows"], c["dim"]
    if not c["train"]:
        return {"bytes": 4 * (4 * n + F + N), "flops": 5 * n}
    # x, residual, dy, dsum in; sum, y, dx (and dresidual) out
    return {"bytes": 4 * ((8 if c["p"] else 7) * n + 2 * F + N), "flops": 15 * n}


# -------------------------------------------------------------------- cases
KINDS = {
    "recurrence": (_rec_prepare, _rec_run, _rec_exact, _rec_work),
    "ffn": (_ffn_prepare, _ffn_run, _ffn_exact, _ffn_work),
    "norm": (_norm_prepare, _norm_run, _norm_exact, _norm_work),
    "dropout": (_drop_prepare, _drop_run, _drop_exact, _drop_work),
}


def _rec(name, batch, steps, dim, rows=BY_SAMPLE, input_gate=False, state=False, ragged=False, train=True):
    return {"name": name, "kind": "recurrence", "batch": batch, "steps": steps, "dim": dim, "rows": rows,
            "input_gate": input_gate, "state": state, "ragged": ragged, "train": train}


def _ffn(name, batch, dim, hidden, act="silu", bias=False, train=True):
    return {"name": name, "kind": "ffn", "batch": batch, "dim": dim, "hidden": hidden, "act": act, "bias": bias,
            "train": train}


def _norm(name, rows, dim, p=0.0, train=True):
    return {"name": name, "kind": "norm", "rows": rows, "dim": dim, "p": p, "train": train}


def _drop(name, rows, dim, p, train=True):
    return {"name": name, "kind": "dropout", "rows": rows, "dim": dim, "p": p, "train": train}


def listed():
    return [
        # generation: one step of eight sequences, state in and out
        _rec("recurrence_token", 8, 1, 512, state=True, train=False),
        # training at the framework's transformer configuration: 32 x 256, width 512
        _rec("recurrence_config", 32, 256, 512),
        # a padded batch in the reference's row order, odd sizes, gates of its own, state carried on
        _rec("recurrence_ragged", 5, 1001, 333, rows=REF, input_gate=True, state=True, ragged=True),
        # long sequences, few of them
        _rec("recurrence_long", 2, 32768, 1024),
        # generation: one token of four sequences through the configuration's feed-forward sizes
        _ffn("ffn_token", 4, 512, 2048, train=False),
        # a small batch of odd sizes
        _ffn("ffn_ragged", 1021, 513, 1365),
        # training of a wide layer with a bias
        _ffn("ffn_large", 8192, 1024, 4096, act="gelu", bias=True),
        # generation: the norm before a block, eight rows
        _norm("norm_token", 8, 512, train=False),
        # training at the configuration's sizes, a tenth of the branch dropped
        _norm("norm_config", 8192, 512, p=0.1),
        # wide rows, an odd number of both
        _norm("norm_wide", 4097, 4099),
        # dropout of a small batch's activations
        _drop("dropout_small", 64, 512, 0.5),
        # of the configuration's feed-forward activations
        _drop("dropout_ffn", 8192, 2048, 0.1),
    ]


def draw(rng):
    kind = rng.choice(["recurrence", "recurrence", "ffn", "ffn", "norm", "dropout"])
    if kind == "recurrence":
        steps = rng.choice([1, 2, _log(rng, 3, 32768), _log(rng, 3, 32768), _log(rng, 64, 4096), _log(rng, 64, 4096)])
        dim = _log(rng, 16, 1024)
        batch = _log(rng, 1, max(1, min(128, 32768 * 1024 // (steps * dim))))
        c = _rec("", batch, steps, dim, rng.choice([REF, BY_SAMPLE]), rng.random() < 0.4, rng.random() < 0.5,
                 rng.random() < 0.4, rng.random() < 0.7)
    elif kind == "ffn":
        batch = _log(rng, 1, 64) if rng.random() < 0.3 else _log(rng, 64, 8192)
        c = _ffn("", batch, _log(rng, 32, 1024), _log(rng, 64, 4096), rng.choice(["silu", "gelu"]), rng.random() < 0.3,
                 rng.random() < 0.6)
    elif kind == "norm":
        dim = _log(rng, 32, 8192)
        rows = _log(rng, 1, max(1, min(16384, 4096 * 4096 // dim)))
        c = _norm("", rows, dim, rng.choice([0.0, 0.0, 0.1, 0.3]), rng.random() < 0.7)
    else:
        c = _drop("", _log(rng, 1, 8192), _log(rng, 16, 2048), rng.choice([0.05, 0.1, 0.3, 0.5]), rng.random() < 0.7)
    c.pop("name", None)
    return c


def prepare(case, seed):
    state = KINDS[case["kind"]][0](case, _gen(seed))
    state["case"] = case
    return state


def run(state):
    c = state["case"]
    return KINDS[c["kind"]][1](c, state)


def exact(case, seed):
    return KINDS[case["kind"]][2](case, KINDS[case["kind"]][0](case, _gen(seed)))


def work(case):
    return KINDS[case["kind"]][3](case)
