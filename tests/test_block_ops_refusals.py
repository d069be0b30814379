"""What the operators of a recurrent block refuse, before any GPU call."""
import ctypes as C

import pytest
import torch

from cppnet_amd import _capi, ops

P = C.c_void_p(16)  # never dereferenced: validation fails first


def refused(name, *args):
    lib = _capi.load()
    st = getattr(lib, name)(*args)
    return st, lib.cnhip_last_error().decode()


@pytest.mark.parametrize("change,word", [
    ({"n": -1}, "negative"), ({"p": 1.0}, "probability"), ({"p": -0.1}, "probability"), ({"p": float("nan")}, "probability"),
    ({"x": None}, "NULL"), ({"y": None}, "NULL"),
])
def test_dropout_refusals(change, word):
    a = dict(x=P, y=P, n=4, p=0.5) | change
    st, msg = refused("cnhip_dropout_seeded", a["x"], a["y"], a["n"], a["p"], 1, 0, None, None)
    assert st == 1 and word in msg and "dropout_seeded" in msg


def test_dropout_of_nothing_and_advance():
    assert refused("cnhip_dropout_seeded", None, None, 0, 0.5, 1, 0, None, None)[0] == 0
    st, msg = refused("cnhip_dropout_advance", None, 4, None)
    assert st == 1 and "NULL" in msg


@pytest.mark.parametrize("change,word", [
    ({"N": 0}, "bad shape"), ({"F": -3}, "bad shape"), ({"N": 1 << 28}, "too large"), ({"F": 1 << 31}, "too large"),
    ({"p": 1.0}, "probability"), ({"x": None}, "NULL"), ({"gamma": None}, "NULL"),
])
def test_norm_refusals(change, word):
    a = dict(x=P, gamma=P, N=2, F=3, p=0.0) | change
    st, msg = refused("cnhip_rms_norm_forward", a["x"], None, a["gamma"], P, None, None, a["N"], a["F"], 1e-5, a["p"], 1, 0,
                      None, None)
    assert st == 1 and word in msg and "rms_norm_forward" in msg
    st, msg = refused("cnhip_rms_norm_backward", a["x"], P, a["gamma"], P, None, P, None, P, a["N"], a["F"], a["p"], 1, 0,
                      None, 0, None)
    assert st == 1 and word in msg and "rms_norm_backward" in msg


@pytest.mark.parametrize("eps", [0.0, -1e-5, float("inf"), float("nan")])
def test_norm_refuses_a_bad_eps(eps):
    st, msg = refused("cnhip_rms_norm_forward", P, None, P, P, None, None, 2, 3, eps, 0.0, 1, 0, None, None)
    assert st == 1 and "eps" in msg


def test_norm_backward_refusals():
    for args in ([None, P, P, P, None, P, None, P], [P, None, P, P, None, P, None, P], [P, P, P, P, None, None, None, P],
                 [P, P, P, P, None, P, None, None], [P, P, P, None, None, P, None, P]):
        st, msg = refused("cnhip_rms_norm_backward", *args, 2, 3, 0.0, 1, 0, None, 0, None)
        assert st == 1 and "NULL" in msg
    st, msg = refused("cnhip_rms_norm_backward", P, P, P, P, None, P, None, P, 2, 3, 0.0, 1, 0, None, 2, None)
    assert st == 1 and "accumulate" in msg


@pytest.mark.parametrize("change,word", [
    ({"B": 0}, "bad shape"), ({"S": 0}, "bad shape"), ({"D": -1}, "bad shape"), ({"rows": 2}, "row order"),
    ({"S": 1 << 30}, "too large"), ({"B": 1 << 25, "D": 1 << 25}, "too large"), ({"x": None}, "NULL"), ({"f": None}, "NULL"),
])
def test_recurrence_refusals(change, word):
    a = dict(x=P, f=P, B=2, S=3, D=4, rows=1) | change
    dims = (a["B"], a["S"], a["D"], None, a["rows"], None)
    st, msg = refused("cnhip_linear_recurrence_forward", a["x"], a["f"], None, None, P, None, *dims)
    assert st == 1 and word in msg and "linear_recurrence_forward" in msg
    st, msg = refused("cnhip_linear_recurrence_backward", a["x"], a["f"], None, None, P, P, None, P, P, None, None, *dims)
    assert st == 1 and word in msg and "linear_recurrence_backward" in msg


def test_recurrence_gradient_of_the_input_gate_goes_with_it():
    for i, di in ((P, None), (None, P)):
        st, msg = refused("cnhip_linear_recurrence_backward", P, P, i, None, P, P, None, P, P, di, None, 2, 3, 4, None, 0, None)
        assert st == 1 and "di goes with i" in msg


@pytest.mark.parametrize("change,word", [
    ({"N": 0}, "bad shape"), ({"D": 0}, "bad shape"), ({"F": -1}, "bad shape"), ({"act": 4}, "activation"),
    ({"act": -1}, "activation"), ({"X": None}, "NULL"), ({"N": 1 << 30}, "too large"), ({"F": 1 << 28}, "too large"),
    ({"D": 1 << 22}, "too large"), ({"N": 1 << 26}, "too large"), ({"F": 1 << 25}, "too large"),
])
def test_ffn_refusals(change, word):
    a = dict(X=P, N=2, D=3, F=4, act=0) | change
    shape = (a["N"], a["D"], a["F"], a["act"])
    st, msg = refused("cnhip_gated_ffn_forward", a["X"], P, None, P, None, *shape, None)
    assert st == 1 and word in msg and "gated_ffn_forward" in msg
    st, msg = refused("cnhip_gated_ffn_backward", a["X"], P, P, P, P, P, None, *shape, 0, None)
    assert st == 1 and word in msg and "gated_ffn_backward" in msg


def test_ffn_backward_refusals():
    st, msg = refused("cnhip_gated_ffn_backward", P, P, P, P, P, P, None, 2, 3, 4, 0, 2, None)
    assert st == 1 and "accumulate" in msg
    for k in range(6):
        args = [P] * 6
        args[k] = None
        st, msg = refused("cnhip_gated_ffn_backward", *args, None, 2, 3, 4, 0, 0, None)
        assert st == 1 and "NULL" in msg


def test_front_end_refusals():
    x, c = torch.zeros(4), torch.zeros(1, dtype=torch.int64)
    with pytest.raises(TypeError, match="device tensor"):
        ops.dropout_seeded(x, x, 0.5, 1)
    with pytest.raises(TypeError, match="device tensor"):
        ops.dropout_advance(c, 4)
    with pytest.raises(TypeError, match="device tensor"):
        ops.rms_norm_forward(x, None, x, x, None, None, 2, 2)
    with pytest.raises(TypeError, match="device tensor"):
        ops.linear_recurrence_forward(x, x, None, None, x, None, 1, 2, 2)
    with pytest.raises(TypeError, match="device tensor"):
        ops.gated_ffn_forward(x, x, None, x, None, 2, 2, 2)
    with pytest.raises(ValueError, match="F must be positive"):
        ops.rms_norm_backward(x, x, x, x, None, x, None, x, 2, 0)
    with pytest.raises(ValueError, match="S must be positive"):
        ops.linear_recurrence_backward(x, x, None, None, x, x, None, x, x, None, None, 1, 0, 2)
    with pytest.raises(ValueError, match="hidden must be positive"):
        ops.gated_ffn_backward(x, x, x, x, x, x, None, 2, 2, 0)
    with pytest.raises(ValueError, match="act must be one of silu, gelu"):
        ops._gate("tanh")


class Fake(torch.Tensor):
    """A tensor that passes for a device tensor."""
    is_cuda = True


def test_a_counter_is_64_bits_wide_and_nothing_else_is():
    x = torch.zeros(6).as_subclass(Fake)
    wide, narrow = torch.zeros(1, dtype=torch.int64).as_subclass(Fake), torch.zeros(1, dtype=torch.int32).as_subclass(Fake)
    assert ops._held(x, (wide, "counter", 1, torch.int64))
    with pytest.raises(TypeError, match="counter: expected torch.int64"):
        ops._held(x, (narrow, "counter", 1, torch.int64))
    with pytest.raises(TypeError, match="ids: expected float32/int32/uint8"):
        ops._held(x, (wide, "ids", 1, torch.int32))
    with pytest.raises(TypeError, match="expected float32/int32/uint8"):
        ops._p(wide)
