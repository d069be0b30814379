"""What the language-model operators refuse, before any GPU call."""
import ctypes as C

import pytest
import torch

from cppnet_amd import _capi, ops

D = C.c_void_p(16)  # never dereferenced: validation fails first


def refused(name, *args):
    lib = _capi.load()
    st = getattr(lib, name)(*args)
    return st, lib.cnhip_last_error().decode()


@pytest.mark.parametrize("change,word", [
    ({"B": 0}, "bad shape"), ({"S": -1}, "bad shape"), ({"V": 0}, "bad shape"), ({"D": 0}, "bad shape"),
    ({"rows": 2}, "row order"), ({"scale": float("nan")}, "scale"), ({"scale": float("inf")}, "scale"),
    ({"ids": None}, "NULL"), ({"V": 1 << 31}, "too many"), ({"S": 1 << 30}, "too many"), ({"B": 1 << 16, "S": 1 << 15}, "too many"),
])
def test_token_embedding_refusals(change, word):
    a = dict(ids=D, B=2, S=3, V=5, D=7, scale=1.0, rows=0) | change
    shape = (a["B"], a["S"], a["V"], a["D"], a["scale"])
    st, msg = refused("cnhip_token_embedding_forward", a["ids"], D, D, *shape, None, a["rows"], None)
    assert st == 1 and word in msg and "token_embedding_forward" in msg
    st, msg = refused("cnhip_token_embedding_backward", a["ids"], D, D, *shape, 0, a["rows"], None)
    assert st == 1 and word in msg and "token_embedding_backward" in msg


def test_token_embedding_refuses_a_bad_accumulate():
    st, msg = refused("cnhip_token_embedding_backward", D, D, D, 1, 1, 1, 1, 1.0, 2, 0, None)
    assert st == 1 and "accumulate" in msg


@pytest.mark.parametrize("change,word,status", [
    ({"B": 0}, "bad shape", 1), ({"Sq": 0}, "bad shape", 1), ({"Sk": 0}, "bad shape", 1), ({"H": 0}, "bad shape", 1),
    ({"KH": 0}, "bad shape", 1), ({"dh": 0}, "bad shape", 1), ({"H": 3}, "multiple", 1), ({"dh": 129}, "128", 4),
    ({"rows": -1}, "row order", 1), ({"causal": 2}, "causal", 1), ({"causal": 0, "q_start": D}, "q_start", 1),
    ({"scale": float("inf")}, "scale", 1), ({"q": None}, "NULL", 1), ({"B": 40000, "H": 2}, "65535", 1),
    ({"Sq": 1 << 30}, "too long", 1), ({"Sk": 1 << 30}, "too long", 1),
])
def test_attention_refusals(change, word, status):
    a = dict(q=D, B=2, Sq=3, Sk=5, H=4, KH=2, dh=8, scale=1.0, causal=1, q_start=None, rows=0) | change
    dims = tuple(a[n] for n in ("B", "Sq", "Sk", "H", "KH", "dh", "scale", "causal"))
    st, msg = refused("cnhip_attention_forward", a["q"], D, D, D, None, *dims, None, a["q_start"], a["rows"], None)
    assert st == status and word in msg and "attention_forward" in msg
    st, msg = refused("cnhip_attention_backward", a["q"], *[D] * 8, *dims, None, a["q_start"], a["rows"], None)
    assert st == status and word in msg and "attention_backward" in msg


def test_attention_backward_needs_lse():
    st, msg = refused("cnhip_attention_backward", D, D, D, D, None, *[D] * 4, 1, 1, 1, 1, 1, 1, 1.0, 0, None, None, 0, None)
    assert st == 1 and "NULL" in msg


@pytest.mark.parametrize("change,word", [
    ({"N": 0}, "bad shape"), ({"D": 0}, "bad shape"), ({"V": 0}, "bad shape"), ({"X": None}, "NULL"),
    ({"red": 2}, "reduction"), ({"V": 1 << 31}, "too large"), ({"N": 1 << 31}, "too large"),
])
def test_linear_ce_refusals(change, word):
    a = dict(X=D, N=2, D=3, V=5, red=0) | change
    shape = (a["N"], a["D"], a["V"], a["red"])
    st, msg = refused("cnhip_linear_ce_forward", a["X"], D, None, D, D, D, *shape, None, None)
    assert st == 1 and word in msg and "linear_ce_forward" in msg
    st, msg = refused("cnhip_linear_ce_head", a["X"], D, None, D, D, D, D, D, None, *shape, 0, None, None)
    assert st == 1 and word in msg and "linear_ce_head" in msg


def test_linear_ce_head_refusals():
    st, msg = refused("cnhip_linear_ce_head", D, D, D, D, D, D, D, D, None, 2, 3, 5, 0, 0, None, None)
    assert st == 1 and "db" in msg
    st, msg = refused("cnhip_linear_ce_head", D, D, None, D, D, D, D, D, None, 2, 3, 5, 0, 2, None, None)
    assert st == 1 and "accumulate" in msg
    st, msg = refused("cnhip_linear_ce_head", D, D, None, D, D, D, None, D, None, 2, 3, 5, 0, 0, None, None)
    assert st == 1 and "NULL" in msg


def test_front_end_refuses_host_tensors_and_bad_sizes():
    x, i = torch.zeros(4), torch.zeros(4, dtype=torch.int32)
    with pytest.raises(TypeError, match="device tensor"):
        ops.token_embedding_forward(i, x, x, 2, 2, 2, 2)
    with pytest.raises(TypeError, match="device tensor"):
        ops.attention_forward(x, x, x, x, None, 1, 2, 2, 1, 1, 2)
    with pytest.raises(TypeError, match="device tensor"):
        ops.linear_ce_forward(x, x, None, i, x, x, 2, 2, 2)
    with pytest.raises(ValueError, match="head_dim must be positive"):
        ops.attention_forward(x, x, x, x, None, 1, 2, 2, 1, 1, 0)
    with pytest.raises(ValueError, match="classes must be positive"):
        ops.linear_ce_forward(x, x, None, i, x, x, 2, 2, 0)
    with pytest.raises(ValueError, match="S must be positive"):
        ops.token_embedding_backward(i, x, x, 2, -2, 2, 2)


def test_operands_are_held_to_their_sizes_types_and_device():
    class Fake(torch.Tensor):
        """A tensor that passes for a device tensor."""
        is_cuda = True

    def fake(n, dtype=torch.float32):
        return torch.zeros(n, dtype=dtype).as_subclass(Fake)

    x = fake(6)
    assert ops._held(x, (x, "x", 6, torch.float32), (None, "y", 3, torch.float32))[1] is None
    with pytest.raises(ValueError, match="y: expected 5 values, got 6"):
        ops._held(x, (fake(6), "y", 5, torch.float32))
    with pytest.raises(TypeError, match="ids: expected torch.int32"):
        ops._held(x, (fake(6), "ids", 6, torch.int32))
    with pytest.raises(ValueError, match="contiguous"):
        ops._held(x, (fake(6)[::2], "y", 3, torch.float32))
    other = fake(6)
    class Elsewhere(Fake):
        device = torch.device("cuda:1")
    with pytest.raises(ValueError, match="is on cuda:1"):
        ops._held(x, (other.as_subclass(Elsewhere), "y", 6, torch.float32))
