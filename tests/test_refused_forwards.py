"""A forward that is refused leaves a layer as the last one left it: backward repeats that one's mask and reads its
matrices, and the next forward takes the offset that this one would have had.  No device is touched: the entry
points are stand-ins."""
import pytest

from lbann_amd import layers as L
from tests.test_cpp_adapter import driver

STATE = ("m_offset", "m_kept", "_next", "branch", "h", "gate", "residual", "activations", "m_statistics", "m_has_residual")


@pytest.fixture
def calls(monkeypatch):
    made = []
    status = {"refuse": False}

    def entry(name, dtype):
        def f(*args):
            if status["refuse"]:
                raise L.LbnError(name, -1, "refused")
            made.append((name, args))
        return f
    monkeypatch.setattr(L, "_stream_for", lambda m: 0)
    monkeypatch.setattr(L, "_entry", entry)
    made_status = made, status
    yield made_status
    L._SAVED.clear()


def matrix(height=8, width=6):
    return L.DeviceMatrix(height, width, device="cpu", fill=1.0)


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("offset", [None, 17])
@pytest.mark.parametrize("how", ["call", "step"])
def test_residual_norm(calls, training, offset, how):
    made, status = calls
    layer = L.residual_norm_layer(8, "rms", "rms", keep_prob=0.5, device="cpu")
    layer.forward(matrix(), matrix())
    layer.forward(matrix(), matrix())
    before = {name: getattr(layer, name) for name in STATE}
    if how == "call":
        status["refuse"] = True
    else:
        layer.m_step = 1.5  # no device vector
    with pytest.raises((L.LbnError, ValueError, AttributeError)):
        layer.forward(matrix(), None, matrix(), training=training, offset=offset)
    for name, value in before.items():
        assert getattr(layer, name) is value or getattr(layer, name) == value, name
    status["refuse"], layer.m_step = False, None
    layer.backward(matrix(), matrix())
    forward = [args for name, args in made if name.endswith("fwd")][-1]
    name, backward = made[-1]
    assert name.endswith("bwd") and backward[8] == forward[8]     # the block's output
    assert (0.5, 0, 1) == tuple(forward[19:22]) == tuple(backward[18:21])   # keep probability, seed, offset
    layer.forward(matrix(), matrix())
    assert layer.m_offset == 2


def test_dropout(calls):
    made, status = calls
    layer = L.dropout_layer(0.5, device="cpu")
    layer.forward(matrix())
    layer.forward(matrix())
    status["refuse"] = True
    for kwargs in ({}, {"training": False}, {"offset": 9}):
        with pytest.raises(L.LbnError):
            layer.forward(matrix(), **kwargs)
        assert (layer.m_offset, layer.m_kept, layer._next) == (1, 0.5, 2)
    status["refuse"] = False
    layer.backward(matrix())
    assert made[-1][1][3:6] == (0.5, 0, 1)
    layer.forward(matrix())
    assert layer.m_offset == 2


def test_adapter():
    assert driver().drv_refused_dropout() == 0
