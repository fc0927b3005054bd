"""Calls that write over what a residual norm's backward is still to read: that backward is refused, no other is.  The
bookkeeping is host code: here the entry points are stand-ins that compute nothing (tests/test_gpu_in_place_streams.py
runs the same on a device)."""
import copy
import gc
import pickle

import numpy as np
import pytest
import torch

from lbann_amd import layers as L

N, W = 8, 6


@pytest.fixture(autouse=True)
def no_device(monkeypatch):
    monkeypatch.setattr(L, "_stream_for", lambda m: 0)
    monkeypatch.setattr(L, "_entry", lambda name, dtype: lambda *args: None)
    monkeypatch.setattr(L, "_stream", lambda: None)
    monkeypatch.setattr(L, "call", lambda *args: None)
    L._SAVED.clear()
    yield
    gc.collect()
    L._SAVED.clear()


def matrix(height=N, width=W):
    return L.DeviceMatrix(height, width, device="cpu", fill=1.0)


def norm(branch_norm="none", output_norm="rms"):
    return L.residual_norm_layer(N, branch_norm, output_norm, device="cpu")


def two_in_a_row(first, second, training=True, view=lambda m: m):
    first.forward(matrix(), matrix())
    second.forward(matrix(), view(first.residual), training=training, in_place=True)


@pytest.mark.parametrize("training", [True, False])
@pytest.mark.parametrize("view", [lambda m: m, lambda m: L.DeviceMatrix.attach(m.tensor, N), lambda m: L.DeviceMatrix.attach(m.tensor[2:], N)],
                         ids=["itself", "attached", "some columns"])
def test_stream_of_the_layer_before(training, view):
    first, second = norm(), norm("rms", "rms")
    first.forward(matrix(), matrix())
    stream = view(first.residual)
    second.forward(matrix(width=stream.width), stream, training=training, in_place=True)
    if training:
        second.backward(matrix(width=stream.width), matrix(width=stream.width))
    with pytest.raises(ValueError, match="overwritten"):
        first.backward(matrix(), matrix())
    # the next forward starts again
    first.forward(matrix(), matrix())
    first.backward(matrix(), matrix())


def test_a_stack_in_one_buffer():
    layers = [norm() for _ in range(4)]
    stream = matrix()
    for layer in layers:
        layer.forward(matrix(), stream, in_place=True)
    layers[-1].backward(matrix(), matrix())
    for layer in layers[:-1]:
        with pytest.raises(ValueError, match="overwritten"):
            layer.backward(matrix(), matrix())


def test_a_stack_without_output_norms_needs_no_stream():
    first, second = norm("rms", "none"), norm("rms", "none")
    two_in_a_row(first, second)
    second.backward(None, matrix())
    first.backward(None, matrix())


def test_streams_of_their_own():
    first, second = norm(), norm()
    both = torch.ones(W, 2 * N)
    lower, upper = L.DeviceMatrix.attach(both[:, :N], N), L.DeviceMatrix.attach(both[:, N:], N)
    first.forward(matrix(), lower, in_place=True)
    second.forward(matrix(), upper, in_place=True)     # beside it, in the same buffer
    first.backward(matrix(), matrix())
    second.backward(matrix(), matrix())
    columns = torch.ones(2 * W, N)
    first.forward(matrix(), L.DeviceMatrix.attach(columns[:W], N), in_place=True)
    second.forward(matrix(), L.DeviceMatrix.attach(columns[W:], N), in_place=True)
    first.backward(matrix(), matrix())
    first.forward(matrix(), L.DeviceMatrix.attach(columns[:W], N), in_place=True)     # its own stream again
    first.backward(matrix(), matrix())
    first.forward(matrix(), matrix())
    second.forward(matrix(), first.residual)           # not in place
    first.backward(matrix(), matrix())


@pytest.mark.parametrize("writer", [lambda m: L.dropout_layer(0.5, device="cpu").forward(m, in_place=True),
                                    lambda m: L.dropout_layer(0.5, device="cpu").backward(m, in_place=True),
                                    lambda m: L.softmax_layer(device="cpu").forward(m, in_place=True),
                                    lambda m: L.logits_adjust_layer(N).forward(m, in_place=True),
                                    lambda m: norm().forward(m, matrix(), training=False, in_place=True)],
                         ids=["dropout", "dropout backward", "softmax", "logits", "y over the branch"])
@pytest.mark.parametrize("which", ["stream", "branch", "gate", "branch that is not read"])
def test_other_writers(writer, which):
    kinds = ("none", "rms") if which.endswith("not read") else ("rms", "rms")
    layer, branch, gate = norm(*kinds), matrix(), matrix() if which == "gate" else None
    layer.forward(branch, matrix(), gate)
    writer({"stream": layer.residual, "gate": gate}.get(which, branch))
    if which.endswith("not read"):
        layer.backward(matrix(), matrix())
    else:
        with pytest.raises(ValueError, match="overwritten"):
            layer.backward(matrix(), matrix())


def test_saved_state():
    first, second = norm(), norm()
    two_in_a_row(first, second)
    kept = matrix()
    first.bind_saved(first.branch, kept, first.m_statistics)
    first.backward(matrix(), matrix())
    second.forward(matrix(), kept, in_place=True)
    with pytest.raises(ValueError, match="overwritten"):
        first.backward(matrix(), matrix())


def test_places_of_their_own():
    x, gate = matrix(), matrix(width=1)
    for args in ((x, x, None, True, "rms", "rms"), (x, x, gate, True, "none", "none"), (x, x, None, False, "none", "rms"),
                 (matrix(), gate, gate, True, "none", "none")):
        branch, residual, g, training, n1, n2 = args
        if residual is gate:
            branch, residual, g = matrix(), x, L.DeviceMatrix.attach(x.tensor[:1], N)
        with pytest.raises(ValueError, match="memory of their own"):
            norm(n1, n2).forward(branch, residual, g, training=training, in_place=True)
    # these are sound: nothing is read after it was written
    norm("none", "rms").forward(x, x, in_place=True)
    norm("rms", "none").forward(x, x, training=False, in_place=True)
    norm("rms", "rms").forward(x, x)
    norm("none", "none").forward(matrix(), x, x, training=False, in_place=True)
    empty = matrix(width=0)
    norm("rms", "rms").forward(empty, empty, in_place=True)


def test_share_memory():
    """Against sets of addresses, every placement of two small matrices in one buffer."""
    rng = np.random.default_rng(5)
    buf = torch.zeros(400)

    def at(start, width, ld, height):
        return L.DeviceMatrix.attach(buf.as_strided((width, max(height, 1)), (ld, 1), start), height)

    def places(m):
        start = (m.tensor.data_ptr() - buf.data_ptr()) // 4
        return {start + c * m.ldim + r for c in range(m.width) for r in range(m.height)}

    met = [0, 0]
    for _ in range(20000):
        ld = int(rng.integers(1, 12))
        a, b = (at(int(rng.integers(0, 120)), int(rng.integers(2, 6)), ld, int(rng.integers(1, ld + 1))) for _ in range(2))
        want = bool(places(a) & places(b))
        assert L._share_memory(a, b) == want and L._share_memory(b, a) == want
        met[want] += 1
        c = at(int(rng.integers(0, 120)), int(rng.integers(1, 3)), 12, int(rng.integers(1, 12)))
        assert L._share_memory(a, c) or not places(a) & places(c)
    assert min(met) > 1000
    assert not L._share_memory(at(0, 0, 4, 4), at(0, 2, 4, 4))


def test_layers_come_and_go():
    layer = norm()
    layer.forward(matrix(), matrix())
    other = pickle.loads(pickle.dumps(layer))
    twin = copy.deepcopy(layer)
    for m in (other, twin):
        m.forward(matrix(), matrix())
    assert len(L._SAVED) == 3
    del m, other, twin
    gc.collect()
    assert len(L._SAVED) == 1
    layer.forward(matrix(), matrix(), training=False)
    assert not L._SAVED
