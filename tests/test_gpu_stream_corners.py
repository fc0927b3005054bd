"""Calls of dropout, residual norm and logits adjustment that the interface allows and that are rarely made."""
import numpy as np
import pytest
import torch

from tests import stream_reference as ref
from tests.test_gpu_stream_operators import TYPES, close, got, matrix, test_logits_adjust as compare_logits

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def L():
    from lbann_amd import layers
    layers.capi.lib()
    return layers


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("n", [1, 5, 72, 200, 1001, 1024, 4096, 9001, 12288, 20001])
def test_a_norm_without_a_stream(L, n, dtype):
    """No stream wanted (h NULL): y alone, also in the place of the input, as from the call that writes both."""
    t = 7
    x, _ = matrix(L, np.random.default_rng(n).standard_normal((t, n)), dtype, 3, 1)
    scale = torch.randn(n, device="cuda")
    layer = L.residual_norm_layer(n, "none", "layer", output_scale=scale)
    want = layer.forward(x, training=False)
    y = L.DeviceMatrix(n, t, dtype=TYPES[dtype])
    f = "lbn_residual_norm_fwd_" + dtype
    for out in (y, x):
        L.call(f, L._stream(), n, t, 0, 2, 1e-5, 1.0, 1.0, *L._buffer(x), None, 0, None, 0, 0, None, None, scale.data_ptr(), None, 1.0, 0,
               0, None, 0, None, 0, *L._buffer(out), None, 0)
        assert np.array_equal(got(out), got(want))


@pytest.mark.parametrize("dtype", list(TYPES))
def test_the_last_columns_of_the_generator(L, dtype):
    """A mini-batch whose last column has the number 2^32 - 1, alone and inside a residual norm, forward and backward."""
    n, t = 77, 6
    drop = (0.7, 5, 2 ** 64 - 1, 2 ** 32 - t)
    factor = ref.keep_factor(n, t, drop)
    assert 0 < (factor == 0).sum() < n * t
    x, xv = matrix(L, np.random.default_rng(2).standard_normal((t, n)), dtype)
    layer = L.dropout_layer(drop[0], seed=drop[1])
    norm = L.residual_norm_layer(n, "none", "none", keep_prob=drop[0], seed=drop[1])
    for m in (layer, norm):
        m.m_column_offset = drop[3]
    want = xv * factor
    close("y", got(layer.forward(x, offset=drop[2])), want, np.abs(want), dtype, 2)
    close("dx", got(layer.backward(x)), want, np.abs(want), dtype, 2)
    norm.forward(x, offset=drop[2])
    close("h", got(norm.residual), want, np.abs(want), dtype, 3)
    close("dbranch", got(norm.backward(None, x)[0]), want, np.abs(want), dtype, 3)
    for m in (layer, norm):
        m.m_column_offset += 1
        with pytest.raises(L.LbnError):
            m.forward(x)


def test_offsets_wrap_with_their_counter(L):
    n, t = 64, 3
    layer = L.dropout_layer(0.5, seed=1)
    layer.m_step = torch.full((1,), 7, dtype=torch.int64, device="cuda")
    x = L.DeviceMatrix(n, t, fill=1.0)
    assert np.array_equal(got(layer.forward(x, offset=2 ** 64 - 3)) != 0, ref.keep_mask(n, t, 0.5, 1, 4))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("v,w,length,biases,masks,pad,shift", [(5, 2, 2, 1, 1, 0, 0), (40, 3, 3, 2, 3, 1, 1), (2048, 1, 4, 2048, 1, 0, 0),
                                                               (2049, 2, 5, 0, 2, 0, 3), (8192, 1, 1024, 0, 0, 0, 0),
                                                               (8193, 2, 1023, 40, 0, 0, 0), (16385, 2, 4096, 1100, 2, 0, 0)])
def test_short_histories_and_whole_slabs(L, v, w, length, biases, masks, pad, shift, dtype):
    compare_logits(L, v, w, length, biases, masks, pad, shift, dtype)


def test_one_gate_for_one_column(L):
    n = 1001
    rng = np.random.default_rng(1)
    p = {"branch_norm": "layer", "output_norm": "rms", "epsilon": 1e-5, "a": 1.0, "b": 1.0, "drop": None, "w1": None, "b1": None, "w2": None,
         "b2": None}
    o, ov = matrix(L, rng.standard_normal((1, n)), "f16")
    gate, gv = matrix(L, rng.standard_normal((1, n)), "f32")
    dy, dyv = matrix(L, rng.standard_normal((1, n)), "f16")
    layer = L.residual_norm_layer(n, "layer", "rms")
    y = layer.forward(o, None, gate)
    h, want, _, size_h, size_y = ref.forward(ov, None, gv, p)
    close("h", got(layer.residual), h, size_h, "f16", ref.roundings(n))
    close("y", got(y), want, size_y, "f16", ref.roundings(n))
    db, dr = layer.backward(dy)
    grads = ref.backward(ov, got(layer.h), gv, got(layer.m_statistics), dyv, None, p, False)
    assert dr is None
    close("dbranch", got(db), *grads["dbranch"], "f16", ref.roundings(n))
    close("dgate", got(layer.m_gate_gradient), *grads["dgate"], "f32", ref.roundings(n, 1))
