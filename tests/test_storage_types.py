"""Storage types that a layer has no kernels for, and calls whose matrices differ in type: refused
before any launch, in every class.  A 2-byte matrix read as fp32 would reach twice past its end."""
import numpy as np
import pytest
import torch

from lbann_amd import layers as L

F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
DIMS = (4, 8)
LAYERS = {  # class -> (constructor, types with kernels)
    "layer_norm": (lambda: L.layer_norm_layer(DIMS, 1e-5, True, True, device="cpu"), (F32, F16)),
    "layer_norm of doubles": (lambda: L.layer_norm_layer(DIMS, device="cpu", datatype=F64), (F64,)),
    "instance_norm": (lambda: L.instance_norm_layer(DIMS, device="cpu"), (F32,)),
    "entrywise_batch_norm": (lambda: L.entrywise_batch_normalization_layer(DIMS, device="cpu"), (F32,)),
    "entrywise_batch_norm over ranks": (lambda: L.entrywise_batch_normalization_layer(DIMS, device="cpu", comm_allreduce=id), (F32,)),
    "batch_norm": (lambda: L.batch_normalization_layer(DIMS, device="cpu"), (F32, F16)),
    "batch_norm of doubles": (lambda: L.batch_normalization_layer(DIMS, device="cpu", datatype=F64), (F64,)),
    "softmax": (lambda: L.softmax_layer(device="cpu"), (F32, F16, F64)),
    "log_softmax": (lambda: L.log_softmax_layer(device="cpu"), (F32, F16, F64)),
    "channelwise_softmax": (lambda: L.channelwise_softmax_layer(DIMS, device="cpu"), (F32, F64)),
    "entrywise_scale_bias": (lambda: L.entrywise_scale_bias_layer(DIMS, device="cpu"), (F32,)),
    "channelwise_scale_bias": (lambda: L.channelwise_scale_bias_layer(DIMS, device="cpu"), (F32,)),
}


def host(dtype, height=32, width=3):
    return L.DeviceMatrix(height, width, dtype=dtype, device="cpu", fill=1)


@pytest.fixture(autouse=True)
def no_launch(monkeypatch):
    """What a refusal must come before: the stream of a call, and the call."""
    class Reached(Exception):
        pass

    def reached(*_):
        raise Reached
    monkeypatch.setattr(L, "_stream", reached)
    monkeypatch.setattr(L, "call", reached)
    return Reached


@pytest.mark.parametrize("name", list(LAYERS))
@pytest.mark.parametrize("dtype", [F32, F16, F64, BF16, torch.int32])
def test_types_without_kernels(name, dtype, no_launch):
    make, types = LAYERS[name]
    # types with kernels get as far as the stream
    with pytest.raises(no_launch if dtype in types else TypeError):
        make().forward(host(dtype))
    layer = make()
    layer.bind_forward(host(dtype))
    with pytest.raises((no_launch, AttributeError) if dtype in types else TypeError):  # no statistics without a forward
        layer.backward(host(dtype))


@pytest.mark.parametrize("name", list(LAYERS))
@pytest.mark.parametrize("dtype", [F32, F16, F64, BF16])
def test_gradients_of_another_type(name, dtype):
    make, types = LAYERS[name]
    layer = make()
    layer.bind_forward(host(types[0]))
    if dtype != types[0]:
        with pytest.raises(TypeError):
            layer.backward(host(dtype))


def test_reference_order_of_half_matrices():
    layer = L.batch_normalization_layer(DIMS, device="cpu", stats_mode=L.LBN_STATS_REFERENCE_ORDER)
    layer.bind_forward(host(F16))
    with pytest.raises(TypeError):
        layer.backward(host(F16))


def test_cross_entropy(no_launch):
    for dtype in (F32, F16, F64, BF16):
        with pytest.raises(no_launch if dtype in (F32, F16) else TypeError):
            L.cross_entropy_layer(DIMS, device="cpu").forward(host(dtype), host(dtype))
        layer = L.cross_entropy_layer(DIMS, device="cpu")
        layer.prev_activations = [host(F32), host(F32)]
        with pytest.raises(no_launch if dtype == F32 else TypeError):
            layer.backward(host(dtype, 1))
        with pytest.raises(no_launch if dtype == F32 else TypeError):
            L.softmax_cross_entropy_forward(L.softmax_layer(device="cpu"), L.cross_entropy_layer(DIMS, device="cpu"), host(dtype), host(dtype))
        if dtype != F32:
            with pytest.raises(TypeError):
                L.softmax_cross_entropy_forward(L.softmax_layer(device="cpu"), L.cross_entropy_layer(DIMS, device="cpu"), host(F32), host(dtype))
        softmax = L.softmax_layer(device="cpu")
        softmax.activations = layer.prev_activations[0]
        with pytest.raises(no_launch if dtype == F32 else TypeError):
            L.softmax_cross_entropy_backward(softmax, layer, host(dtype, 1))


def test_gradient_buffer(no_launch):
    for dtype in (F32, F16, BF16, F64):
        buffer = L.gradient_buffer(32, 3, device="cpu")
        for contribution in (host(dtype), torch.zeros(96, dtype=dtype)):
            with pytest.raises(no_launch if dtype == F32 else TypeError):
                buffer.add_to_gradient(contribution)
        if dtype != F32:
            assert buffer.status == buffer.CLEARED
    with pytest.raises(no_launch):
        buffer.add_to_gradient(L._Vector(96, "cpu", np.zeros(96)))
