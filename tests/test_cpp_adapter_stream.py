"""The C++ adapter's dropout, residual norm and logits adjustment classes: what they refuse (CPU), and one
step through all of them against the 64-bit forms and against the Python layer classes (GPU)."""
import ctypes

import numpy as np
import pytest

from tests import stream_reference as ref
from tests.test_cpp_adapter import driver

i64, vp, cint, dbl = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_double


def test_adapter_stream_classes_refuse():
    assert driver().drv_stream_error_cases() == 0


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_adapter_stream_step(dtype):
    import torch

    from lbann_amd import layers as L
    from tests.test_gpu_stream_operators import TYPES, close
    n, w, gates, keep, length = 515, 12, 3, 0.75, 40
    gen = torch.Generator(device="cuda").manual_seed(3)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    m = [new(w, n).to(TYPES[dtype]) if i in (0, 1, 5, 6) else torch.full((w, n), float("nan"), dtype=TYPES[dtype], device="cuda")
         for i in range(11)]
    gate, dgate = new(gates, n), torch.empty(gates, n, device="cuda")
    weights, grads = [1 + 0.1 * new(n) for _ in range(4)], [torch.empty(n, device="cuda") for _ in range(4)]
    tokens = torch.randint(0, n, (w, length), generator=gen, device="cuda").to(torch.int32)
    rho = 1.0 + torch.rand(w, generator=gen, device="cuda")
    p = lambda t: vp(t.data_ptr())  # noqa: E731
    err = ctypes.create_string_buffer(512)
    rc = driver().drv_stream(cint(list(TYPES).index(dtype)), i64(n), i64(w), i64(gates), cint(1), cint(2), dbl(keep),
                             (vp * 11)(*[t.data_ptr() for t in m]), p(gate), p(dgate), (vp * 4)(*[t.data_ptr() for t in weights]),
                             (vp * 4)(*[t.data_ptr() for t in grads]), p(tokens), i64(length), p(rho),
                             vp(torch.cuda.current_stream().cuda_stream), err, cint(512))
    assert rc == 0, err.value
    A = L.DeviceMatrix.attach
    drop = L.dropout_layer(keep, seed=11)
    layer = L.residual_norm_layer(n, "rms", "layer", 1e-5, 0.75, 1.25, *weights, keep_prob=keep, seed=77)
    dropped = drop.forward(A(m[0], n))
    y = layer.forward(A(m[1], n), dropped, A(gate, n), offset=5)
    db, dd = layer.backward(A(m[5], n), A(m[6], n))
    dr = drop.backward(dd)
    adjusted = L.logits_adjust_layer(n).forward(y, A(tokens, length), repetition=rho)
    for i, t in ((2, dropped), (3, layer.residual), (4, y), (7, db), (8, dd), (9, dr), (10, adjusted)):
        assert torch.equal(m[i], t.tensor), i
    assert torch.equal(dgate, layer.m_gate_gradient.tensor)
    for t, name in zip(grads, ("branch_scale", "branch_bias", "output_scale", "output_bias")):
        assert torch.equal(t, getattr(layer, f"m_{name}_gradient").tensor), name
    # and the step's output against 64 bits
    f64 = lambda t: t.double().cpu().numpy()  # noqa: E731
    form = {"branch_norm": "rms", "output_norm": "layer", "epsilon": 1e-5, "a": 0.75, "b": 1.25, "drop": (keep, 77, 5, 0),
            **{k: f64(t) for k, t in zip(("w1", "b1", "w2", "b2"), weights)}}
    _, want, _, _, size = ref.forward(f64(m[1]), f64(m[2]), f64(gate), form)
    close("y", f64(m[4]), want, size, dtype, ref.roundings(n))
    assert np.array_equal(f64(m[2]) != 0, ref.keep_mask(n, w, keep, 11, 0) & (f64(m[0]) != 0))
