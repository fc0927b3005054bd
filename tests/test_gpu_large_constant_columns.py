"""Columns of one large number: normalised they are zeros, like columns of zeros, and nothing that stands beside them (lanes
without entries, whose distance from the mean overflows when it is scaled) may show."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

# powers of two, whose fp32 means are exact in teams of any make-up; lengths below eight, where one sum is divided; and
# lengths of one wave whose rounded reciprocal times the length is one again
LENGTHS = [1, 2, 3, 5, 7, 8, 16, 32, 64, 128, 256, 1024, 2048] + [n for n in (9, 13, 24, 25, 51, 77, 99, 101, 131, 200, 333, 400, 401, 511)
                                                                  if np.float32(n) * (np.float32(1) / np.float32(n)) == 1]


def outputs(L, n, t, dtype, branch_norm, output_norm, gates, keep, o, r, dy, dh, weights, epsilon):
    A = L.DeviceMatrix.attach
    names = ("branch_scale", "branch_bias") * (branch_norm != "none") + ("output_scale", "output_bias") * (output_norm != "none")
    layer = L.residual_norm_layer(n, branch_norm, output_norm, epsilon=epsilon, keep_prob=keep, seed=3, **{k: weights[k] for k in names})
    gate = A(weights["gate"][:gates], n) if gates else None
    y = layer.forward(A(o, n), None if r is None else A(r, n), gate, offset=1)
    out = [layer.residual.tensor] + ([y.tensor] if y is not None else [])
    db, dr = layer.backward(A(dy, n) if y is not None else None, A(dh, n))
    out += [db.tensor] + ([] if dr is None else [dr.tensor])
    out += [getattr(layer, f"m_{k}_gradient").tensor for k in names]
    if gates:
        out.append(layer.m_gate_gradient.tensor)
    return out


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("gates", [0, 1])
@pytest.mark.parametrize("n", LENGTHS + [20001])
def test_branch(n, gates, dtype):
    """Behind a layer norm the branch is its bias, whatever number it held."""
    from lbann_amd import layers as L
    t = 6
    gen = torch.Generator(device="cuda").manual_seed(n)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    weights = {k: new(n) for k in ("branch_scale", "branch_bias", "output_scale", "output_bias")}
    weights["gate"] = new(1, n)
    r, dy, dh = (new(t, n).to(dtype) for _ in range(3))
    # sums stay below the largest number: n 2^k < 2^128; (0 - 2^k) / sqrt(epsilon) does not
    k, epsilon = (120, 1e-5) if n < 200 else (112, 1e-13)
    for output_norm in ("layer", "rms", "none"):
        if n == 20001:
            k, epsilon = 100, 1e-20
        args = lambda o: outputs(L, n, t, dtype, "layer", output_norm, gates, 0.9, o, r, dy, dh, weights, epsilon)  # noqa: E731
        o = torch.full((t, n), 2.0 ** k, device="cuda", dtype=dtype)
        for i, (a, b) in enumerate(zip(args(o), args(torch.zeros_like(o)))):
            assert torch.isfinite(b).all() and torch.equal(a, b), (output_norm, i)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("n", LENGTHS)
def test_stream(n, dtype):
    """A stream of one large number behind the layer norm of the next block; the gradients of both norms."""
    from lbann_amd import layers as L
    t = 5
    gen = torch.Generator(device="cuda").manual_seed(n)
    new = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    weights = {k: new(n) for k in ("branch_scale", "branch_bias", "output_scale", "output_bias")}
    dy, dh = (new(t, n).to(dtype) for _ in range(2))
    k, epsilon = (120, 1e-5) if n < 200 else (112, 1e-13)
    args = lambda o: outputs(L, n, t, dtype, "none", "layer", 0, 1.0, o, None, dy, dh, weights, epsilon)  # noqa: E731
    o = torch.full((t, n), 2.0 ** k, device="cuda", dtype=dtype)
    a, b = args(o), args(torch.zeros_like(o))
    assert torch.equal(a[0], o)
    for i, (x, y) in enumerate(zip(a[1:], b[1:])):
        assert torch.isfinite(y).all() and torch.equal(x, y), i
