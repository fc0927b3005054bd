"""Residual norm without an epsilon over columns so small that their variance is a subnormal number."""
import numpy as np
import pytest
import torch

from tests import stream_reference as ref
from tests.test_gpu_stream_operators import KINDS, TYPES, check_backward, close, got, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["rms", "layer"])
@pytest.mark.parametrize("n", [2, 6, 64, 200, 1000, 4096, 20000])
def test_subnormal_variances(n, kind):
    """Entries of +-2^-k: their squares down to 2^-148 are exact in fp32, and so are the variances."""
    from lbann_amd import layers as L
    A = L.DeviceMatrix.attach
    powers = [-60, -63, -64, -66, -70, -74]
    sign = np.where(np.arange(n) % 2 == 0, 1.0, -1.0)
    v = np.outer([2.0 ** k for k in powers], sign)
    x = torch.from_numpy(v).float().cuda()
    dy = torch.randn(len(powers), n, generator=torch.Generator().manual_seed(n)).cuda()
    p = {"epsilon": 0.0, "a": 1.0, "b": 1.0, "drop": None, "w1": None, "b1": None, "w2": None, "b2": None}
    for branch_norm, output_norm in (("none", kind), (kind, "none")):
        layer = L.residual_norm_layer(n, branch_norm, output_norm, epsilon=0.0)
        y = layer.forward(A(x, n))
        out = y if y is not None else layer.residual
        # the variance 2^(2 k) to within one step of the subnormal numbers' grid, in sums of n / 64 + 16 additions at most
        # (all exact: multiples of it below 2^24) and one product
        stats = layer.m_statistics.tensor.double().cpu().numpy()
        assert np.array_equal(stats[:, 3 if y is not None else 1], [2.0 ** (2 * k) for k in powers])
        close("normalised", got(out), np.tile(sign, (len(powers), 1)), np.ones_like(v), "f32", ref.roundings(n))
        grads = layer.backward(A(dy, n) if y is not None else None, None if y is not None else A(dy, n))
        want = ref.backward(v, v if y is not None else got(out), None, stats, dy.double().cpu().numpy() if y is not None else None,
                            None if y is not None else dy.double().cpu().numpy(), {**p, "branch_norm": branch_norm, "output_norm": output_norm}, False)
        close("dbranch", got(grads[0]), *want["dbranch"], "f32", ref.roundings(n))


@pytest.mark.parametrize("dtype", list(TYPES))
@pytest.mark.parametrize("kinds", KINDS + [("none", "layer", 0, 0.9, True), ("layer", "rms", 0, 1.0, True)], ids=lambda k: "-".join(map(str, k)))
@pytest.mark.parametrize("n,t,pad,shift", [(8, 40, 0, 0), (72, 60, 3, 1), (200, 30, 0, 0), (640, 70, 0, 0), (1024, 66, 0, 0), (4096, 9, 0, 0),
                                           (4104, 6, 8, 8), (8192, 4, 0, 0), (12288, 3, 0, 0)])
def test_no_epsilon(n, t, pad, shift, kinds, dtype):
    """Ordinary columns of whole units without an epsilon, which the kernels for any length serve."""
    from lbann_amd import layers as L
    rng = np.random.default_rng(n + t)
    p, layer, gate, gate_v, data = make(L, rng, n, t, kinds, dtype, pad, shift)
    p["epsilon"] = layer.m_epsilon = 0.0
    h, y, _, size_h, size_y = ref.forward(data["o"][1], data["r"][1], gate_v, p)
    out = layer.forward(data["o"][0], data["r"][0], gate, offset=5)
    close("h", got(layer.residual), h, size_h, dtype, ref.roundings(n))
    if y is not None:
        close("y", got(out), y, size_y, dtype, ref.roundings(n))
    check_backward(layer, p, gate_v, data, dtype, n, t)
