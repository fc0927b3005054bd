"""Gradients of the block's output for more columns than a launch has workgroups, against the formula in 64 bits."""
import numpy as np
import pytest
import torch

from tests import stream_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [3, 8, 20])
@pytest.mark.parametrize("norm", ["rms", "layer"])
def test_block_gradient_of_many_short_columns(n, norm):
    from lbann_amd import layers as L
    t = (1 << 21) + 77
    gen = torch.Generator(device="cuda").manual_seed(n)
    o, dy = (torch.randn(t, n, generator=gen, device="cuda") for _ in range(2))
    w = 1 + 0.25 * torch.randn(n, generator=gen, device="cuda")
    A = L.DeviceMatrix.attach
    layer = L.residual_norm_layer(n, "none", norm, output_scale=w)
    layer.forward(A(o, n))
    got, none = layer.backward(A(dy, n))
    assert none is None
    worst = 0.0
    stats = layer.m_statistics.tensor.double()
    for part in torch.arange(t, device="cuda").split(1 << 18):   # a few columns at a time in 64 bits
        x, p = o[part].double(), dy[part].double() * w.double()
        mean, rstd = stats[part, 2:3], 1 / torch.sqrt(stats[part, 3:4] + 1e-5)
        hat, size_hat = (x - mean) * rstd, (x.abs() + mean.abs()) * rstd
        m = lambda a: a.mean(1, keepdim=True)  # noqa: E731
        want = rstd * (p - (m(p) if norm == "layer" else 0) - hat * m(p * hat))
        size = rstd * (p.abs() + m(p.abs()) + size_hat * m(p.abs() * size_hat))
        bound = ref.HALF_STEP["f32"] * want.abs() + ref.roundings(n) * ref.U * (size + want.abs())
        worst = max(worst, ((got.tensor[part].double() - want).abs() / bound).max().item())
    assert worst <= 1, worst
    last = ref.backward(o[-50:].double().cpu().numpy(), o[-50:].double().cpu().numpy(), None, stats[-50:].cpu().numpy(),
                        dy[-50:].double().cpu().numpy(), None,
                        {"branch_norm": "none", "output_norm": norm, "epsilon": 1e-5, "a": 1.0, "b": 1.0, "drop": None, "w1": None,
                         "b1": None, "w2": w.double().cpu().numpy(), "b2": None}, False)["dbranch"][0]
    assert np.allclose(last, want[-50:].cpu().numpy(), rtol=1e-12, atol=1e-12)   # the two forms of the formula
