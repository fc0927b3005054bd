"""Two residual norms in a row with the stream in one buffer: what backward gives, and what it refuses."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make(L, n, output_norm, gen):
    new = lambda: torch.randn(n, generator=gen, device="cuda")  # noqa: E731
    scale = {"output_scale": new()} if output_norm != "none" else {}
    first = L.residual_norm_layer(n, "rms", output_norm, branch_scale=new(), keep_prob=0.8, seed=1, **scale)
    second = L.residual_norm_layer(n, "layer", "rms", branch_scale=new(), output_scale=new(), keep_prob=0.7, seed=2)
    return first, second


@pytest.mark.parametrize("output_norm", ["rms", "layer", "none"])
@pytest.mark.parametrize("n,t", [(72, 40), (1023, 9), (4096, 12), (12289, 3)])
def test_two_in_a_row(n, t, output_norm):
    from lbann_amd import layers as L
    gen = torch.Generator(device="cuda").manual_seed(n)
    new = lambda: torch.randn(t, n, generator=gen, device="cuda").bfloat16()  # noqa: E731
    A = L.DeviceMatrix.attach
    first, second = make(L, n, output_norm, gen)
    o1, o2, r, dy1, dy2, dh = (new() for _ in range(6))
    top = lambda dy: A(dy, n) if output_norm != "none" else None  # noqa: E731

    def forward(in_place):
        first.forward(A(o1, n), A(r.clone(), n), offset=0, in_place=in_place)
        return second.forward(A(o2, n), first.residual, offset=0, in_place=in_place)

    y = forward(False)
    do2, ds = second.backward(A(dy2, n), A(dh, n))
    do1, dr = first.backward(top(dy1), ds)
    want = [m.tensor for m in (y, second.residual, do2, ds, do1, dr, first.m_branch_scale_gradient)]
    y = forward(True)
    assert first.residual is second.residual
    do2, ds = second.backward(A(dy2, n), A(dh, n))
    same = [y, second.residual, do2, ds]
    if output_norm == "none":   # the first layer's backward does not read its stream
        do1, dr = first.backward(None, ds)
        same += [do1, dr, first.m_branch_scale_gradient]
    else:                       # it would read the second one's
        with pytest.raises(ValueError, match="overwritten"):
            first.backward(A(dy1, n), ds)
    for a, b in zip(same, want):
        assert torch.equal(a.tensor, b)
