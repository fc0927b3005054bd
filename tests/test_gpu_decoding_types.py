"""The logits of a decoding step on their way into the softmax layers, for every storage type."""
import numpy as np
import pytest
import torch

from tests import stream_reference as ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("log", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "f16", "bf16"])
def test_adjusted_logits_into_softmax(dtype, log):
    """fp32 and fp16 pass; bfloat16, for which softmax has no kernels, is refused and nothing is touched."""
    from lbann_amd import layers as L
    v, w = 1003, 5
    rng = np.random.default_rng(3)
    kind = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}[dtype]
    x = torch.from_numpy(rng.standard_normal((w, v))).to(device="cuda", dtype=kind)
    tokens = torch.from_numpy(rng.integers(0, v, (w, 40)).astype(np.int32)).cuda()
    logits = L.logits_adjust_layer(v).forward(L.DeviceMatrix.attach(x, v), L.DeviceMatrix.attach(tokens, 40),
                                              repetition=torch.full((w,), 1.25, device="cuda"))
    softmax = L.log_softmax_layer() if log else L.softmax_layer()
    if dtype == "bf16":
        before = logits.tensor.clone()
        with pytest.raises(TypeError, match="f32 or f16 or f64"):
            softmax.forward(logits)
        with pytest.raises(TypeError):
            softmax.forward(logits, in_place=True)
        assert torch.equal(logits.tensor, before)
        return
    z, _ = ref.logits(x.double().cpu().numpy(), tokens.cpu().numpy(), None, None, np.full(w, 1.25), *[None] * 6)
    got = softmax.forward(logits).tensor.double().cpu().numpy()
    m = z.max(1, keepdims=True)
    p = np.exp(z - m)
    want = z - m - np.log(p.sum(1, keepdims=True)) if log else p / p.sum(1, keepdims=True)
    # a logit is rounded once to its type: half a step of at most |z| <= 8, for the entry and for the sum alike; then the
    # result once, half a step of itself; fp32 arithmetic within: 2^-24 times some tens of roundings of values up to 16
    half = ref.HALF_STEP[dtype]
    shift = 2 * 8 * half + 64 * 16 * 2.0 ** -24
    assert np.abs(z).max() <= 8
    bound = shift + half * np.abs(want) if log else want * (np.expm1(shift) + half) + ref.TINY[dtype]
    assert (np.abs(got - want) <= bound).all()
