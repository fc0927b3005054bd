"""How many sequences one call of the logits adjustment takes: the limits that include/lbnorm.h states, by length of history
and vocabulary.  Beyond them a call is refused before it touches a device; at them it runs (GPU)."""
import ctypes

import pytest

P = ctypes.c_void_p(0x1000)  # never dereferenced: refused before any launch
UNSUPPORTED = -3


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("tokens,slab,most", [(0, 2048, 2 ** 23), (1, 2048, 2 ** 23), (1023, 2048, 2 ** 23), (1024, 8192, 2 ** 22),
                                              (4095, 8192, 2 ** 22), (4096, 16384, 2 ** 21), (131072, 16384, 2 ** 21)])
def test_first_width_beyond(tokens, slab, most, suffix):
    from lbann_amd import capi
    f = getattr(capi.lib(), f"lbn_logits_adjust_{suffix}")
    for vocabulary in (1, slab, slab + 1, 5 * slab - 1, 5 * slab):
        slabs = -(-vocabulary // slab)
        for width in (-(-most // slabs), 2 * most):
            assert f(None, vocabulary, width, P, vocabulary, P, vocabulary, P if tokens else None, tokens, tokens,
                     *[None] * 5, None, 0, None, 0, 0, None, 0, 0, None) == UNSUPPORTED, (vocabulary, width)


@pytest.mark.gpu
@pytest.mark.parametrize("vocabulary,tokens,width", [(1, 1, 2 ** 23 - 1), (3, 1024, 2 ** 22 - 1), (2, 4096, 2 ** 21 - 1)])
def test_last_width_within(vocabulary, tokens, width):
    import torch

    from lbann_amd import layers as L
    A = L.DeviceMatrix.attach
    x = torch.arange(vocabulary * width, device="cuda", dtype=torch.int32).remainder_(1000).float().view(width, vocabulary)
    history = torch.zeros(width, tokens, device="cuda", dtype=torch.int32)   # entry 0 was generated once in every third sequence
    lengths = (torch.arange(width, device="cuda") % 3 == 0).int()
    two = torch.full((width,), 2.0, device="cuda")
    y = L.logits_adjust_layer(vocabulary).forward(A(x, vocabulary), A(history, tokens), lengths, presence=two).tensor
    want = x.clone()
    want[:, 0] -= 2.0 * lengths
    assert torch.equal(y, want)
