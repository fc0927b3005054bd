"""The size query of the residual norm's backward: any numbers, also those that the call itself refuses."""
import pytest


def size(*args):
    from lbann_amd import capi
    return capi.lib().lbn_residual_norm_bwd_workspace_bytes(*args)


@pytest.mark.parametrize("n,width,gates", [(100, 4, 8), (100, 1, 2), (4096, 512, 513), (16, 6, 4), (16, 6, 2 ** 40), (20000, 3, 7)])
@pytest.mark.parametrize("weights", [0, 1])
def test_gates_that_do_not_divide_the_width(n, width, gates, weights):
    """More gates than columns once divided by zero, which ends the process."""
    assert size(n, width, weights, gates, 4) == 0


def test_sizes_beyond_the_limits():
    assert size(2 ** 26 + 1, 4, 1, 0, 2) == 0 and size(2 ** 62, 2 ** 62, 1, 0, 2) == 0
    assert size(64, 2 ** 32 + 1, 1, 0, 2) == 0 and size(64, 2 ** 62, 1, 2, 2) == 0
    assert size(2 ** 26, 4, 1, 0, 2) > 0 and size(64, 2 ** 32, 1, 0, 2) > 0
    assert size(-1, 4, 1, 0, 2) == 0 and size(4, -1, 1, 0, 2) == 0 and size(4, 4, 1, -1, 2) == 0


def test_gates_that_do():
    for n in (1, 7, 64, 1000, 4096, 20000):
        for width in (1, 6, 300, 7200):
            for gates in (1, 2, 3, width):
                if width % gates == 0:
                    assert size(n, width, 1, gates, 4) >= size(n, width, 1, 0, 4) * (gates == 1) and size(n, width, 0, gates, 2) >= 16 * width


def test_size_kept_by_a_layer_while_another_thread_asks(monkeypatch):
    """A call that comes between the size query of another and its use gets the size of its own shape."""
    from lbann_amd import layers as L
    made, inside = [], []

    class Library:
        @staticmethod
        def lbn_residual_norm_bwd_workspace_bytes(n, width, *rest):
            if width not in inside:   # as another thread would, at the worst moment
                inside.append(width)
                backward(width)
            return 1000 + width

    monkeypatch.setattr(L.capi, "lib", lambda: Library)
    monkeypatch.setattr(L, "_stream_for", lambda m: 0)
    monkeypatch.setattr(L, "_entry", lambda name, dtype: lambda *args: made.append((args[2], args[-1])))
    layer = L.residual_norm_layer(8, device="cpu")

    def matrix(width, height=8):
        return L.DeviceMatrix(height, width, device="cpu", fill=1.0)

    def backward(width):
        layer.bind_saved(matrix(width), matrix(width), matrix(width, 4))
        layer.backward(matrix(width), matrix(width))

    for width in (5, 9, 5):
        backward(width)
    assert len(made) == 5 and all(need == 1000 + width for width, need in made), made
    L._SAVED.clear()
