"""CPU-side checks of dropout, residual norm and logits adjustment: the 64-bit forms the GPU
tests compare against (known answers of the generator, gradients against differences), and what
the entry points and the layer classes refuse.  Nothing here needs a device: a refused call
returns before it touches one."""
import ctypes

import numpy as np
import pytest

from tests import stream_reference as ref


def test_generator_known_answers():
    """The answers of Philox-4x32-10 that its authors publish for their reference implementation."""
    zero = ref.philox([0, 0, 0, 0], (0, 0))
    assert [int(w) for w in zero] == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    ones = ref.philox([0xFFFFFFFF] * 4, (0xFFFFFFFF, 0xFFFFFFFF))
    assert [int(w) for w in ones] == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
    digits = ref.philox([0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344], (0xA4093822, 0x299F31D0))
    assert [int(w) for w in digits] == [0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1]


def test_mask_statistics():
    """The share of kept entries, its spread over columns and the independence of neighbours:
    each within five standard deviations of what independent draws give."""
    n, t, keep = 4096, 256, 0.9
    m = ref.keep_mask(n, t, keep, 0x123456789ABCDEF, 7).astype(float)
    q = ref.threshold(keep) / 65536
    sd = np.sqrt(q * (1 - q))
    assert abs(m.mean() - q) < 5 * sd / np.sqrt(m.size)
    assert np.abs(m.mean(1) - q).max() < 5 * sd / np.sqrt(n)
    assert np.abs(m.mean(0) - q).max() < 5 * sd / np.sqrt(t)
    d = (m - q) / sd
    for a, b in ((d[:, 1:], d[:, :-1]), (d[:, 8:], d[:, :-8]), (d[1:], d[:-1])):
        assert abs((a * b).mean()) < 5 / np.sqrt(a.size)
    other = (ref.keep_mask(n, t, keep, 0x123456789ABCDEF, 8) - q) / sd
    assert abs((other * d).mean()) < 5 / np.sqrt(d.size)
    # a batch cut in two has the mask of the whole
    assert np.array_equal(ref.keep_mask(n, 100, keep, 5, 6, 56), ref.keep_mask(n, 156, keep, 5, 6)[56:])


CASES = [(b, o, g, k) for b in ("none", "rms", "layer") for o in ("none", "rms", "layer") for g, k in ((0, 1.0), (1, 0.8), (3, 0.6))]


@pytest.mark.parametrize("branch_norm,output_norm,gates,keep", CASES)
def test_gradient_formula_against_differences(branch_norm, output_norm, gates, keep):
    rng = np.random.default_rng(11)
    t, n = 6, 13
    p = {"branch_norm": branch_norm, "output_norm": output_norm, "epsilon": 1e-3, "a": 0.7, "b": 1.3,
         "drop": (keep, 99, 4, 2)}
    x = {"o": rng.standard_normal((t, n)), "r": rng.standard_normal((t, n)),
         "gate": rng.standard_normal((gates, n)) if gates else None}
    for w, kind, base in (("w1", branch_norm, 1.0), ("b1", branch_norm, 0.0), ("w2", output_norm, 1.0), ("b2", output_norm, 0.0)):
        x[w] = base + 0.3 * rng.standard_normal(n) if kind != "none" else None
    dy = rng.standard_normal((t, n)) if output_norm != "none" else None
    dh = rng.standard_normal((t, n))

    def loss(x):
        h, y, *_ = ref.forward(x["o"], x["r"], x["gate"], {**p, **{k: x[k] for k in ("w1", "b1", "w2", "b2")}})
        return (h * dh).sum() + (0.0 if y is None else (y * dy).sum())

    pw = {**p, **{k: x[k] for k in ("w1", "b1", "w2", "b2")}}
    h, _, stats, *_ = ref.forward(x["o"], x["r"], x["gate"], pw)
    got = ref.backward(x["o"], h, x["gate"], stats, dy, dh, pw)
    names = {"o": "dbranch", "r": "dresidual", "gate": "dgate", "w1": "dbranch_scale", "b1": "dbranch_bias",
             "w2": "doutput_scale", "b2": "doutput_bias"}
    step = 1e-5
    for key, name in names.items():
        if x[key] is None:
            continue
        for _ in range(3):
            d = rng.standard_normal(x[key].shape)
            ahead, behind = ({**x, key: x[key] + s * step * d} for s in (1, -1))
            want = (loss(ahead) - loss(behind)) / (2 * step)
            # truncation step^2 times third derivatives (some hundreds at most here), rounding 2^-53 |loss| / step
            assert abs((got[name][0] * d).sum() - want) < 1e-6 * max(1.0, abs(want)), name


# ---------------------------------------------------------------- refusals (no device is touched)
def lib():
    from lbann_amd import capi
    return capi.lib()


P = ctypes.c_void_p(0x1000)  # never dereferenced: refused before any launch
INVALID, WORKSPACE, UNSUPPORTED = -1, -2, -3


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("direction", ["fwd", "bwd"])
def test_dropout_refusals(direction, suffix):
    f = getattr(lib(), f"lbn_dropout_{direction}_{suffix}")
    ok = dict(h=16, w=4, keep=0.5, seed=1, off=2, step=None, col=0, x=P, ldx=16, y=P, ldy=16)
    call = lambda **kw: f(None, *({**ok, **kw}).values())  # noqa: E731
    assert call(h=0) == 0 and call(w=0) == 0
    for bad in (dict(h=-1), dict(w=-1), dict(keep=0.0), dict(keep=-0.1), dict(keep=1.5), dict(keep=float("nan")),
                dict(x=None), dict(y=None), dict(ldx=15), dict(ldy=15), dict(col=-1)):
        assert call(**bad) == INVALID, bad
    assert call(col=2 ** 32 - 3) == UNSUPPORTED
    assert call(h=2 ** 34 + 8, w=1) == UNSUPPORTED


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
def test_residual_norm_forward_refusals(suffix):
    f = getattr(lib(), f"lbn_residual_norm_fwd_{suffix}")
    ok = dict(n=16, w=6, n1=1, n2=2, eps=1e-5, a=1.0, b=1.0, o=P, ldo=16, r=P, ldr=16, g=P, ldg=16, gates=3, w1=P, b1=P, w2=P,
              b2=P, keep=0.9, seed=0, off=0, step=None, col=0, h=P, ldh=16, y=P, ldy=16, st=P, ldst=4)
    call = lambda **kw: f(None, *({**ok, **kw}).values())  # noqa: E731
    assert call(n=0) == 0 and call(w=0) == 0
    for bad in (dict(n=-1), dict(w=-1), dict(n1=3), dict(n2=-1), dict(o=None), dict(y=None), dict(ldo=15), dict(ldr=15),
                dict(ldg=15), dict(ldh=15), dict(ldy=15), dict(ldst=3), dict(gates=4), dict(gates=0), dict(gates=-1), dict(g=None),
                dict(n1=0), dict(n1=0, w1=None), dict(n2=0), dict(n2=0, y=None), dict(n2=0, y=None, w2=None, b2=None, h=None),
                dict(keep=0.0), dict(keep=float("nan")), dict(col=-1)):
        assert call(**bad) == INVALID, bad
    assert call(col=2 ** 32 - 5) == UNSUPPORTED
    big = {k: 2 ** 26 + 1 for k in ("n", "ldo", "ldr", "ldg", "ldh", "ldy")}
    assert call(**big) == UNSUPPORTED


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
def test_residual_norm_backward_refusals(suffix):
    f = getattr(lib(), f"lbn_residual_norm_bwd_{suffix}")
    need = lib().lbn_residual_norm_bwd_workspace_bytes(16, 6, 1, 3, 4 if suffix == "f32" else 2)
    assert need > 0
    ok = dict(n=16, w=6, n1=1, n2=2, eps=1e-5, a=1.0, b=1.0, o=P, ldo=16, h=P, ldh=16, g=P, ldg=16, gates=3, w1=P, b1=P, w2=P,
              keep=0.9, seed=0, off=0, step=None, col=0, st=P, ldst=4, dy=P, lddy=16, dh=P, lddh=16, do=P, lddo=16, dr=P, lddr=16,
              dg=P, lddg=16, dw1=P, db1=P, dw2=P, db2=P, ws=P, nb=need)
    call = lambda **kw: f(None, *({**ok, **kw}).values())  # noqa: E731
    assert call(n=0) == 0 and call(w=0) == 0
    for bad in (dict(n=-1), dict(w=-1), dict(n1=3), dict(n2=7), dict(o=None), dict(h=None), dict(dy=None), dict(do=None), dict(st=None),
                dict(ldo=15), dict(ldh=15), dict(ldg=15), dict(ldst=3), dict(lddy=15), dict(lddh=15), dict(lddo=15), dict(lddr=15),
                dict(lddg=15), dict(gates=4), dict(gates=0), dict(g=None), dict(n1=0), dict(n2=0), dict(keep=2.0), dict(col=-1)):
        assert call(**bad) == INVALID, bad
    no_norm = dict(n2=0, dy=None, w2=None, dw2=None, db2=None)
    assert call(**no_norm, dh=None) == INVALID      # nothing to differentiate
    assert call(ws=None) == WORKSPACE and call(nb=need - 1) == WORKSPACE and call(ws=ctypes.c_void_p(0x1008)) == WORKSPACE
    assert call(col=2 ** 32 - 5) == UNSUPPORTED
    size = lib().lbn_residual_norm_bwd_workspace_bytes
    assert size(0, 5, 1, 0, 4) == 0 and size(5, 0, 1, 0, 4) == 0
    assert size(4096, 8192, 1, 0, 2) >= 4 * 256 * 4096 * 4     # four quantities of 256 ranges of columns


@pytest.mark.parametrize("suffix", ["f32", "f16", "bf16"])
def test_logits_adjust_refusals(suffix):
    f = getattr(lib(), f"lbn_logits_adjust_{suffix}")
    ok = dict(v=100, w=3, x=P, ldx=100, y=P, ldy=100, tok=P, ldt=20, most=20, len=P, prompt=P, rep=P, pres=P, freq=P, bt=P, ldbt=7,
              bv=P, ldbv=7, k=7, m=P, ldm=4, masks=2, index=P)
    call = lambda **kw: f(None, *({**ok, **kw}).values())  # noqa: E731
    assert call(v=0) == 0 and call(w=0) == 0
    for bad in (dict(v=-1), dict(w=-1), dict(x=None), dict(y=None), dict(ldx=99), dict(ldy=99), dict(most=-1), dict(tok=None),
                dict(ldt=19), dict(k=-1), dict(bt=None), dict(bv=None), dict(ldbt=6), dict(ldbv=6), dict(masks=-1), dict(masks=0),
                dict(m=None), dict(ldm=3), dict(index=None)):
        assert call(**bad) == INVALID, bad
    assert call(v=2 ** 31, ldx=2 ** 31, ldy=2 ** 31, ldm=2 ** 26) == UNSUPPORTED
    assert call(w=2 ** 24, ldx=2 ** 31, ldy=2 ** 31) == UNSUPPORTED
    assert call(most=131072, ldt=131072, k=8192, ldbt=8192, ldbv=8192) == UNSUPPORTED


def test_layer_classes_refuse():
    import torch

    from lbann_amd import layers as L
    with pytest.raises(ValueError):
        L.dropout_layer(keep_prob=0.0)
    with pytest.raises(ValueError):
        L.residual_norm_layer(8, branch_norm="batch")
    with pytest.raises(ValueError):
        L.residual_norm_layer(8, branch_norm="none", branch_scale=np.ones(8), device="cpu")
    with pytest.raises(ValueError):
        L.residual_norm_layer(8, output_scale=np.ones(7), device="cpu")
    host = L.DeviceMatrix(8, 2, device="cpu")
    with pytest.raises(ValueError):
        L.residual_norm_layer(9, device="cpu").forward(host)                       # another height
    with pytest.raises(ValueError):
        L.residual_norm_layer(8, device="cpu").forward(host, L.DeviceMatrix(8, 3, device="cpu"))
    with pytest.raises(ValueError):
        L.residual_norm_layer(8, device="cpu").forward(host, L.DeviceMatrix(8, 2, dtype=torch.bfloat16, device="cpu"))
    with pytest.raises(ValueError):
        L.residual_norm_layer(8, device="cpu").backward(host)                      # no forward yet
    with pytest.raises(ValueError):
        L.DeviceMatrix.attach(torch.zeros(2, 8).t(), 2)                            # columns not contiguous
    with pytest.raises(ValueError):
        L.DeviceMatrix.attach(torch.zeros(2, 8), 9)
    m = L.DeviceMatrix.attach(torch.arange(24.0).reshape(2, 12)[:, :10], 9)
    assert (m.height, m.width, m.ldim) == (9, 2, 12)


def test_dropout_offsets_advance():
    from lbann_amd import layers as L
    d = L.dropout_layer(keep_prob=0.5, seed=3)
    taken = []
    for training, offset in ((True, None), (True, None), (False, None), (True, 40), (True, None)):
        d._start(training, offset)
        taken.append((d.m_offset, d.m_kept))
    assert taken == [(0, 0.5), (1, 0.5), (1, 1.0), (40, 0.5), (2, 0.5)]


def test_layers_refuse_host_memory():
    """Without a GPU too: a refusal, not an error of the runtime."""
    from lbann_amd import layers as L
    host = L.DeviceMatrix(8, 2, device="cpu")
    weights = L.residual_norm_layer(8, output_scale=np.ones(8), device="cpu")
    for call in (lambda: L.dropout_layer(0.5).forward(host), lambda: L.logits_adjust_layer(8).forward(host), lambda: weights.forward(host)):
        with pytest.raises(ValueError, match="device memory"):
            call()
